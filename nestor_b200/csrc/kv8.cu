// Key/value cache in 8 bits: append (quantise), read back, attention over it.
//
// A list is what one attention column has seen of one sequence. The cache of a (list, head) is a run of blocks of 64
// entries with one fp32 scale per block for the keys and one for the values; a value is code * scale, codes are int8
// or e4m3. A step's rows are packed by list, `seg[l] .. seg[l + 1]`.
//
// Layout. A block's codes are units of 8 head dims x 64 entries = 32 lanes x 16 bytes, the order in which the lanes of
// a warp need them as the 16-bit A operand of mma.m16n8k16 (g = lane / 4, t = lane % 4, bytes (m, h, i)):
//   keys   : entry 16m + 8h + g,       dim 8u + 2t + i      (rows = entries, reduction = dims)
//   values : entry 16m + 8h + 2t + i,  dim 8u + g           (rows = dims, reduction = entries)
// A unit is therefore one 16-byte load per lane, coalesced in memory and without bank conflicts in shared memory, that
// needs no shuffle before the product, and the keys (the values) of a (list, head) are one contiguous stream. Head dims
// need rounding up to a multiple of 8 only; codes of dims past the head are zero.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <atomic>
#include <math.h>
#include <type_traits>
#include <stdint.h>

#include "kv8.h"
#include "sm100.cuh"

namespace nbk {

constexpr int kBlock = 64;
constexpr int kStatusRange = 7;      // a list would exceed the cache, or bounds that are not ascending: rows were skipped

// Largest l with seg[l] <= r (seg ascending, seg[0] <= r): a 32-way search, two or three dependent loads for any
// realistic number of lists. Called by whole warps.
__device__ __forceinline__ int find_list(const int* __restrict__ seg, int L, int r) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = L;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) >> 5;
    const int at = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, at < hi && seg[at] <= r);
    const int n = __popc(below);
    if (n == 0) return lo;
    lo += (n - 1) * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(float x) { return x; }
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f(float x) { return x; }
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }

// ------------------------------------------------------------------------------------------------------- append
// One CTA stores a block of one head, keys and values: entries [0, t0) come from the originals that the cache keeps
// (`open`), entries [t0, t0 + m) are new rows. The block's largest magnitude gives scale = amax / Q and
// code = round_half_even(x * (Q / amax)), Q = 127 or 448. A block with an infinity or a NaN takes the scale NaN: all its
// values are NaN. A block below 2^-100 holds zeros.
//
// A warp owns a unit (two of them above 8): its lanes load the pairs of dims of eight entries that they hold in the keys'
// layout, so nothing passes through shared memory but the warps' maxima. The values' layout is the transpose of each
// 8 x 8 tile: their codes go through movmatrix as 16-bit numbers. Instructions, not HBM, are the bound: about 14 an
// element, half of what a tile in shared memory took (197k rows x 3 heads x 40 in bf16: 55 us instead of 108; HBM alone
// would take 22). Four CTAs an SM leave 64 registers a thread, of which 16-bit rows in pairs spill 12 (48 to 52 bytes).
__device__ __forceinline__ unsigned transpose8x8(unsigned x) {
  unsigned y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {      // (a NaN stays)
  float c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}

// Two neighbouring elements as they stand in memory (one register for 16-bit types). PAIR: as one access of that size.
template <typename T> struct Raw { using type = unsigned; };
template <> struct Raw<float> { using type = float2; };
template <typename T> using Two = typename Raw<T>::type;

__device__ __forceinline__ float2 floats(unsigned v, __nv_bfloat16) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
__device__ __forceinline__ float2 floats(unsigned v, __half) { return __half22float2(reinterpret_cast<const __half2&>(v)); }
__device__ __forceinline__ float2 floats(float2 v, float) { return v; }
__device__ __forceinline__ void make_zero(unsigned& v) { v = 0u; }
__device__ __forceinline__ void make_zero(float2& v) { v = make_float2(0.f, 0.f); }

// larger of a and |v|, element by element (a NaN stays)
__device__ __forceinline__ unsigned larger(unsigned a, unsigned v, __nv_bfloat16) {
  const __nv_bfloat162 m = __hmax2_nan(reinterpret_cast<const __nv_bfloat162&>(a), __habs2(reinterpret_cast<const __nv_bfloat162&>(v)));
  return reinterpret_cast<const unsigned&>(m);
}
__device__ __forceinline__ unsigned larger(unsigned a, unsigned v, __half) {
  const __half2 m = __hmax2_nan(reinterpret_cast<const __half2&>(a), __habs2(reinterpret_cast<const __half2&>(v)));
  return reinterpret_cast<const unsigned&>(m);
}
__device__ __forceinline__ float2 larger(float2 a, float2 v, float) { return make_float2(max_nan(a.x, fabsf(v.x)), max_nan(a.y, fabsf(v.y))); }

template <typename T, bool PAIR>
__device__ __forceinline__ Two<T> load_two(const T* p, bool second) {
  if constexpr (PAIR) return *reinterpret_cast<const Two<T>*>(p);
  if constexpr (sizeof(T) == 4) return make_float2(p[0], second ? p[1] : 0.f);
  else {
    const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
    return unsigned(h[0]) | (second ? unsigned(h[1]) << 16 : 0u);
  }
}
template <typename T, bool PAIR>
__device__ __forceinline__ void store_two(T* p, Two<T> v, bool second) {
  if constexpr (PAIR) *reinterpret_cast<Two<T>*>(p) = v;
  else if constexpr (sizeof(T) == 4) {
    p[0] = v.x;
    if (second) p[1] = v.y;
  } else {
    unsigned short* h = reinterpret_cast<unsigned short*>(p);
    h[0] = static_cast<unsigned short>(v & 0xffffu);
    if (second) h[1] = static_cast<unsigned short>(v >> 16);
  }
}
__device__ __forceinline__ unsigned rounded(float2 y, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(y.x, y.y);
  return reinterpret_cast<const unsigned&>(v);
}
__device__ __forceinline__ unsigned rounded(float2 y, __half) {
  const __half2 v = __floats2half2_rn(y.x, y.y);
  return reinterpret_cast<const unsigned&>(v);
}
__device__ __forceinline__ float2 rounded(float2 y, float) { return y; }

template <int CODE>
__device__ __forceinline__ unsigned code_pair(float2 y) {          // codes of y.x and y.y in bits 0..7 and 8..15
  if constexpr (CODE == 0)
    // adding 1.5 * 2^23 leaves the integer, rounded half to even, in the low bits; |y| <= 127 (1 + 2^-23)
    return __byte_perm(__float_as_uint(__fadd_rn(y.x, 12582912.f)), __float_as_uint(__fadd_rn(y.y, 12582912.f)), 0x0040) & 0xffffu;
  else
    return __nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3);
}

struct Source {            // where a block's entries are: the first t0 in `held`, the next m in `rows`
  const void *held, *rows;
  long row_stride;
};

template <typename T, bool PAIR, int CODE, int NU>
__device__ __forceinline__ void store_block(const nb_kv8_cache& c, long lh, int b, int t0, int m, const Source (&src)[2], bool keep, float (*red)[8]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, g = lane >> 2, t = lane & 3, D = c.D, n = t0 + m;
  // (entries and dims that are not there load one that is, so that all loads are in flight at once, and become zeros)
  Two<T> x[2][NU][8];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const T* held = reinterpret_cast<const T*>(src[kv].held) + g * D;
    const T* rows = reinterpret_cast<const T*>(src[kv].rows) + (g - t0) * src[kv].row_stride;
    const T* first = t0 ? reinterpret_cast<const T*>(src[kv].held) : reinterpret_cast<const T*>(src[kv].rows);
    const long step = 8 * src[kv].row_stride;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = 8 * i + g;
      const T* from = e >= n ? first : e < t0 ? held : rows;
      held += 8 * D;
      rows += step;
#pragma unroll
      for (int a = 0; a < NU; ++a) {
        const int d = 8 * (warp + a * warps) + 2 * t;
        x[kv][a][i] = load_two<T, PAIR>(from + (d < D ? d : 0), d + 1 < D);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int a = 0; a < NU; ++a)
      if (8 * i + g >= n || 8 * (warp + a * warps) + 2 * t >= D)
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) make_zero(x[kv][a][i]);
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    Two<T> tops;
    make_zero(tops);
#pragma unroll
    for (int a = 0; a < NU; ++a)
#pragma unroll
      for (int i = 0; i < 8; ++i) tops = larger(tops, x[kv][a][i], T{});
    const float2 both = floats(tops, T{});
    float top = max_nan(both.x, both.y);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, s));
    if (lane == 0) red[kv][warp] = top;
  }
  __syncthreads();      // (behind it no thread has an older original left to load)
  if (keep) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int a = 0; a < NU; ++a) {
        const int e = 8 * i + g, d = 8 * (warp + a * warps) + 2 * t;
        if (e >= t0 && e < n && d < D)
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            T* to = reinterpret_cast<T*>(c.open[kv]) + ((lh * 2 + (b & 1)) * kBlock + e) * D + d;
            store_two<T, PAIR>(to, x[kv][a][i], d + 1 < D);
          }
      }
  }
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    float amax = red[kv][0];
    for (int w = 1; w < warps; ++w) amax = max_nan(amax, red[kv][w]);
    constexpr float Q = CODE == 0 ? 127.f : 448.f;
    const bool poison = !(amax < INFINITY), empty = amax < 0x1p-100f;
    const float fit = poison || empty ? 0.f : __fdiv_rn(Q, amax);
    uint4* out = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(c.codes[kv]) + (lh * c.nb + b) * (long(c.U) * 512)) + lane;
    if (threadIdx.x == 0) c.scale[kv][lh * c.nb + b] = poison ? __uint_as_float(0x7fc00000u) : (empty ? 0.f : __fdiv_rn(amax, Q));
    if (poison)      // (zero times a NaN is a NaN: the codes are made zero)
#pragma unroll
      for (int a = 0; a < NU; ++a)
#pragma unroll
        for (int i = 0; i < 8; ++i) make_zero(x[kv][a][i]);
#pragma unroll
    for (int a = 0; a < NU; ++a) {
      const int u = warp + a * warps;
      unsigned word[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        unsigned half[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 v = floats(x[kv][a][2 * w + i], T{});
          half[i] = code_pair<CODE>(make_float2(__fmul_rn(v.x, fit), __fmul_rn(v.y, fit)));
          if (kv == 1) half[i] = transpose8x8(__byte_perm(half[i], 0u, 0x4140));
        }
        word[w] = __byte_perm(half[0], half[1], kv == 0 ? 0x5410 : 0x6420);
      }
      if (u < c.U) out[u * 32] = make_uint4(word[0], word[1], word[2], word[3]);
    }
  }
}

// grid ceil(rows / chunk) * H (the heads of a row are neighbours, in memory and in time), a warp for each unit or two. A
// CTA looks through its chunk of rows for those that begin a
// block or a list and stores the block that each of them begins; the others exit. The two youngest blocks' new rows are
// kept as originals, by the CTA that stores the block. One case is different: an append that begins inside a block b0
// and goes on to b0 + 2 and further. Those blocks take the slot from which b0's older originals are read, so the CTA of
// the list's first row files their rows itself, after it has read them.
template <typename T, bool PAIR, int CODE, int NU>
__global__ void __launch_bounds__(256, NU == 1 ? 4 : 2) append_kernel(nb_kv8_cache c, nb_kv8_rows p, int chunk) {
  __shared__ float red[2][2][8];
  const int h = blockIdx.x % c.H, cap = c.nb * kBlock, D = c.D;
  const int end = min(p.seg[c.L], p.rows);
  int r = int(blockIdx.x / c.H) * chunk, turn = 0;
  const int r1 = min(r + chunk, end);
  const T* rows[2] = {reinterpret_cast<const T*>(p.src[0]) + h * p.head_stride[0], reinterpret_cast<const T*>(p.src[1]) + h * p.head_stride[1]};
  while (r < r1) {
    const int l = find_list(p.seg, c.L, r);
    const int s0 = p.seg[l], s1 = p.seg[l + 1], at = p.start[l];
    if (s0 > r || s1 <= r || s0 < 0) {
      if (threadIdx.x == 0) atomicCAS(c.status, 0, kStatusRange);
      if (s0 <= r) return;
      r = s0;      // (rows before the first list)
      continue;
    }
    if (s1 > end || at < 0 || long(at) + (s1 - s0) > cap) {
      if (threadIdx.x == 0) atomicCAS(c.status, 0, kStatusRange);
      r = s1;
      continue;
    }
    const long lh = long(l) * c.H + h;
    while (r < s1 && r < r1) {
      const int e = at + (r - s0), b = e / kBlock, t = e & (kBlock - 1), m = min(kBlock - t, s1 - r);
      if (r == s0 || t == 0) {
        Source src[2];
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          src[kv].held = reinterpret_cast<const T*>(c.open[kv]) + (lh * 2 + (b & 1)) * kBlock * long(D);
          src[kv].rows = rows[kv] + long(r) * p.row_stride[kv];
          src[kv].row_stride = p.row_stride[kv];
        }
        const int b0 = at / kBlock, last = (at + (s1 - s0) - 1) / kBlock;
        const bool clash = (at & (kBlock - 1)) != 0 && last >= b0 + 2;
        store_block<T, PAIR, CODE, NU>(c, lh, b, t, m, src, b >= last - 1 && (!clash || b < b0 + 2), red[turn]);
        turn ^= 1;
        if (r == s0 && clash) {
          const int from = max(last - 1, b0 + 2) * kBlock;
#pragma unroll 4
          for (int i = threadIdx.x; i < (at + (s1 - s0) - from) * D; i += blockDim.x) {
            const int q = i / D, d = i - q * D, to = from + q;
            const long place = (lh * 2 + (to / kBlock & 1)) * kBlock * long(D) + (to & (kBlock - 1)) * D + d;
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) reinterpret_cast<T*>(c.open[kv])[place] = rows[kv][long(s0 + to - at) * p.row_stride[kv] + d];
          }
        }
      }
      r += m;
    }
  }
}

// grid (L, H): re-quantises the partly filled youngest block of every list from its first len % 64 originals.
template <typename T, bool PAIR, int CODE, int NU>
__global__ void __launch_bounds__(256) truncate_kernel(nb_kv8_cache c, const int* __restrict__ len) {
  __shared__ float red[2][8];
  const int l = blockIdx.x, n = len[l];
  if (n < 0 || n > c.nb * kBlock) {
    if (threadIdx.x == 0) atomicCAS(c.status, 0, kStatusRange);
    return;
  }
  if ((n & (kBlock - 1)) == 0) return;
  const long lh = long(l) * c.H + blockIdx.y;
  Source src[2];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) src[kv] = {reinterpret_cast<const T*>(c.open[kv]) + (lh * 2 + (n / kBlock & 1)) * kBlock * long(c.D), nullptr, 0};
  store_block<T, PAIR, CODE, NU>(c, lh, n / kBlock, n & (kBlock - 1), 0, src, false, red);
}

// --------------------------------------------------------------------------------------------------------- read
template <int CODE>
__device__ __forceinline__ float2 decoded(unsigned pair) {         // of codes in bits 0..7 and 8..15
  if constexpr (CODE == 0) {
    // (128 + x in the low bits of a float with the exponent of 2^23; the subtraction is exact)
    const unsigned u = pair ^ 0x8080u;
    return make_float2(__fsub_rn(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)), 8388736.f),
                       __fsub_rn(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441)), 8388736.f));
  } else {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(pair), __NV_E4M3);
    return __half22float2(reinterpret_cast<const __half2&>(h));
  }
}

// The inverse of append, with the same division of rows over CTAs and of units over warps; rows behind the last list
// become zeros.
template <typename T, bool PAIR, int CODE, int NU>
__global__ void __launch_bounds__(256) read_kernel(nb_kv8_cache c, nb_kv8_rows p, int chunk) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, g = lane >> 2, t = lane & 3;
  const int h = blockIdx.x % c.H, cap = c.nb * kBlock, D = c.D;
  const int end = max(0, min(p.seg[c.L], p.rows));
  T* dst[2] = {reinterpret_cast<T*>(p.dst[0]) + long(h) * D, reinterpret_cast<T*>(p.dst[1]) + long(h) * D};
  const long rs = long(c.H) * D;
  // (rows are as far apart as the head of one row is wide or a multiple of it, so they share its alignment)
  const bool by16 = D * sizeof(T) % 16 == 0 && ((reinterpret_cast<uintptr_t>(p.dst[0]) | reinterpret_cast<uintptr_t>(p.dst[1])) & 15) == 0;
  auto zeros = [&](int a, int b) {
    if (by16) {
      const int n = D * int(sizeof(T)) / 16;
      for (int i = threadIdx.x; i < (b - a) * n; i += blockDim.x) {
        const int e = i / n;
        const long at = long(a + e) * rs;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) reinterpret_cast<uint4*>(dst[kv] + at)[i - e * n] = make_uint4(0u, 0u, 0u, 0u);
      }
      return;
    }
    const int n = (D + 1) / 2;
    for (int i = threadIdx.x; i < (b - a) * n; i += blockDim.x) {
      const int e = i / n, d = 2 * (i - e * n);
      Two<T> z;
      make_zero(z);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) store_two<T, PAIR>(dst[kv] + long(a + e) * rs + d, z, d + 1 < D);
    }
  };
  int r = int(blockIdx.x / c.H) * chunk;
  const int r_end = min(r + chunk, p.rows), r1 = min(r_end, end);
  if (r_end > max(r, end)) zeros(max(r, end), r_end);
  while (r < r1) {
    const int l = find_list(p.seg, c.L, r);
    const int s0 = p.seg[l], s1 = p.seg[l + 1], at = p.start[l];
    if (s0 > r || s1 <= r || s0 < 0) {
      if (threadIdx.x == 0) atomicCAS(c.status, 0, kStatusRange);
      zeros(r, s0 > r ? min(s0, r1) : r1);
      if (s0 <= r) return;
      r = s0;
      continue;
    }
    if (s1 > end || at < 0 || long(at) + (s1 - s0) > cap) {
      if (threadIdx.x == 0) atomicCAS(c.status, 0, kStatusRange);
      zeros(r, min(s1, r1));
      r = s1;
      continue;
    }
    const long lh = long(l) * c.H + h;
    while (r < s1 && r < r1) {
      const int e0 = at + (r - s0), t0 = e0 & (kBlock - 1), m = min(kBlock - t0, s1 - r), b = e0 / kBlock;
      if (r == s0 || t0 == 0) {
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const uint4* in = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(c.codes[kv]) + (lh * c.nb + b) * (long(c.U) * 512)) + lane;
          const float scale = c.scale[kv][lh * c.nb + b];
#pragma unroll
          for (int a = 0; a < NU; ++a) {
            const int u = warp + a * warps, d = 8 * u + 2 * t;
            const uint4 w4 = u < c.U ? in[u * 32] : make_uint4(0, 0, 0, 0);
            const unsigned word[4] = {w4.x, w4.y, w4.z, w4.w};
            unsigned pair[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              pair[i] = (word[i >> 1] >> (16 * (i & 1))) & 0xffffu;
              if (kv == 1) pair[i] = __byte_perm(transpose8x8(__byte_perm(pair[i], 0u, 0x4140)), 0u, 0x4420);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int e = 8 * i + g - t0;
              if (e >= 0 && e < m && d < D) {
                const float2 y = decoded<CODE>(pair[i]);
                store_two<T, PAIR>(dst[kv] + long(r + e) * rs + d, rounded(make_float2(__fmul_rn(y.x, scale), __fmul_rn(y.y, scale)), T{}), d + 1 < D);
              }
            }
          }
        }
      }
      r += m;
    }
  }
}

// ---------------------------------------------------------------------------------------------------- attention
// S^T = K q^T and O^T = V^T P^T with mma.m16n8k16 (fp16 operands, fp32 sums): the cache is the A operand, up to 8
// query columns (new rows x heads that share a key head) are the n side of one tile, NT tiles reuse a converted block.
// Both code types convert to fp16 without rounding. One pass over the entries with the running maximum and sum of the
// softmax; a block's scales multiply its scores and its partial output in fp32.
//
// What bounds it: one query reads 2 bytes of cache for 4 flops, so HBM does (192 lists of 6144 to 12288 entries x 5 x 40,
// int8, 0.71 GB: 127 us, 5.6 TB/s with both launches; 143 us with a cold L2). The tensor pipe is used because a column tile of 8 costs no more
// than one query; the conversion (0.75 instructions a code) is then the largest part of a warp's work.
//
// Precision. q is scaled per column by a power of two that takes its largest element into [2^14, 2^15), and rounded to
// fp16 (to two fp16 numbers for fp32 queries). fp16 elements above 2^-28 and bf16 elements above 2^-31 of the largest are
// exact, fp32 elements above 2^-17 of it keep 22 bits, and no element is off by more than 2^-39 of it. int8 codes x enter
// the products of 16-bit queries as 128 + x, so their fp32 sums carry 128 times the sum of the queries (of the weights),
// which is taken off at the end: a rounding of such a sum is up to 2^-23 of that. The sum of the softmax adds the rounded weights.
// For bf16 outputs (8 bits) a probability is one fp16 number, 2^7 at the running maximum: weights down to 2^-21 of the
// largest keep 11 bits, smaller ones are off by up to 2^-32 of it. For the other outputs it is two fp16 numbers, 2^15 at
// the maximum of its own block, whose sums take the block's factor in fp32: weights down to 2^-18 of their block's largest
// keep 22 bits, smaller ones are off by up to 2^-40 of it. Relative to the running maximum they would all end at 2^-32 of
// the largest weight, and 20001 entries of e^-20 beside a dominating one with the value zero would come out 10 % off.
// For bf16 the blocks' own maxima cost 3 % on long lists (134 us instead of 130), for the others nothing that shows.
//
// Division of work, without the host knowing the lengths. Few tasks (list, head, column tile) over a short cache: a CTA
// takes a task, its warps take equal runs of the blocks and join their results in shared memory. Otherwise all blocks of
// all tasks form one line that is cut into units, a warp each. A warp that owns a whole task writes its output; pieces of
// a task that is cut go to a workspace and `attn_join` adds them in order, so results do not depend on the schedule. Short
// lines: one unit a warp, of two blocks at least. Long ones (32 blocks a warp and more): five sixths in one unit a warp,
// the rest in as many smaller ones that the warps fetch as they finish, because equal shares end up to a quarter apart
// (0.7 GB: the last warp at 128 us instead of 117). A unit costs some 3 us beside its blocks (queries, scales, its piece)
// and twice the units cost the join 4 us: a line of 20 blocks a warp took 92 us so and takes 82 without, and more and
// smaller units lost as well.
//
// Prompts. A piece of hundreds of rows a list takes a tile of 16 columns through the whole list at a time, and every tile
// converts its codes again: 64 lists x 384 rows over 1152 entries, 3 x 40, take 165 us (69 TFLOP/s), 8 x 512 over 1536,
// 16 x 60, 227 us (89 TFLOP/s), a twentieth of the tensor rate. Tiles of 64 rows and more would need a kernel of their own.
constexpr float kShift = 7.f;        // log2 of the factor on the probabilities
constexpr float kTop = 15.f;         // the same where they are relative to their block's maximum
constexpr float kSlack = 8.f;        // how far (log2) a score may pass the running maximum; 2^(kShift + kSlack) fits fp16
constexpr int kMaxLists = 1024;      // lists in one launch (their prefix sums stay in shared memory)

struct Attn {
  nb_kv8_cache c;
  nb_kv8_attn a;
  int* next;          // units handed out beyond the first `workers`
  int* bad;           // whether some list's bounds were refused
  int2* cut;          // [rows][query heads]: of the item's task the first unit; the number of pieces * 16 + the item's column
  float* ws;          // pieces: slot 2u for a task that unit u continues, 2u + 1 for one that it begins
  int workers, dynamic, by_task;
  int first;          // whether these lists are the first (their rows begin at 0)
  unsigned polls;     // looks at a copy's barrier before the wait for it gives up
};

constexpr int kShares = 1;           // small units for each warp of a long line
constexpr int kLong = 32;            // blocks a warp from which on a line is long (a small unit has 5 blocks then)
struct Cuts {
  long total, head;                  // blocks; those in the first `workers` units
  int workers, units;
  __device__ __forceinline__ Cuts(const Attn& k, long t) : total(t) {
    if (k.dynamic && t >= long(kLong) * k.workers) {
      workers = k.workers;
      units = (1 + kShares) * workers;
      head = t - t / 6;
    } else {
      units = workers = int(max(1l, min(long(k.workers), t / 2)));
      head = t;
    }
  }
  __device__ __forceinline__ long begin(int u) const {
    return u <= workers ? u * head / workers : head + (u - workers) * (total - head) / (units - workers);
  }
  __device__ __forceinline__ int of(long pos) const {
    return pos < head ? int(((pos + 1) * workers - 1) / head) : workers + int(((pos - head + 1) * (units - workers) - 1) / (total - head));
  }
};

__device__ __forceinline__ void mma(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d = a b + (c0, c1, c0, c1): the first product of a chain, with what a column's sums begin at
__device__ __forceinline__ void mma_from(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1, float c0, float c1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %10, %11};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ unsigned pack(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return reinterpret_cast<const unsigned&>(h);
}
__device__ __forceinline__ float2 unpack(unsigned x) { return __half22float2(reinterpret_cast<const __half2&>(x)); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Four codes -> two half2 (bytes 0, 1 and bytes 2, 3). e4m3 is a subset of fp16. An int8 with its sign bit flipped is
// u = 128 + x. RAW: the byte alone, the fp16 subnormal u 2^-24; the products' sums carry 128 sum(q), which the caller
// takes off (3 instructions for 4 codes). Otherwise the byte in the low bits of an fp16 with the exponent of 1024 reads
// 1152 + x, and the subtraction is exact (5 instructions, for results that keep more than 16 bits).
template <int CODE, bool RAW>
__device__ __forceinline__ void widen(unsigned w, unsigned& lo, unsigned& hi) {
  if constexpr (CODE == 0 && RAW) {
    const unsigned x = w ^ 0x80808080u;
    lo = __byte_perm(x, 0u, 0x4140);
    hi = __byte_perm(x, 0u, 0x4342);
  } else if constexpr (CODE == 0) {
    const unsigned x = w ^ 0x80808080u;
    const __half2 bias = __floats2half2_rn(1152.f, 1152.f);
    unsigned a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
    __half2 p = __hsub2(reinterpret_cast<__half2&>(a), bias), q = __hsub2(reinterpret_cast<__half2&>(b), bias);
    lo = reinterpret_cast<unsigned&>(p);
    hi = reinterpret_cast<unsigned&>(q);
  } else {
    const __half2_raw p = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w & 0xffffu), __NV_E4M3);
    const __half2_raw q = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w >> 16), __NV_E4M3);
    lo = reinterpret_cast<const unsigned&>(p);
    hi = reinterpret_cast<const unsigned&>(q);
  }
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}

__device__ __forceinline__ void store_any(void* base, long i, int type, float x) {
  if (type == 2) reinterpret_cast<float*>(base)[i] = x;
  else if (type == 1) reinterpret_cast<__half*>(base)[i] = __float2half_rn(x);
  else reinterpret_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(x);
}

// What a list brings to a launch: rows n from s0 on, entries len, blocks nb, column tiles.
struct ListWork { int s0, n, len, nb, tiles; };
__device__ __forceinline__ ListWork sized(int s0, int n, int len, int group, int columns) {
  ListWork w;
  w.s0 = s0;
  w.n = n;
  w.len = len;
  w.nb = max(1, (len + kBlock - 1) / kBlock);
  w.tiles = (n * group + columns - 1) / columns;
  return w;
}
__device__ __forceinline__ ListWork list_work(const Attn& k, int l, int end, int columns) {      // end = seg[L]
  const int s0 = k.a.seg[l], s1 = k.a.seg[l + 1], len = k.a.len[l];
  return sized(s0, s0 >= 0 && s1 <= min(k.a.rows, end) ? max(0, s1 - s0) : 0, min(max(len, 0), k.c.nb * kBlock), k.a.group, columns);
}

__device__ __forceinline__ bool covered(const Attn& k, int row, int end, int columns) {      // by a list whose bounds hold
  const ListWork w = list_work(k, find_list(k.a.seg, k.c.L, row), end, columns);
  return row >= w.s0 && row < w.s0 + w.n;
}

__device__ __forceinline__ float tile_max(const float (&s)[4][4], int i) {
  return fmaxf(fmaxf(fmaxf(s[0][i], s[0][2 + i]), fmaxf(s[1][i], s[1][2 + i])), fmaxf(fmaxf(s[2][i], s[2][2 + i]), fmaxf(s[3][i], s[3][2 + i])));
}

// One CTA an SM, as many warps as its registers carry. Shared memory of one warp: a ring filled by bulk copies that the
// warp itself issues. Nothing is shared between warps after the prologue, so there is no barrier but the copies' own.
// Narrow heads: two stages of a block (keys and values together, one wait a block). Wide heads: three stages of half a
// block, which leaves room for more warps. 16 x 10 KB, 16 x 12 KB, 12 x 15 KB or 8 x 24 KB. Measured against the other ring,
// with as many warps as then fit (long lists on the device, us): heads of 40 127 and 130, 5 rows x 2 heads of 40 74 and 79;
// heads of 60 155 and 154 (12 warps), 5 rows of 60 82 and 83, 5 rows x 2 heads of 80 63 and 60, heads of 80 106 and 106 (10
// warps), heads of 128 119 and 120 (6 warps), 8 heads of 128 on one in fp32 38 and 40 (6 warps).
__host__ __device__ constexpr int halves_of(int umax) { return umax <= 5 ? 2 : 1; }
__host__ __device__ constexpr int stages_of(int umax) { return umax <= 5 ? 2 : 3; }
__host__ __device__ constexpr int warps_of(int umax, int nt) { return nt > 1 ? (umax <= 5 ? 12 : 8) : umax <= 8 ? 16 : umax <= 10 ? 12 : 8; }

__device__ __forceinline__ uint4 lds(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}

// A place in the line of blocks: list, head, column tile, block and the blocks from here on that follow in one run.
struct Run {
  int l, h, tile, b, blocks;
  ListWork w;
};
// (By tasks the line counts tasks, and the run is the share of one of `warps` warps.)
__device__ __forceinline__ Run run_at(const Attn& k, const long* cum, const int* lists, long pos, long end, int columns, int warp, int warps) {
  int lo = 0, hi = k.c.L;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cum[mid] <= pos) lo = mid; else hi = mid;
  }
  const ListWork w = sized(lists[3 * lo], lists[3 * lo + 1], lists[3 * lo + 2], k.a.group, columns);
  const int in_list = int(pos - cum[lo]), task = k.by_task ? in_list : in_list / w.nb;
  Run r;
  r.l = lo;
  r.h = task / w.tiles;
  r.tile = task - r.h * w.tiles;
  if (k.by_task) {
    r.b = warp * w.nb / warps;
    r.blocks = (warp + 1) * w.nb / warps - r.b;
  } else {
    r.b = in_list - task * w.nb;
    r.blocks = int(min(long(w.nb - r.b), end - pos));
  }
  r.w = w;
  return r;
}

template <int UMAX, int NT, int CODE, typename T>
__global__ void __launch_bounds__(warps_of(UMAX, NT) * 32, 1) attn_kernel(const Attn k) {
  constexpr int PAIRS = (UMAX + 1) / 2, COLS = 8 * NT, STAGES = stages_of(UMAX), HALVES = halves_of(UMAX), WARPS = warps_of(UMAX, NT);
  // fp16 numbers that a query element and a probability are held in
  constexpr int QS = sizeof(T) == 4 ? 2 : 1, PS = std::is_same_v<T, __nv_bfloat16> ? 1 : 2;
  // int8 codes enter the products as (128 + x) 2^-24
  constexpr bool RAW = QS == 1, BIASED = RAW && CODE == 0;
  constexpr bool LOCAL = PS == 2;      // probabilities are relative to their own block's maximum
  constexpr float kUnit = BIASED ? 0x1p24f : 1.f;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long part[WARPS];
  __shared__ uint64_t bars[WARPS][STAGES];
  const int L = k.c.L, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int U = k.c.U, D = k.c.D;
  const uint32_t half = U * 512;
  const uint32_t stage = half * HALVES;
  uint8_t* ring = smem + warp * STAGES * stage;
  long* cum = reinterpret_cast<long*>(smem + WARPS * STAGES * stage);      // [L + 1] blocks (or tasks) before list l
  int* lists = reinterpret_cast<int*>(cum + L + 1);                         // [L][3] first row, rows, entries
  asm volatile("griddepcontrol.launch_dependents;");      // (attn_join waits for this grid before it reads what it wrote)

  // ---- prefix sums of the lists' work
  const int seg_end = k.a.seg[L];
  bool bad = false;
#pragma unroll 4
  for (int l = threadIdx.x; l < L; l += WARPS * 32) {
    const ListWork w = list_work(k, l, seg_end, COLS);
    cum[l + 1] = w.n ? k.c.H * w.tiles * (k.by_task ? 1 : w.nb) : 0;
    lists[3 * l] = w.s0;
    lists[3 * l + 1] = w.n;
    lists[3 * l + 2] = w.len;
    bad = bad || k.a.seg[l + 1] > min(k.a.rows, seg_end) || k.a.seg[l] < 0 || k.a.seg[l + 1] < k.a.seg[l];
    bad = bad || (k.first && l == 0 && w.s0 != 0);
    if (k.a.len[l] > k.c.nb * kBlock && blockIdx.x == 0) atomicCAS(k.c.status, 0, kStatusRange);
  }
  if (lane < STAGES) nb::mbar_init(&bars[warp][lane], 1);
  nb::fence_barrier_init();
  bad = __syncthreads_or(bad);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    if (!k.by_task) *k.bad = bad;
    if (bad) atomicCAS(k.c.status, 0, kStatusRange);
  }
  const int each = (L + blockDim.x - 1) / blockDim.x, l0 = min(L, int(threadIdx.x) * each), l1 = min(L, l0 + each);
  long sum = 0;
  for (int l = l0; l < l1; ++l) sum += cum[l + 1];
  long incl = sum;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const long v = __shfl_up_sync(0xffffffffu, incl, s);
    if (lane >= s) incl += v;
  }
  if (lane == 31) part[warp] = incl;
  __syncthreads();
  long base = incl - sum;
  for (int w = 0; w < warp; ++w) base += part[w];
  for (int l = l0; l < l1; ++l) {
    base += cum[l + 1];
    cum[l + 1] = base;
  }
  if (threadIdx.x == 0) cum[0] = 0;
  __syncthreads();
  const long total = cum[L];
  if (k.by_task && (k.a.zero_tail || bad))      // (with units attn_join does this)
    for (int r = blockIdx.x * WARPS + warp; r < k.a.rows; r += gridDim.x * WARPS)
      if (r >= seg_end ? k.a.zero_tail : bad && !covered(k, r, seg_end, COLS))
        for (int i = lane; i < k.c.H * k.a.group * D; i += 32)
          reinterpret_cast<T*>(k.a.out)[long(r) * k.a.o_row + long(i / D) * k.a.o_head + i % D] = from_f<T>(0.f);
  if (total == 0) return;
  const Cuts cuts(k, total);
  int unit = warp * gridDim.x + blockIdx.x;
  if (!k.by_task && unit >= cuts.workers) return;

  // ---- the copies, over run and unit borders, STAGES ahead: keys of a block and its values (in one stage or in two), the
  // next block, ... A unit that the copies fetch is `unit_next` until the arithmetic gets there (units are longer than the
  // ring, so there is never more than one).
  long feed_pos = 0, feed_end = 0, feed_at = 0;
  int feed_left = 0, feed_slot = 0, unit_next = -1;
  bool feed_values = false, more = !k.by_task && cuts.units > cuts.workers;
  if (!k.by_task) {
    feed_pos = cuts.begin(unit);
    feed_end = cuts.begin(unit + 1);
  }
  auto feed = [&]() {
    if (feed_left == 0) {
      if (feed_pos >= feed_end) {
        if (!more) return;
        int u = 0;
        if (lane == 0) u = cuts.workers + atomicAdd(k.next, 1);
        u = __shfl_sync(0xffffffffu, u, 0);
        more = u < cuts.units;
        if (!more) return;
        unit_next = u;
        feed_pos = cuts.begin(u);
        feed_end = cuts.begin(u + 1);
      }
      const Run r = run_at(k, cum, lists, feed_pos, feed_end, COLS, 0, 1);
      feed_at = ((long(r.l) * k.c.H + r.h) * k.c.nb + r.b) * long(half);
      feed_left = r.blocks;
      feed_pos += r.blocks;
    }
    if (lane == 0) {
      uint64_t* bar = &bars[warp][feed_slot];
      uint8_t* to = ring + feed_slot * stage;
      nb::mbar_expect_tx(bar, stage);
      if (HALVES == 2) {
        nb::bulk_load(to, reinterpret_cast<const uint8_t*>(k.c.codes[0]) + feed_at, half, bar);
        nb::bulk_load(to + half, reinterpret_cast<const uint8_t*>(k.c.codes[1]) + feed_at, half, bar);
      } else {
        nb::bulk_load(to, reinterpret_cast<const uint8_t*>(k.c.codes[feed_values ? 1 : 0]) + feed_at, half, bar);
      }
    }
    feed_slot = feed_slot + 1 == STAGES ? 0 : feed_slot + 1;
    if (HALVES == 2 || feed_values) {
      feed_at += half;
      --feed_left;
    }
    feed_values = !feed_values;
  };
  if (!k.by_task)
#pragma unroll 1
    for (int i = 0; i < STAGES; ++i) feed();
  int slot = 0;
  uint32_t parity = 0;
  const uint32_t ring_at = nb::smem_u32(ring) + lane * 16;
  // Waits for the copy in `slot`. Where the wait gives up, the status word is set, whatever is still in flight gets a
  // bounded time of its own, and the warp goes on at `gave_up`.
  auto landed = [&]() {
    for (uint32_t i = 0; i < k.polls; ++i)
      if (__all_sync(0xffffffffu, nb::mbar_try_wait(&bars[warp][slot], parity))) return true;
    if (lane == 0) atomicCAS(k.c.status, 0, int(nb::kTimeoutFull));
    do {
      for (uint32_t j = 0; j < nb::kSpinLimit; ++j)
        if (nb::mbar_try_wait(&bars[warp][slot], parity)) break;
      slot = slot + 1 == STAGES ? 0 : slot + 1;
      if (slot == 0) parity ^= 1;
    } while (slot != feed_slot);
    __syncwarp();
    return false;
  };
  auto release = [&]() {
    __syncwarp();
    feed();
    slot = slot + 1 == STAGES ? 0 : slot + 1;
    if (slot == 0) parity ^= 1;
  };

  // (floats of a column's piece: its output, not yet divided, the maximum and the sum)
  const int width = 8 * U + 2;
  // by tasks: joins what the warps left in their rings; all warps call it together
  auto join_task = [&](const ListWork& w, int h, int tile) {
    __syncthreads();
    const int n = min(COLS, w.n * k.a.group - tile * COLS);
    for (int i = threadIdx.x; i < n * D; i += WARPS * 32) {
      const int in_tile = i / D, d = i - in_tile * D, c = tile * COLS + in_tile, row = c / k.a.group;
      const float* from = reinterpret_cast<const float*>(smem) + in_tile * width;
      float top = -INFINITY, x = 0.f, z = 0.f;
#pragma unroll
      for (int q = 0; q < WARPS; ++q) top = fmaxf(top, from[q * (STAGES * stage / 4) + 8 * U]);
#pragma unroll
      for (int q = 0; q < WARPS; ++q) {
        const float m = from[q * (STAGES * stage / 4) + 8 * U], f = m == top ? 1.f : ex2(m - top);
        x += f * from[q * (STAGES * stage / 4) + d];
        z += f * from[q * (STAGES * stage / 4) + 8 * U + 1];
      }
      reinterpret_cast<T*>(k.a.out)[long(w.s0 + row) * k.a.o_row + long(h * k.a.group + c - row * k.a.group) * k.a.o_head + d] =
          from_f<T>(z == 0.f ? 0.f : x / z);
    }
    nb::fence_async_smem();      // (the rings are written by copies again)
    __syncthreads();
  };

  long pos = k.by_task ? long(blockIdx.x) : cuts.begin(unit), pos_end = k.by_task ? total : cuts.begin(unit + 1), run_from = 0;
  while (true) {
    if (pos >= pos_end) {
      if (unit_next < 0) break;
      unit = unit_next;
      unit_next = -1;
      pos = cuts.begin(unit);
      pos_end = cuts.begin(unit + 1);
    }
    const Run run = run_at(k, cum, lists, pos, pos_end, COLS, warp, WARPS);
    const ListWork w = run.w;
    const int h = run.h, tile = run.tile, b0 = run.b, b1 = run.b + run.blocks;
    run_from = pos;
    pos += k.by_task ? long(gridDim.x) : run.blocks;
    if (k.by_task) {
      feed_at = ((long(run.l) * k.c.H + run.h) * k.c.nb + run.b) * long(half);
      feed_left = run.blocks;
#pragma unroll 1
      for (int i = 0; i < STAGES; ++i) feed();
    }
    const long lh = long(run.l) * k.c.H + h;
    const float* ksp = k.c.scale[0] + lh * k.c.nb;
    const float* vsp = k.c.scale[1] + lh * k.c.nb;
    float ks_32 = 0.f, vs_32 = 0.f;            // scales of 32 blocks, one a lane
    if (b0 + lane < b1) {
      ks_32 = ksp[b0 + lane];
      vs_32 = vsp[b0 + lane];
    }

    // ---- queries: column g of each tile as the B operand, scaled by a power of two
    unsigned qb[NT][PAIRS][2][QS];
    float qf[NT][2], s_from[NT][2];      // factor on a column's scores; what its sums begin at
    int see[NT][2], seen_least = 0x7fffffff;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int col = tile * COLS + nt * 8 + g, a = col / k.a.group;
      const bool valid = a < w.n;
      // (columns and dims that are not there load one that is, so that all loads are in flight at once)
      const T* from = reinterpret_cast<const T*>(k.a.q) + long(w.s0 + (valid ? a : 0)) * k.a.q_row +
                      long(h * k.a.group + (valid ? col - a * k.a.group : 0)) * k.a.q_head;
      T raw[PAIRS][4];
#pragma unroll
      for (int j = 0; j < PAIRS; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = 16 * j + (i >> 1) * 8 + 2 * t + (i & 1);
          raw[j][i] = from[d < D ? d : 0];
        }
      float x[PAIRS][4], top = 0.f;
#pragma unroll
      for (int j = 0; j < PAIRS; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = 16 * j + (i >> 1) * 8 + 2 * t + (i & 1);
          x[j][i] = valid && d < D ? to_f(raw[j][i]) : 0.f;
          top = fmaxf(top, fabsf(x[j][i]));
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      constexpr unsigned LIFT = 14;
      const unsigned ex = min(max(__float_as_uint(top) >> 23, LIFT + 1u), 254u);       // biased exponent
      const float down = __uint_as_float((254u + LIFT - ex) << 23), up = __uint_as_float((ex - LIFT) << 23);
      float q_sum = 0.f;
#pragma unroll
      for (int j = 0; j < PAIRS; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float a0 = x[j][2 * i] * down, a1 = x[j][2 * i + 1] * down;
          qb[nt][j][i][0] = pack(a0, a1);
          const float2 r = unpack(qb[nt][j][i][0]);
          if constexpr (QS == 2) qb[nt][j][i][QS - 1] = pack(a0 - r.x, a1 - r.y);
          if constexpr (BIASED) q_sum += r.x + r.y;
        }
      if constexpr (BIASED) {
        q_sum += __shfl_xor_sync(0xffffffffu, q_sum, 1);
        q_sum += __shfl_xor_sync(0xffffffffu, q_sum, 2);
      }
      // the score fragment holds columns 2t and 2t + 1
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        qf[nt][i] = __shfl_sync(0xffffffffu, up, (2 * t + i) * 4) * k.a.scale_log2;
        s_from[nt][i] = BIASED ? -128.f / kUnit * __shfl_sync(0xffffffffu, q_sum, (2 * t + i) * 4) : 0.f;
        const int c = tile * COLS + nt * 8 + 2 * t + i, row = c / k.a.group;
        see[nt][i] = row < w.n ? max(0, w.len - (w.n - 1 - row)) : 0;
        if (row < w.n) seen_least = min(seen_least, see[nt][i]);
      }
    }
    seen_least = __reduce_min_sync(0xffffffffu, seen_least);
    // Beyond 2^16 a fused product and difference, against a maximum that was rounded, can end above what fp16 holds. Where
    // 32 blocks' scales allow such scores (a score is at most the factors times D codes times 2^15), both are rounded.
    float q_top = qf[0][0];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) q_top = fmaxf(q_top, fmaxf(qf[nt][0], qf[nt][1]));
    q_top = fmaxf(q_top, __shfl_xor_sync(0xffffffffu, q_top, 1));
    q_top = fmaxf(q_top, __shfl_xor_sync(0xffffffffu, q_top, 2)) * (0.5f * (CODE == 0 ? 127.f : 448.f) * D);
    bool far = __any_sync(0xffffffffu, q_top * ks_32 >= 1.f);

    // Sums of the weights come from the tensor pipe too: rows of ones, the unused second half of the last pair where
    // UMAX is odd, a product of their own where it is even.
    constexpr bool SPARE = UMAX & 1;
    constexpr unsigned kOnes = 0x3c003c00u;
    float o[PAIRS][NT][4], mx[NT][2], sm[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < PAIRS; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][nt][i] = 0.f;
      mx[nt][0] = mx[nt][1] = -INFINITY;
      sm[nt][0] = sm[nt][1] = 0.f;
    }

    for (int b = b0; b < b1; ++b) {
      const int in_32 = (b - b0) & 31;
      if (in_32 == 0 && b != b0 && b + lane < b1) {
        ks_32 = ksp[b + lane];
        vs_32 = vsp[b + lane];
      }
      if (in_32 == 0 && b != b0) far = __any_sync(0xffffffffu, q_top * ks_32 >= 1.f);
      // (kUnit here and not in qf, which it would take past fp32 for queries of 2^122 and more)
      const float ks_now = __shfl_sync(0xffffffffu, ks_32, in_32) * kUnit, vs_now = __shfl_sync(0xffffffffu, vs_32, in_32);
      // ---- scores of 64 entries
      if (!landed()) goto gave_up;
      const uint32_t keys_at = ring_at + slot * stage;
      float s[NT][4][4];
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        const uint4 z0 = 2 * j < U ? lds(keys_at + 2 * j * 512) : make_uint4(0, 0, 0, 0);
        uint4 z1 = make_uint4(0, 0, 0, 0);
        if (2 * j + 1 < UMAX && 2 * j + 1 < U) z1 = lds(keys_at + (2 * j + 1) * 512);
        const unsigned x[4] = {z0.x, z0.y, z0.z, z0.w}, y[4] = {z1.x, z1.y, z1.z, z1.w};
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          unsigned a0, a1, a2 = 0, a3 = 0;
          widen<CODE, RAW>(x[m], a0, a1);
          if (2 * j + 1 < UMAX) widen<CODE, RAW>(y[m], a2, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < QS; ++q) {
              if (j == 0 && q == 0) mma_from(s[nt][m], a0, a1, a2, a3, qb[nt][j][0][q], qb[nt][j][1][q], s_from[nt][0], s_from[nt][1]);
              else mma(s[nt][m], a0, a1, a2, a3, qb[nt][j][0][q], qb[nt][j][1][q]);
            }
        }
      }
      if (HALVES == 1) release();
      // ---- softmax; a block in which some column's view ends takes the masked form
      const bool masked = (b + 1) * kBlock > seen_least;
      float f[NT][2], vs_col[NT][2], base[NT][2], by_block[NT][2];      // by_block: factor on the block's sums (LOCAL)
      bool grows = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (masked) {
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (b * kBlock + 16 * m + (i >> 1) * 8 + g >= see[nt][i & 1]) s[nt][m][i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          f[nt][i] = qf[nt][i] * ks_now;
          vs_col[nt][i] = vs_now;
          if (masked && b * kBlock >= see[nt][i]) vs_col[nt][i] = 0.f;
          if constexpr (!LOCAL) grows |= tile_max(s[nt], i) * f[nt][i] > mx[nt][i] + kSlack;
        }
      }
      if constexpr (LOCAL) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = tile_max(s[nt], i);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16)) * f[nt][i];
            const bool some = top > -INFINITY;      // (no entry of the block is visible, or all scores are NaN)
            const float now = fmaxf(mx[nt][i], top), keep = now == mx[nt][i] ? 1.f : ex2(mx[nt][i] - now);
            base[nt][i] = some ? top : 0.f;
            by_block[nt][i] = some ? ex2(top - now) : 0.f;
            vs_col[nt][i] *= by_block[nt][i];
            mx[nt][i] = now;
            sm[nt][i] *= keep;
#pragma unroll
            for (int j = 0; j < PAIRS; ++j) {
              o[j][nt][i] *= keep;
              o[j][nt][2 + i] *= keep;
            }
          }
      }
      // The running maximum follows a column's true one with a lag of at most kSlack, so most blocks leave it (and the
      // accumulators) alone: one vote instead of six shuffles and a rescaling.
      if (!LOCAL && __any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = tile_max(s[nt], i);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const float now = fmaxf(mx[nt][i], top * f[nt][i]), keep = now == mx[nt][i] ? 1.f : ex2(mx[nt][i] - now);
            mx[nt][i] = now;
            sm[nt][i] *= keep;
#pragma unroll
            for (int j = 0; j < PAIRS; ++j) {
              o[j][nt][i] *= keep;
              o[j][nt][2 + i] *= keep;
            }
          }
      }
      if constexpr (!LOCAL)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) base[nt][i] = mx[nt][i];
      if (far) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const float x = __fsub_rn(__fmul_rn(s[nt][m][2 * q + i], f[nt][i]), base[nt][i]);
                s[nt][m][2 * q + i] = x > kSlack ? kSlack : x;      // (a NaN stays)
              }
            f[nt][i] = 1.f;
            base[nt][i] = 0.f;
          }
      }
      unsigned pb[NT][4][2][PS];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        constexpr float SHIFT = LOCAL ? kTop : kShift;
        const float2 from = make_float2(SHIFT - base[nt][0], SHIFT - base[nt][1]);
        const float2 by = make_float2(f[nt][0], f[nt][1]);
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 e = fma2(make_float2(s[nt][m][2 * i], s[nt][m][2 * i + 1]), by, from);
            s[nt][m][2 * i] = ex2(e.x);
            s[nt][m][2 * i + 1] = ex2(e.y);
          }
        if (masked) {
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (b * kBlock + 16 * m + (i >> 1) * 8 + g >= see[nt][i & 1]) s[nt][m][i] = 0.f;
        }
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const unsigned hi = pack(s[nt][m][2 * i], s[nt][m][2 * i + 1]);
            pb[nt][m][i][0] = transpose8x8(hi);
            if constexpr (PS == 2) {
              const float2 r = unpack(hi);
              pb[nt][m][i][PS - 1] = transpose8x8(pack(s[nt][m][2 * i] - r.x, s[nt][m][2 * i + 1] - r.y));
            }
          }
      }
      // ---- output of these entries
      if (HALVES == 1 && !landed()) goto gave_up;
      const uint32_t values_at = ring_at + slot * stage + (HALVES - 1) * half;
      const bool past_end = CODE != 0 && (b + 1) * kBlock > w.len;
      // (the last pair first: its spare rows bring the sums of the weights, from which the others' bias follows)
      float ones[NT][2];
      if constexpr (!SPARE) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float acc[4];
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int q = 0; q < PS; ++q) {
              if (m == 0 && q == 0) mma_from(acc, kOnes, kOnes, kOnes, kOnes, pb[nt][m][0][q], pb[nt][m][1][q], 0.f, 0.f);
              else mma(acc, kOnes, kOnes, kOnes, kOnes, pb[nt][m][0][q], pb[nt][m][1][q]);
            }
          ones[nt][0] = acc[0];
          ones[nt][1] = acc[1];
        }
      }
      float v_from[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) v_from[nt][i] = BIASED && !SPARE ? -128.f / kUnit * ones[nt][i] : 0.f;
#pragma unroll
      for (int j = PAIRS - 1; j >= 0; --j) {
        float acc[NT][4];
        const uint4 z0 = 2 * j < U ? lds(values_at + 2 * j * 512) : make_uint4(0, 0, 0, 0);
        uint4 z1 = make_uint4(0, 0, 0, 0);
        if (2 * j + 1 < UMAX && 2 * j + 1 < U) z1 = lds(values_at + (2 * j + 1) * 512);
        unsigned x[4] = {z0.x, z0.y, z0.z, z0.w}, y[4] = {z1.x, z1.y, z1.z, z1.w};
        if (past_end) {      // entries that the list does not hold may be any bytes, NaN codes too
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            unsigned keep_bytes = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (b * kBlock + 16 * m + (q >> 1) * 8 + 2 * t + (q & 1) < w.len) keep_bytes |= 0xffu << (8 * q);
            x[m] &= keep_bytes;
            y[m] &= keep_bytes;
          }
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          unsigned a0, a1 = kOnes, a2, a3 = kOnes;
          widen<CODE, RAW>(x[m], a0, a2);
          if (2 * j + 1 < UMAX) widen<CODE, RAW>(y[m], a1, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < PS; ++q) {
              if (m == 0 && q == 0) mma_from(acc[nt], a0, a1, a2, a3, pb[nt][m][0][q], pb[nt][m][1][q], v_from[nt][0], v_from[nt][1]);
              else mma(acc[nt], a0, a1, a2, a3, pb[nt][m][0][q], pb[nt][m][1][q]);
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (SPARE && j == PAIRS - 1) {
            ones[nt][0] = acc[nt][2];
            ones[nt][1] = acc[nt][3];
            if constexpr (BIASED) {
              v_from[nt][0] = -128.f / kUnit * ones[nt][0];
              v_from[nt][1] = -128.f / kUnit * ones[nt][1];
              acc[nt][0] += v_from[nt][0];
              acc[nt][1] += v_from[nt][1];
            }
          }
          const float2 vs = make_float2(vs_col[nt][0], vs_col[nt][1]);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            if (q == 1 && SPARE && j == PAIRS - 1) continue;
            const float2 into = fma2(make_float2(acc[nt][2 * q], acc[nt][2 * q + 1]), vs, make_float2(o[j][nt][2 * q], o[j][nt][2 * q + 1]));
            o[j][nt][2 * q] = into.x;
            o[j][nt][2 * q + 1] = into.y;
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 2; ++i) sm[nt][i] = LOCAL ? fmaf(ones[nt][i], by_block[nt][i], sm[nt][i]) : sm[nt][i] + ones[nt][i];
      }
      release();
    }

    // ---- the piece's result
    const bool whole = !k.by_task && b0 == 0 && b1 == w.nb;
    // (by tasks into the warp's own ring, which holds nothing by now)
    float* to_piece = k.by_task ? reinterpret_cast<float*>(ring) : k.ws + long(2 * unit + (b0 == 0 ? 1 : 0)) * COLS * width;
    int pieces = 1;
    if (!whole && !k.by_task && b0 == 0) pieces = cuts.of(run_from + w.nb - 1) - unit + 1;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float z = sm[nt][i];
        const int in_tile = nt * 8 + 2 * t + i, c = tile * COLS + in_tile, row = c / k.a.group, head = h * k.a.group + c - row * k.a.group;
        if (row >= w.n) continue;
        if (whole) {
          const float inv = z == 0.f ? 0.f : kUnit / z;
          const long at = long(w.s0 + row) * k.a.o_row + long(head) * k.a.o_head;
#pragma unroll
          for (int j = 0; j < PAIRS; ++j)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int d = 16 * j + 8 * q + g;
              if (d < D) reinterpret_cast<T*>(k.a.out)[at + d] = from_f<T>(o[j][nt][2 * q + i] * inv);
            }
        } else {
          float* to = to_piece + in_tile * width;
#pragma unroll
          for (int j = 0; j < PAIRS; ++j)
#pragma unroll
            for (int q = 0; q < 2; ++q)
              if (16 * j + 8 * q + g < 8 * U) to[16 * j + 8 * q + g] = o[j][nt][2 * q + i] * kUnit;
          if (g == 0) {
            to[8 * U] = mx[nt][i];
            to[8 * U + 1] = z;
          }
        }
        if (!k.by_task && b0 == 0 && g == 0) k.cut[long(w.s0 + row) * k.c.H * k.a.group + head] = make_int2(unit, pieces * 16 + in_tile);
      }
    if (k.by_task) join_task(w, h, tile);
  }
  return;

gave_up:      // The warp copies nothing more, but walks through the rest of its work, units that it can still fetch
              // included, and leaves NaN: every piece that a join reads is written, and no row looks computed.
  pos = run_from;
  while (true) {
    if (pos >= pos_end) {
      if (unit_next < 0 && more) {
        int u = 0;
        if (lane == 0) u = cuts.workers + atomicAdd(k.next, 1);
        u = __shfl_sync(0xffffffffu, u, 0);
        more = u < cuts.units;
        if (more) unit_next = u;
      }
      if (unit_next < 0) break;
      unit = unit_next;
      unit_next = -1;
      pos = cuts.begin(unit);
      pos_end = cuts.begin(unit + 1);
    }
    const Run run = run_at(k, cum, lists, pos, pos_end, COLS, warp, WARPS);
    const ListWork& w = run.w;
    const bool whole = !k.by_task && run.b == 0 && run.blocks == w.nb;
    const int n = min(COLS, w.n * k.a.group - run.tile * COLS), pieces = whole ? 1 : cuts.of(pos + w.nb - 1) - unit + 1;
    const float nan = __uint_as_float(0x7fc00000u);
    float* piece = k.by_task ? reinterpret_cast<float*>(ring) : k.ws + long(2 * unit + (run.b == 0 ? 1 : 0)) * COLS * width;
    for (int i = lane; i < n * (whole ? D : width); i += 32) {
      const int in_tile = i / D, c = run.tile * COLS + in_tile, row = c / k.a.group, head = run.h * k.a.group + c - row * k.a.group;
      if (whole) reinterpret_cast<T*>(k.a.out)[long(w.s0 + row) * k.a.o_row + long(head) * k.a.o_head + i - in_tile * D] = from_f<T>(nan);
      else piece[i] = nan;
    }
    if (!k.by_task && run.b == 0 && lane < n) {
      const int c = run.tile * COLS + lane, row = c / k.a.group;
      k.cut[long(w.s0 + row) * k.c.H * k.a.group + run.h * k.a.group + c - row * k.a.group] = make_int2(unit, pieces * 16 + lane);
    }
    pos += k.by_task ? long(gridDim.x) : run.blocks;
    if (k.by_task) join_task(w, run.h, run.tile);
  }
}

// Adds the pieces of each (row, query head) whose task was cut, in their order. TEAM warps share an item: the fewer items,
// the more pieces their tasks are cut into, so 16, 4 or 1. Rows behind the last list become zeros when
// `zero_tail` is set. What it is bound by is the chain of loads behind the main kernel's end: the item's cut, then all
// pieces at once.
template <int TEAM>
__global__ void __launch_bounds__((TEAM < 4 ? 4 : TEAM) * 32) attn_join(const Attn k, int cols) {
  constexpr int WARPS = TEAM < 4 ? 4 : TEAM;
  __shared__ float tops[WARPS], sums[WARPS], acc_s[WARPS][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, member = warp % TEAM, heads = k.c.H * k.a.group;
  const long item = blockIdx.x * long(WARPS / TEAM) + warp / TEAM;
  const int row = int(item / heads), head = int(item - long(row) * heads);
  const int L = k.c.L, D = k.c.D, width = 8 * k.c.U + 2, seg_begin = k.a.seg[0], seg_end = k.a.seg[L];
  const bool exists = item < long(k.a.rows) * heads;
  bool live = exists && (row >= seg_begin || k.first) && row < seg_end;      // (rows before the first list: bounds that are bad)
  const long at = long(row) * k.a.o_row + long(head) * k.a.o_head;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int2 cut = live ? k.cut[item] : make_int2(0, 0);
  bool zero = exists && k.a.zero_tail && row >= seg_end;
  if (*k.bad && live && !covered(k, row, seg_end, cols)) {
    live = false;
    zero = true;
  }
  if (zero)
    for (int d = lane + 32 * member; d < D; d += 32 * TEAM) store_any(k.a.out, at + d, k.a.q_type, 0.f);
  const int n = live ? cut.y >> 4 : 0, col = cut.y & 15;      // (at most 16 columns a tile)
  if (n <= 1) return;                  // (with TEAM > 1 the CTA has one item)
  float top = -INFINITY, acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll 4
  for (int i = member; i < n; i += TEAM) {
    const float* from = k.ws + (long(2 * (cut.x + i) + (i == 0 ? 1 : 0)) * cols + col) * width;
    const float m = from[8 * k.c.U], z = from[8 * k.c.U + 1];
    float x[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] = from[min(lane + 32 * q, D - 1)];      // (no branch: the loads of four pieces are in flight at once)
    const float now = fmaxf(top, m), keep = top == now ? 1.f : ex2(top - now), f = m == now ? 1.f : ex2(m - now);
    top = now;
    sum = sum * keep + f * z;
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[q] = acc[q] * keep + f * x[q];
  }
  if constexpr (TEAM > 1) {
#pragma unroll
    for (int q = 0; q < 4; ++q) acc_s[warp][lane + 32 * q] = acc[q];
    if (lane == 0) {
      tops[warp] = top;
      sums[warp] = sum;
    }
    __syncthreads();
    top = -INFINITY;
#pragma unroll
    for (int i = 0; i < TEAM; ++i) top = fmaxf(top, tops[i]);
    float x = 0.f;
    sum = 0.f;
    const int d = threadIdx.x;         // (at least 128 threads, at most 128 dims)
    if (d >= D) return;
#pragma unroll
    for (int i = 0; i < TEAM; ++i) {
      const float f = tops[i] == top ? 1.f : ex2(tops[i] - top);
      sum += f * sums[i];
      x += f * acc_s[i][d];
    }
    store_any(k.a.out, at + d, k.a.q_type, sum == 0.f ? 0.f : x / sum);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (lane + 32 * q < D) store_any(k.a.out, at + lane + 32 * q, k.a.q_type, sum == 0.f ? 0.f : acc[q] / sum);
  }
}

// ------------------------------------------------------------------------------------------------------ launches
using AttnFn = void (*)(const Attn);

template <int UMAX, int NT, int CODE>
AttnFn pick_type(int type) {
  return type == 0 ? attn_kernel<UMAX, NT, CODE, __nv_bfloat16> : type == 1 ? attn_kernel<UMAX, NT, CODE, __half> : attn_kernel<UMAX, NT, CODE, float>;
}
template <int UMAX, int NT>
AttnFn pick_code(int code, int type) {
  return code == 0 ? pick_type<UMAX, NT, 0>(type) : pick_type<UMAX, NT, 1>(type);
}

// Column tiles of 8: one for single tokens, two when several rows or shared heads bring more columns (a converted
// block then serves both); four would not fit the registers of the wider heads.
int tiles_for(long columns) { return columns <= 8 ? 1 : 2; }

int width_of(int U) { return U <= 5 ? 5 : U <= 8 ? 8 : U <= 10 ? 10 : 16; }

AttnFn pick(int U, int nt, int code, int type) {
  if (U <= 5) return nt == 1 ? pick_code<5, 1>(code, type) : pick_code<5, 2>(code, type);
  if (U <= 8) return nt == 1 ? pick_code<8, 1>(code, type) : pick_code<8, 2>(code, type);
  if (U <= 10) return nt == 1 ? pick_code<10, 1>(code, type) : pick_code<10, 2>(code, type);
  return nt == 1 ? pick_code<16, 1>(code, type) : pick_code<16, 2>(code, type);
}

int multiprocessors() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

int variant(int U, int nt, int code, int type) {
  const int w = U <= 5 ? 0 : U <= 8 ? 1 : U <= 10 ? 2 : 3;
  return ((w * 2 + (nt - 1)) * 2 + code) * 3 + type;
}

// Lets `fn` use up to `kSmem` bytes of dynamic shared memory (once for each device and variant: the call takes a
// microsecond and the answer does not change).
constexpr int kSmem = 226 * 1024;
cudaError_t allow_smem(AttnFn fn, int which) {
  constexpr int kDevices = 16;
  static std::atomic<bool> done[kDevices][48];
  int dev = 0;
  cudaError_t rc = cudaGetDevice(&dev);
  if (rc != cudaSuccess || (dev < kDevices && done[dev][which].load(std::memory_order_relaxed))) return rc;
  rc = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (rc == cudaSuccess && dev < kDevices) done[dev][which].store(true, std::memory_order_relaxed);
  return rc;
}

long slot_floats(int U, int cols) { return long(cols) * (8 * U + 2); }


// Whether every pair of dims (2i, 2i + 1) of every row is aligned to the pair's size.
bool pairs(int D, int size, const long* strides, int n_strides, const void* const* ptrs, int n_ptrs) {
  bool ok = D % 2 == 0;
  for (int i = 0; i < n_strides; ++i) ok = ok && strides[i] % 2 == 0;
  for (int i = 0; i < n_ptrs; ++i) ok = ok && reinterpret_cast<uintptr_t>(ptrs[i]) % (2 * size) == 0;
  return ok;
}

// f(type tag, pair tag, code tag, units-a-warp tag) for the run-time values
template <typename F>
void with_types(int type, bool pair, int code, int U, F f) {
  auto by_units = [&](auto t, auto v, auto k) {
    if (U <= 8) f(t, v, k, std::integral_constant<int, 1>{});
    else f(t, v, k, std::integral_constant<int, 2>{});
  };
  auto by_code = [&](auto t, auto v) {
    if (code == 0) by_units(t, v, std::integral_constant<int, 0>{});
    else by_units(t, v, std::integral_constant<int, 1>{});
  };
  auto by_pair = [&](auto t) {
    if (pair) by_code(t, std::true_type{});
    else by_code(t, std::false_type{});
  };
  if (type == 0) by_pair(__nv_bfloat16{});
  else if (type == 1) by_pair(__half{});
  else by_pair(float{});
}
int unit_threads(int U) { return 32 * (U <= 8 ? U : (U + 1) / 2); }

// Rows that one CTA looks through: as many as a list brings on average (at most `max_rows`), so that it finds one block or
// two, up to a block. Long runs take four blocks where that still leaves two waves of CTAs (the search for the list and
// the first load are paid once).
int chunk_of(int rows, int max_rows, int heads, int lists) {
  const int each = std::max(1, std::min((rows + lists - 1) / lists, max_rows));
  if (each < kBlock) return each;
  return long(rows) * heads / (4 * kBlock) >= 2l * 12 * multiprocessors() ? 4 * kBlock : kBlock;
}

bool bad_cache(const nb_kv8_cache* c) {
  return c->D < 1 || c->D > 128 || c->U != (c->D + 7) / 8 || c->H < 1 || c->H > 65535 || c->L < 1 || c->nb < 1 || c->nb >= (1 << 25) || !c->status || c->code < 0 || c->code > 1;
}

}  // namespace nbk

extern "C" {

int nb_kv8_append(const nb_kv8_cache* c, const nb_kv8_rows* p, cudaStream_t st) {
  using namespace nbk;
  if (bad_cache(c) || p->rows < 0) return -1;
  if (p->rows == 0) return 0;
  const long strides[4] = {p->row_stride[0], p->row_stride[1], p->head_stride[0], p->head_stride[1]};
  const void* ptrs[4] = {p->src[0], p->src[1], c->open[0], c->open[1]};
  const bool pair = pairs(c->D, c->type == 2 ? 4 : 2, strides, 4, ptrs, 4);
  const int chunk = chunk_of(p->rows, p->max_rows, c->H, c->L);
  const long grid = (long(p->rows) + chunk - 1) / chunk * c->H;
  if (grid > 0x7fffffffl) return -1;
  with_types(c->type, pair, c->code, c->U, [&](auto t, auto v, auto k, auto n) {
    append_kernel<decltype(t), decltype(v)::value, decltype(k)::value, decltype(n)::value><<<unsigned(grid), unit_threads(c->U), 0, st>>>(*c, *p, chunk);
  });
  return int(cudaGetLastError());
}

int nb_kv8_truncate(const nb_kv8_cache* c, const int* len, cudaStream_t st) {
  using namespace nbk;
  if (bad_cache(c)) return -1;
  const void* ptrs[2] = {c->open[0], c->open[1]};
  const bool pair = pairs(c->D, c->type == 2 ? 4 : 2, nullptr, 0, ptrs, 2);
  with_types(c->type, pair, c->code, c->U, [&](auto t, auto v, auto k, auto n) {
    truncate_kernel<decltype(t), decltype(v)::value, decltype(k)::value, decltype(n)::value><<<dim3(c->L, c->H), unit_threads(c->U), 0, st>>>(*c, len);
  });
  return int(cudaGetLastError());
}

int nb_kv8_read(const nb_kv8_cache* c, const nb_kv8_rows* p, int type, cudaStream_t st) {
  using namespace nbk;
  if (bad_cache(c) || p->rows < 0) return -1;
  if (p->rows == 0) return 0;
  const void* ptrs[2] = {p->dst[0], p->dst[1]};
  const bool pair = pairs(c->D, type == 2 ? 4 : 2, nullptr, 0, ptrs, 2);
  const int chunk = chunk_of(p->rows, p->max_rows, c->H, c->L);
  const long grid = (long(p->rows) + chunk - 1) / chunk * c->H;
  if (grid > 0x7fffffffl) return -1;
  with_types(type, pair, c->code, c->U, [&](auto t, auto v, auto k, auto n) {
    read_kernel<decltype(t), decltype(v)::value, decltype(k)::value, decltype(n)::value><<<unsigned(grid), unit_threads(c->U), 0, st>>>(*c, *p, chunk);
  });
  return int(cudaGetLastError());
}

}      // extern "C"
namespace nbk {
// What the host knows of an attention call: tile columns, whether a CTA takes whole tasks, the most tasks, the workspace.
struct Plan {
  int nt, cols, width, warps, sms;
  bool by_task;
  long tasks, bytes;
};
Plan plan_of(int L, int H, int nb, int D, int rows, int max_rows, int group) {
  Plan p;
  const int U = (D + 7) / 8;
  const long columns = std::min(long(max_rows), long(rows)) * group;
  p.nt = tiles_for(columns);
  p.cols = 8 * p.nt;
  p.width = width_of(U);
  p.warps = warps_of(p.width, p.nt);
  p.sms = multiprocessors();
  p.tasks = std::min(long(rows) * group, std::min(long(rows), long(L)) * ((columns + p.cols - 1) / p.cols)) * H;
  // by tasks: at most two a CTA and four blocks a warp (4096 entries of a narrow head); beyond that the longest task would
  // decide. 8 lists x 2 heads of 400 entries take 7.4 us instead of 11.2 with units, and a call costs the host 19 us instead
  // of 23 (one launch, no workspace). Towards the rule's end the device gains nothing (80 x 3 x 40 of 2000 entries: 17.5 and
  // 17.4; 80 x 3 x 60 of 2250: 24.5 instead of 21.9), the host's call still does.
  p.by_task = L <= kMaxLists && nb <= 4 * p.warps && p.tasks <= 2l * p.sms;
  p.bytes = p.by_task ? 0 : 16 + 8l * rows * H * group + long(p.sms) * p.warps * (1 + kShares) * 2 * slot_floats(U, p.cols) * 4;
  return p;
}
}      // namespace nbk
extern "C" {

// Bytes of workspace that such an attention call takes (0: none).
long nb_kv8_attention_workspace(int L, int H, int nb, int D, int rows, int max_rows, int group) {
  return nbk::plan_of(L, H, nb, D, rows, max_rows, group).bytes;
}

// `polls`: looks at a copy's barrier before a wait for it gives up (0: at once).
int nb_kv8_attention(const nb_kv8_cache* c, const nb_kv8_attn* a, void* ws, long ws_bytes, unsigned polls, cudaStream_t st) {
  using namespace nbk;
  if (bad_cache(c) || a->rows < 0 || a->group < 1 || a->max_rows < 1) return -1;
  // (a list's tasks are counted in 32 bits)
  if (long(a->rows) * a->group > (1l << 30) || long(c->H) * ((long(a->rows) * a->group + 7) / 8) * c->nb > 0x7fffffffl) return -3;
  if (a->rows == 0) return 0;
  const Plan plan = plan_of(c->L, c->H, c->nb, c->D, a->rows, a->max_rows, a->group);
  if (plan.bytes > ws_bytes) return -2;
  AttnFn fn = pick(c->U, plan.nt, c->code, a->q_type);
  const int L_smem = c->L < kMaxLists ? c->L : kMaxLists;
  const size_t smem = size_t(plan.warps) * stages_of(plan.width) * halves_of(plan.width) * c->U * 512 + 8 + L_smem * 20;
  cudaError_t rc = allow_smem(fn, variant(c->U, plan.nt, c->code, a->q_type));
  if (rc != cudaSuccess) return int(rc);
  Attn k;
  k.c = *c;
  k.a = *a;
  k.by_task = plan.by_task;
  k.first = 1;
  k.polls = polls;
  k.dynamic = k.workers = 0;
  k.next = k.bad = nullptr;
  k.cut = nullptr;
  k.ws = nullptr;
  if (plan.by_task) {
    fn<<<int(std::min(long(plan.sms), plan.tasks)), plan.warps * 32, smem, st>>>(k);
    return int(cudaGetLastError());
  }
  k.next = reinterpret_cast<int*>(ws);
  k.bad = k.next + 1;
  k.cut = reinterpret_cast<int2*>(k.next + 4);
  const long items = long(a->rows) * c->H * a->group;
  k.ws = reinterpret_cast<float*>(k.cut + items);
  for (int l0 = 0; l0 < c->L; l0 += kMaxLists) {      // (more lists than one launch holds: slices, in stream order)
    k.c.L = c->L - l0 < kMaxLists ? c->L - l0 : kMaxLists;
    const long lh = long(l0) * c->H * c->nb;
    for (int i = 0; i < 2; ++i) {
      k.c.codes[i] = reinterpret_cast<uint8_t*>(c->codes[i]) + lh * c->U * 512;
      k.c.scale[i] = c->scale[i] + lh;
    }
    k.first = l0 == 0;
    k.a.seg = a->seg + l0;
    k.a.len = a->len + l0;
    k.a.zero_tail = a->zero_tail && l0 + k.c.L >= c->L;
    k.dynamic = plan.tasks * c->nb >= long(kLong) * plan.sms * plan.warps;
    if (k.dynamic && (rc = cudaMemsetAsync(k.next, 0, sizeof(int), st)) != cudaSuccess) return int(rc);
    const int grid = k.dynamic ? plan.sms : int(std::min(long(plan.sms), std::max(plan.tasks * c->nb, 1l)));
    k.workers = grid * plan.warps;
    fn<<<grid, plan.warps * 32, smem, st>>>(k);
    if ((rc = cudaGetLastError()) != cudaSuccess) return int(rc);
    const int team = items <= 2l * plan.sms ? 16 : items <= 32l * plan.sms ? 4 : 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(team > 1 ? items : (items + 3) / 4));
    cfg.blockDim = dim3(team > 4 ? team * 32 : 128);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    using Join = void (*)(const Attn, int);
    const Join join = team == 16 ? attn_join<16> : team == 4 ? attn_join<4> : attn_join<1>;
    rc = cudaLaunchKernelEx(&cfg, join, k, plan.cols);
    if (rc != cudaSuccess) return int(rc);
  }
  return 0;
}

}  // extern "C"
