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
// A unit is therefore one fully coalesced 16-byte load per lane straight into registers: the attention stages nothing
// in shared memory, has no bank conflicts and no barriers, and a (list, head) is one contiguous stream. Head dims need
// rounding up to a multiple of 8 only.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <type_traits>
#include <stdint.h>

#include "kv8.h"

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

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Vec { T x[VEC]; };

// Entry and dim of byte b (0..15) of lane (g, t) in unit u.
__device__ __forceinline__ int unit_entry(int kv, int g, int t, int b) {
  return ((b >> 2) << 4) + (((b >> 1) & 1) << 3) + (kv ? 2 * t + (b & 1) : g);
}
__device__ __forceinline__ int unit_dim(int kv, int g, int t, int b) { return kv ? g : 2 * t + (b & 1); }

// ------------------------------------------------------------------------------------------------------- append
// One CTA stores one block of one head of the keys or the values: entries [0, t0) come from the originals that the
// cache keeps (`open`), entries [t0, t0 + m) are new rows. The block's largest magnitude (compared as integers, so that
// a NaN counts as the largest) gives scale = amax / Q and code = round_half_even(x * (Q / amax)), Q = 127 or 448.
// A block with an infinity or a NaN takes the scale NaN: all its values are NaN. A block below 2^-100 holds zeros.
template <typename T, int VEC, int CODE>
__device__ __forceinline__ void store_block(const nb_kv8_cache& c, int kv, long lh, int b, int t0, int m,
                                            const T* __restrict__ src, long row_stride, float* tile, unsigned* red) {
  const int D = c.D, pitch = D | 1, nv = D / VEC, T_tok = t0 + m;
  const T* held = reinterpret_cast<const T*>(c.open[kv]) + ((lh * 2 + (b & 1)) * kBlock) * long(D);
  unsigned top = 0;
  for (int i = threadIdx.x; i < T_tok * nv; i += blockDim.x) {
    const int e = i / nv, j = (i - e * nv) * VEC;
    const T* from = e < t0 ? held + long(e) * D + j : src + long(e - t0) * row_stride + j;
    const Vec<T, VEC> v = *reinterpret_cast<const Vec<T, VEC>*>(from);
#pragma unroll
    for (int q = 0; q < VEC; ++q) {
      const float f = to_f(v.x[q]);
      top = max(top, __float_as_uint(f) & 0x7fffffffu);
      tile[e * pitch + j + q] = f;
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int w = 0; w < int(blockDim.x >> 5); ++w) top = max(top, red[w]);
  constexpr float Q = CODE == 0 ? 127.f : 448.f;
  const float amax = __uint_as_float(top);
  const bool poison = top >= 0x7f800000u, empty = amax < 0x1p-100f;
  const float fit = poison || empty ? 0.f : __fdiv_rn(Q, amax);
  const float scale = poison ? __uint_as_float(0x7fc00000u) : (empty ? 0.f : __fdiv_rn(amax, Q));
  uint4* out = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(c.codes[kv]) + (lh * c.nb + b) * (long(c.U) * 512));
  for (int i = threadIdx.x; i < c.U * 32; i += blockDim.x) {
    const int u = i >> 5, g = (i >> 2) & 7, t = i & 3;
    unsigned word[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float y[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int e = unit_entry(kv, g, t, 4 * w + q), d = 8 * u + unit_dim(kv, g, t, 4 * w + q);
        y[q] = fit != 0.f && e < T_tok && d < D ? __fmul_rn(tile[e * pitch + d], fit) : 0.f;
      }
      if constexpr (CODE == 0) {
        // adding 1.5 * 2^23 leaves the integer, rounded half to even, in the low bits; |y| <= 127 (1 + 2^-23)
        unsigned r[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) r[q] = __float_as_uint(__fadd_rn(y[q], 12582912.f)) & 0xffu;
        word[w] = r[0] | (r[1] << 8) | (r[2] << 16) | (r[3] << 24);
      } else {
        const unsigned a = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
        const unsigned z = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
        word[w] = a | (z << 16);
      }
    }
    out[i] = make_uint4(word[0], word[1], word[2], word[3]);
  }
  if (threadIdx.x == 0) c.scale[kv][lh * c.nb + b] = scale;
}

// grid (ceil(rows / chunk), H, 2). A CTA looks through its chunk of rows for those that begin a block or a list and
// stores the block that each of them begins; the others exit. `chunk` is 1 for steps of few rows a list (every row may
// begin a block: one CTA each) and 64 for prompts (one block a CTA). The CTA of a list's first row also files the
// originals of the new rows of the youngest two blocks: it alone reads the older originals, so nothing races with it.
template <typename T, int VEC, int CODE>
__global__ void __launch_bounds__(128) append_kernel(nb_kv8_cache c, nb_kv8_rows p, int chunk) {
  extern __shared__ float tile[];
  __shared__ unsigned red[4];
  const int kv = blockIdx.z, h = blockIdx.y, cap = c.nb * kBlock;
  const int end = min(p.seg[c.L], p.rows);
  int r = blockIdx.x * chunk;
  const int r1 = min(r + chunk, end);
  const long rs = p.row_stride[kv];
  const T* rows = reinterpret_cast<const T*>(p.src[kv]) + h * p.head_stride[kv];
  while (r < r1) {
    const int l = find_list(p.seg, c.L, r);
    const int s0 = p.seg[l], s1 = p.seg[l + 1], at = p.start[l];
    if (s0 > r || s1 <= r || s0 < 0) {
      if (threadIdx.x == 0) atomicCAS(c.status, 0, kStatusRange);
      return;
    }
    if (s1 > end || at < 0 || long(at) + (s1 - s0) > cap) {
      if (threadIdx.x == 0) atomicCAS(c.status, 0, kStatusRange);
      r = s1;
      continue;
    }
    const long lh = long(l) * c.H + h;
    while (r < s1 && r < r1) {
      const int e = at + (r - s0), t = e & (kBlock - 1), m = min(kBlock - t, s1 - r);
      if (r == s0 || t == 0) {
        store_block<T, VEC, CODE>(c, kv, lh, e / kBlock, t, m, rows + long(r) * rs, rs, tile, red);
        __syncthreads();
        if (r == s0) {
          const int last = (at + (s1 - s0) - 1) / kBlock, from = max(at, (last - 1) * kBlock), nv = c.D / VEC;
          T* held = reinterpret_cast<T*>(c.open[kv]) + lh * 2 * kBlock * long(c.D);
          for (int i = threadIdx.x; i < (at + (s1 - s0) - from) * nv; i += blockDim.x) {
            const int q = i / nv, j = (i - q * nv) * VEC, to = from + q;
            *reinterpret_cast<Vec<T, VEC>*>(held + ((to / kBlock & 1) * kBlock + (to & (kBlock - 1))) * long(c.D) + j) =
                *reinterpret_cast<const Vec<T, VEC>*>(rows + long(s0 + to - at) * rs + j);
          }
        }
      }
      r += m;
    }
  }
}

// grid (L, H, 2): re-quantises the partly filled youngest block of every list from its first len % 64 originals.
template <typename T, int VEC, int CODE>
__global__ void __launch_bounds__(128) truncate_kernel(nb_kv8_cache c, const int* __restrict__ len) {
  extern __shared__ float tile[];
  __shared__ unsigned red[4];
  const int l = blockIdx.x, n = len[l];
  if (n < 0 || n > c.nb * kBlock) {
    if (threadIdx.x == 0) atomicCAS(c.status, 0, kStatusRange);
    return;
  }
  if ((n & (kBlock - 1)) == 0) return;
  store_block<T, VEC, CODE>(c, blockIdx.z, long(l) * c.H + blockIdx.y, n / kBlock, n & (kBlock - 1), 0, nullptr, 0, tile, red);
}

// --------------------------------------------------------------------------------------------------------- read
// The inverse of append, with the same division of rows over CTAs; rows behind the last list become zeros.
template <typename T, int VEC, int CODE>
__global__ void __launch_bounds__(128) read_kernel(nb_kv8_cache c, nb_kv8_rows p, int chunk) {
  extern __shared__ float tile[];
  const int kv = blockIdx.z, h = blockIdx.y, cap = c.nb * kBlock, D = c.D, pitch = D | 1, nv = D / VEC;
  const int end = max(0, min(p.seg[c.L], p.rows));
  T* dst = reinterpret_cast<T*>(p.dst[kv]) + long(h) * D;
  const long rs = long(c.H) * D;
  auto zeros = [&](int a, int b) {
    Vec<T, VEC> z;
#pragma unroll
    for (int q = 0; q < VEC; ++q) z.x[q] = from_f<T>(0.f);
    for (int i = threadIdx.x; i < (b - a) * nv; i += blockDim.x) {
      const int e = i / nv, j = (i - e * nv) * VEC;
      *reinterpret_cast<Vec<T, VEC>*>(dst + long(a + e) * rs + j) = z;
    }
  };
  int r = blockIdx.x * chunk;
  const int r_end = min(r + chunk, p.rows), r1 = min(r_end, end);
  if (r_end > max(r, end)) zeros(max(r, end), r_end);
  while (r < r1) {
    const int l = find_list(p.seg, c.L, r);
    const int s0 = p.seg[l], s1 = min(p.seg[l + 1], p.rows), at = p.start[l];
    if (s0 > r || s1 <= r || s0 < 0) {
      if (threadIdx.x == 0) atomicCAS(c.status, 0, kStatusRange);
      zeros(r, r1);
      return;
    }
    if (at < 0 || long(at) + (p.seg[l + 1] - s0) > cap || p.seg[l + 1] > end) {
      if (threadIdx.x == 0) atomicCAS(c.status, 0, kStatusRange);
      zeros(r, min(s1, r1));
      r = s1;
      continue;
    }
    const long lh = long(l) * c.H + h;
    while (r < s1 && r < r1) {
      const int e0 = at + (r - s0), t0 = e0 & (kBlock - 1), m = min(kBlock - t0, s1 - r), b = e0 / kBlock;
      if (r == s0 || t0 == 0) {
        const uint4* in = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(c.codes[kv]) + (lh * c.nb + b) * (long(c.U) * 512));
        const float scale = c.scale[kv][lh * c.nb + b];
        __syncthreads();
        for (int i = threadIdx.x; i < c.U * 32; i += blockDim.x) {
          const uint4 w4 = in[i];
          const unsigned word[4] = {w4.x, w4.y, w4.z, w4.w};
          const int u = i >> 5, g = (i >> 2) & 7, t = i & 3;
#pragma unroll
          for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int e = unit_entry(kv, g, t, 4 * w + q), d = 8 * u + unit_dim(kv, g, t, 4 * w + q);
              const unsigned byte = (word[w] >> (8 * q)) & 0xffu;
              float x;
              if constexpr (CODE == 0) x = float(int8_t(byte));
              else x = __half2float(__half(__nv_cvt_fp8_to_halfraw(__nv_fp8_storage_t(byte), __NV_E4M3)));
              if (d < D) tile[e * pitch + d] = __fmul_rn(x, scale);
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < m * nv; i += blockDim.x) {
          const int e = i / nv, j = (i - e * nv) * VEC;
          Vec<T, VEC> v;
#pragma unroll
          for (int q = 0; q < VEC; ++q) v.x[q] = from_f<T>(tile[(t0 + e) * pitch + j + q]);
          *reinterpret_cast<Vec<T, VEC>*>(dst + long(r + e) * rs + j) = v;
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
// What bounds it: one query reads 2 bytes of cache for 4 flops, so HBM does; the tensor pipe is used because a column
// tile of 8 costs no more than one query, and because the conversion (1.25 instructions a code) is then the largest
// part of a warp's work.
//
// Precision. q is scaled per column by a power of two into [1, 2) and rounded to fp16 (exact for bf16 and fp16
// queries); probabilities are multiplied by 2^14 before their rounding to fp16, so that weights down to 2^-28 keep 11
// bits, and the sum of the softmax adds the rounded weights. With SPLIT (fp32 queries) both are
// split into two fp16 numbers, which keeps 22 bits.
//
// Division of work. All blocks of all (list, head, column tile) tasks form one line that is cut into equal pieces, one
// for each warp of the grid: no tail, whatever the lengths, and no host knowledge of them. A warp that owns a whole
// task writes its output; pieces of a task that is cut go to a workspace and `attn_join` adds them in order, so results
// do not depend on the schedule.
constexpr float kShift = 14.f;       // log2 of the factor on the probabilities
constexpr int kWarps = 4;
constexpr int kMaxLists = 4096;      // lists in one launch (their prefix sums stay in shared memory)

struct Attn {
  nb_kv8_cache c;
  nb_kv8_attn a;
  float* ws;
  long* cum;
  int workers, min_blocks;
};

__device__ __forceinline__ uint4 ld_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void mma(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned transpose8x8(unsigned x) {
  unsigned y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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

// Four codes -> two half2 (bytes 0, 1 and bytes 2, 3). int8: the byte with its sign bit flipped is 128 + x; in the low
// bits of an fp16 with the exponent of 1024 it reads 1152 + x, and the subtraction is exact. e4m3 is a subset of fp16.
template <int CODE>
__device__ __forceinline__ void widen(unsigned w, unsigned& lo, unsigned& hi) {
  if constexpr (CODE == 0) {
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

__device__ __forceinline__ float load_any(const void* base, long i, int type) {
  if (type == 2) return reinterpret_cast<const float*>(base)[i];
  if (type == 1) return __half2float(reinterpret_cast<const __half*>(base)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[i]);
}
__device__ __forceinline__ void store_any(void* base, long i, int type, float x) {
  if (type == 2) reinterpret_cast<float*>(base)[i] = x;
  else if (type == 1) reinterpret_cast<__half*>(base)[i] = __float2half_rn(x);
  else reinterpret_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(x);
}

// What a list brings to a launch: rows n from s0 on, entries len, blocks nb, column tiles.
struct ListWork { int s0, n, len, nb, tiles; };
__device__ __forceinline__ ListWork list_work(const Attn& k, int l, int columns) {
  ListWork w;
  w.s0 = k.a.seg[l];
  const int s1 = k.a.seg[l + 1], cap = k.c.nb * kBlock, len = k.a.len[l];
  w.n = w.s0 >= 0 && s1 <= min(k.a.rows, k.a.seg[k.c.L]) ? max(0, s1 - w.s0) : 0;
  w.len = min(max(len, 0), cap);
  w.nb = max(1, (w.len + kBlock - 1) / kBlock);
  w.tiles = (w.n * k.a.group + columns - 1) / columns;
  return w;
}

__device__ __forceinline__ int pieces(long total, int workers, int min_blocks) {
  return int(max(1l, min(long(workers), (total + min_blocks - 1) / min_blocks)));
}

template <int UMAX, int NT, int CODE, bool SPLIT>
__global__ void __launch_bounds__(kWarps * 32) attn_kernel(const Attn k) {
  constexpr int PAIRS = (UMAX + 1) / 2, COLS = 8 * NT, SP = SPLIT ? 2 : 1;
  extern __shared__ long cum[];                 // [L + 1] blocks of all tasks before list l
  __shared__ long part[kWarps];
  const int L = k.c.L, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int U = k.c.U, D = k.c.D;

  // ---- prefix sums of the lists' work
  for (int l = threadIdx.x; l < L; l += blockDim.x) {
    const ListWork w = list_work(k, l, COLS);
    cum[l + 1] = w.n ? k.c.H * w.tiles * w.nb : 0;
    if (blockIdx.x == 0 && (k.a.len[l] > k.c.nb * kBlock || k.a.seg[l + 1] > min(k.a.rows, k.a.seg[L]) || k.a.seg[l] < 0 || k.a.seg[l + 1] < k.a.seg[l]))
      atomicCAS(k.c.status, 0, kStatusRange);
  }
  __syncthreads();
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
  if (blockIdx.x == 0)
    for (int l = threadIdx.x; l <= L; l += blockDim.x) k.cum[l] = cum[l];
  const long total = cum[L];
  if (total == 0) return;
  const int P = pieces(total, k.workers, k.min_blocks);
  const int worker = warp * gridDim.x + blockIdx.x;
  if (worker >= P) return;
  long pos = worker * total / P;
  const long pos_end = (worker + 1) * total / P;

  while (pos < pos_end) {
    // ---- which task
    int lo = 0, hi = L;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cum[mid] <= pos) lo = mid; else hi = mid;
    }
    const int l = lo;
    const ListWork w = list_work(k, l, COLS);
    const int in_list = int(pos - cum[l]), task = in_list / w.nb, b0 = in_list - task * w.nb;
    const int h = task / w.tiles, tile = task - h * w.tiles;
    const int b1 = int(min(long(w.nb), b0 + (pos_end - pos)));
    pos += b1 - b0;
    const long lh = long(l) * k.c.H + h;
    const uint4* kp = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(k.c.codes[0]) + lh * k.c.nb * (long(U) * 512)) + lane;
    const uint4* vp = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(k.c.codes[1]) + lh * k.c.nb * (long(U) * 512)) + lane;
    const float* ksp = k.c.scale[0] + lh * k.c.nb;
    const float* vsp = k.c.scale[1] + lh * k.c.nb;

    uint4 kr[UMAX];
#pragma unroll
    for (int u = 0; u < UMAX; ++u) kr[u] = u < U ? ld_stream(kp + (long(b0) * U + u) * 32) : make_uint4(0, 0, 0, 0);
    float k_scale = ksp[b0], v_scale = vsp[b0];

    // ---- queries: column g of each tile as the B operand, scaled into [1, 2)
    unsigned qb[NT][PAIRS][2][SP];
    float qf[NT][2];
    int see[NT][2], seen_least = 0x7fffffff;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int col = tile * COLS + nt * 8 + g, a = col / k.a.group;
      const bool valid = a < w.n;
      const long qi = valid ? long(w.s0 + a) * k.a.q_row + long(h * k.a.group + col - a * k.a.group) * k.a.q_head : 0;
      float x[PAIRS][4], top = 0.f;
#pragma unroll
      for (int j = 0; j < PAIRS; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = 16 * j + (i >> 1) * 8 + 2 * t + (i & 1);
          x[j][i] = valid && d < D ? load_any(k.a.q, qi + d, k.a.q_type) : 0.f;
          top = fmaxf(top, fabsf(x[j][i]));
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const unsigned ex = min(max(__float_as_uint(top) >> 23, 1u), 253u);       // biased exponent
      const float down = __uint_as_float((254u - ex) << 23), up = __uint_as_float(ex << 23);
#pragma unroll
      for (int j = 0; j < PAIRS; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float a0 = x[j][2 * i] * down, a1 = x[j][2 * i + 1] * down;
          qb[nt][j][i][0] = pack(a0, a1);
          if constexpr (SPLIT) {
            const float2 r = unpack(qb[nt][j][i][0]);
            qb[nt][j][i][SP - 1] = pack(a0 - r.x, a1 - r.y);
          }
        }
      // the score fragment holds columns 2t and 2t + 1
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        qf[nt][i] = __shfl_sync(0xffffffffu, up, (2 * t + i) * 4) * k.a.scale_log2;
        const int c = tile * COLS + nt * 8 + 2 * t + i, row = c / k.a.group;
        see[nt][i] = row < w.n ? max(0, w.len - (w.n - 1 - row)) : 0;
        if (row < w.n) seen_least = min(seen_least, see[nt][i]);
      }
    }
    seen_least = __reduce_min_sync(0xffffffffu, seen_least);

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
      uint4 vr[UMAX];
#pragma unroll
      for (int u = 0; u < UMAX; ++u) vr[u] = u < U ? ld_stream(vp + (long(b) * U + u) * 32) : make_uint4(0, 0, 0, 0);
      // ---- scores of 64 entries
      float s[NT][4][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[nt][m][i] = 0.f;
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        const unsigned x[4] = {kr[2 * j].x, kr[2 * j].y, kr[2 * j].z, kr[2 * j].w};
        unsigned y[4] = {0, 0, 0, 0};
        if (2 * j + 1 < UMAX) {
          const uint4 z = kr[2 * j + 1 < UMAX ? 2 * j + 1 : 0];
          y[0] = z.x; y[1] = z.y; y[2] = z.z; y[3] = z.w;
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          unsigned a0, a1, a2 = 0, a3 = 0;
          widen<CODE>(x[m], a0, a1);
          if (2 * j + 1 < UMAX) widen<CODE>(y[m], a2, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < SP; ++q) mma(s[nt][m], a0, a1, a2, a3, qb[nt][j][0][q], qb[nt][j][1][q]);
        }
      }
      const float ks_now = k_scale, vs_now = v_scale;
      if (b + 1 < b1) {
#pragma unroll
        for (int u = 0; u < UMAX; ++u) kr[u] = u < U ? ld_stream(kp + (long(b + 1) * U + u) * 32) : make_uint4(0, 0, 0, 0);
        k_scale = ksp[b + 1];
        v_scale = vsp[b + 1];
      }
      // ---- softmax; columns whose view ends inside (or before) this block take the masked form
      const bool masked = (b + 1) * kBlock > seen_least;
      unsigned pb[NT][4][2][SP];
      float keep[NT][2], vs_col[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (masked) {
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (b * kBlock + 16 * m + (i >> 1) * 8 + g >= see[nt][i & 1]) s[nt][m][i] = -INFINITY;
        }
        float off[2], f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          f[i] = qf[nt][i] * ks_now;
          float top = fmaxf(fmaxf(fmaxf(s[nt][0][i], s[nt][0][2 + i]), fmaxf(s[nt][1][i], s[nt][1][2 + i])),
                            fmaxf(fmaxf(s[nt][2][i], s[nt][2][2 + i]), fmaxf(s[nt][3][i], s[nt][3][2 + i])));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          const float now = fmaxf(mx[nt][i], top * f[i]);
          keep[nt][i] = now == mx[nt][i] ? 1.f : ex2(mx[nt][i] - now);
          off[i] = kShift - now;
          mx[nt][i] = now;
          vs_col[nt][i] = !masked || b * kBlock < see[nt][i] ? vs_now : 0.f;
        }
        float add[2] = {0.f, 0.f};
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          float p[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[i] = ex2(fmaf(s[nt][m][i], f[i & 1], off[i & 1]));
            if (masked && s[nt][m][i] == -INFINITY && b * kBlock + 16 * m + (i >> 1) * 8 + g >= see[nt][i & 1]) p[i] = 0.f;
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const unsigned hi = pack(p[2 * i], p[2 * i + 1]);
            const float2 r = unpack(hi);
            pb[nt][m][i][0] = transpose8x8(hi);
            if constexpr (SPLIT) {
              pb[nt][m][i][SP - 1] = transpose8x8(pack(p[2 * i] - r.x, p[2 * i + 1] - r.y));
              add[0] += p[2 * i];
              add[1] += p[2 * i + 1];
            } else {
              add[0] += r.x;
              add[1] += r.y;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) sm[nt][i] = sm[nt][i] * keep[nt][i] + add[i];
      }
      if (CODE != 0 && (b + 1) * kBlock > w.len) {      // entries that the list does not hold may be any bytes, NaN codes too
#pragma unroll
        for (int u = 0; u < UMAX; ++u) {
          unsigned* words = reinterpret_cast<unsigned*>(&vr[u]);
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            unsigned keep_bytes = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (b * kBlock + 16 * m + (q >> 1) * 8 + 2 * t + (q & 1) < w.len) keep_bytes |= 0xffu << (8 * q);
            words[m] &= keep_bytes;
          }
        }
      }
      // ---- output of these entries
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        float acc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[nt][i] = 0.f;
        const unsigned x[4] = {vr[2 * j].x, vr[2 * j].y, vr[2 * j].z, vr[2 * j].w};
        unsigned y[4] = {0, 0, 0, 0};
        if (2 * j + 1 < UMAX) {
          const uint4 z = vr[2 * j + 1 < UMAX ? 2 * j + 1 : 0];
          y[0] = z.x; y[1] = z.y; y[2] = z.z; y[3] = z.w;
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          unsigned a0, a1 = 0, a2, a3 = 0;
          widen<CODE>(x[m], a0, a2);
          if (2 * j + 1 < UMAX) widen<CODE>(y[m], a1, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < SP; ++q) mma(acc[nt], a0, a1, a2, a3, pb[nt][m][0][q], pb[nt][m][1][q]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[j][nt][i] = fmaf(o[j][nt][i], keep[nt][i & 1], acc[nt][i] * vs_col[nt][i & 1]);
      }
    }

    // ---- the piece's result
    const bool whole = b0 == 0 && b1 == w.nb;
    float* slot = k.ws + long(2 * worker + (b0 == 0 ? 1 : 0)) * COLS * (8 * U + 2);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float z = sm[nt][i];
        z += __shfl_xor_sync(0xffffffffu, z, 4);
        z += __shfl_xor_sync(0xffffffffu, z, 8);
        z += __shfl_xor_sync(0xffffffffu, z, 16);
        const int in_tile = nt * 8 + 2 * t + i, c = tile * COLS + in_tile, row = c / k.a.group;
        if (row >= w.n) continue;
        if (whole) {
          const float inv = z == 0.f ? 0.f : 1.f / z;
          const long at = long(w.s0 + row) * k.a.o_row + long(h * k.a.group + c - row * k.a.group) * k.a.o_head;
#pragma unroll
          for (int j = 0; j < PAIRS; ++j)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int d = 16 * j + 8 * q + g;
              if (d < D) store_any(k.a.out, at + d, k.a.q_type, o[j][nt][2 * q + i] * inv);
            }
        } else {
          float* to = slot + in_tile * (8 * U + 2);
#pragma unroll
          for (int j = 0; j < PAIRS; ++j)
#pragma unroll
            for (int q = 0; q < 2; ++q)
              if (16 * j + 8 * q + g < 8 * U) to[16 * j + 8 * q + g] = o[j][nt][2 * q + i];
          if (g == 0) {
            to[8 * U] = mx[nt][i];
            to[8 * U + 1] = z;
          }
        }
      }
  }
}

// One CTA for each (row, query head): adds the pieces of its task in their order. Rows whose task was one piece are
// done already. Rows behind the last list become zeros when `zero_tail` is set.
__global__ void __launch_bounds__(kWarps * 32) attn_join(const Attn k, int cols) {
  const int row = blockIdx.x, head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int L = k.c.L, D = k.c.D, width = 8 * k.c.U + 2;
  if (row < k.a.seg[0]) return;
  const long at = long(row) * k.a.o_row + long(head) * k.a.o_head;
  if (row >= k.a.seg[L]) {
    if (k.a.zero_tail)
      for (int d = threadIdx.x; d < D; d += blockDim.x) store_any(k.a.out, at + d, k.a.q_type, 0.f);
    return;
  }
  const int l = find_list(k.a.seg, L, row);
  const ListWork w = list_work(k, l, cols);
  if (row < w.s0 || row >= w.s0 + w.n) {      // bounds that the main kernel refused
    for (int d = threadIdx.x; d < D; d += blockDim.x) store_any(k.a.out, at + d, k.a.q_type, 0.f);
    return;
  }
  const long total = k.cum[L];
  const int P = pieces(total, k.workers, k.min_blocks);
  const int h = head / k.a.group, col = (row - w.s0) * k.a.group + head - h * k.a.group;
  const long begin = k.cum[l] + (h * w.tiles + col / cols) * w.nb;
  const int w0 = int(((begin + 1) * P - 1) / total), w1 = int(((begin + w.nb) * P - 1) / total);
  if (w0 == w1) return;
  auto piece = [&](int i) { return k.ws + (long(2 * (w0 + i) + (i == 0 ? 1 : 0)) * cols + col % cols) * width; };
  const int n = w1 - w0 + 1;
  __shared__ float red[kWarps], sums[kWarps], acc_s[kWarps][128];
  float top = -INFINITY;
  for (int i = threadIdx.x; i < n; i += blockDim.x) top = fmaxf(top, piece(i)[8 * k.c.U]);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
  if (lane == 0) red[warp] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) top = fmaxf(top, red[i]);
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll 4
  for (int i = warp; i < n; i += kWarps) {
    const float* from = piece(i);
    const float m = from[8 * k.c.U], f = m == top ? 1.f : ex2(m - top);
    sum += f * from[8 * k.c.U + 1];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (lane + 32 * q < D) acc[q] += f * from[lane + 32 * q];
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) acc_s[warp][lane + 32 * q] = acc[q];
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  float z = 0.f;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) z += sums[i];
  const float inv = z == 0.f ? 0.f : 1.f / z;
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) x += acc_s[i][d];
    store_any(k.a.out, at + d, k.a.q_type, x * inv);
  }
}

// ------------------------------------------------------------------------------------------------------ launches
using AttnFn = void (*)(const Attn);

template <int UMAX, int NT>
AttnFn pick_code(int code, bool split) {
  if (code == 0) return split ? attn_kernel<UMAX, NT, 0, true> : attn_kernel<UMAX, NT, 0, false>;
  return split ? attn_kernel<UMAX, NT, 1, true> : attn_kernel<UMAX, NT, 1, false>;
}

// Column tiles of 8: one for single tokens, more when several rows or shared heads bring more columns (a converted
// block then serves them all); wide heads take at most two because their accumulators fill the registers.
int tiles_for(int U, int columns) { return columns <= 8 ? 1 : (U <= 8 && columns > 16 ? 4 : 2); }

AttnFn pick(int U, int nt, int code, bool split) {
  if (U <= 5) return nt == 1 ? pick_code<5, 1>(code, split) : nt == 2 ? pick_code<5, 2>(code, split) : pick_code<5, 4>(code, split);
  if (U <= 8) return nt == 1 ? pick_code<8, 1>(code, split) : nt == 2 ? pick_code<8, 2>(code, split) : pick_code<8, 4>(code, split);
  if (U <= 10) return nt == 1 ? pick_code<10, 1>(code, split) : pick_code<10, 2>(code, split);
  return nt == 1 ? pick_code<16, 1>(code, split) : pick_code<16, 2>(code, split);
}

int multiprocessors() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

constexpr int kMaxCtas = 12;      // CTAs of attn_kernel on one SM that the workspace is sized for

long slot_floats(int U, int cols) { return long(cols) * (8 * U + 2); }


// The widest vector (at most 16 bytes) that divides the head and that every row start is aligned to.
int vector_of(int D, int size, const long* strides, int n_strides, const void* const* ptrs, int n_ptrs) {
  for (int v = 16 / size; v > 1; v >>= 1) {
    bool ok = D % v == 0;
    for (int i = 0; i < n_strides; ++i) ok = ok && strides[i] % v == 0;
    for (int i = 0; i < n_ptrs; ++i) ok = ok && (reinterpret_cast<uintptr_t>(ptrs[i]) % (v * size)) == 0;
    if (ok) return v;
  }
  return 1;
}

// f(type tag, vector tag, code tag) for the run-time triple
template <typename F>
void with_types(int type, int vec, int code, F f) {
  auto by_code = [&](auto t, auto v) {
    if (code == 0) f(t, v, std::integral_constant<int, 0>{});
    else f(t, v, std::integral_constant<int, 1>{});
  };
  auto by_vec = [&](auto t) {
    if (vec == 8 && sizeof(t) == 2) by_code(t, std::integral_constant<int, 8>{});
    else if (vec == 4) by_code(t, std::integral_constant<int, 4>{});
    else if (vec == 2) by_code(t, std::integral_constant<int, 2>{});
    else by_code(t, std::integral_constant<int, 1>{});
  };
  if (type == 0) by_vec(__nv_bfloat16{});
  else if (type == 1) by_vec(__half{});
  else by_vec(float{});
}

bool bad_cache(const nb_kv8_cache* c) {
  return c->D < 1 || c->D > 128 || c->U != (c->D + 7) / 8 || c->H < 1 || c->H > 65535 || c->L < 1 || c->nb < 1 || !c->status || c->code < 0 || c->code > 1;
}

}  // namespace nbk

extern "C" {

int nb_kv8_append(const nb_kv8_cache* c, const nb_kv8_rows* p, cudaStream_t st) {
  using namespace nbk;
  if (bad_cache(c) || p->rows < 0) return -1;
  if (p->rows == 0) return 0;
  const int size = c->type == 2 ? 4 : 2;
  const long strides[4] = {p->row_stride[0], p->row_stride[1], p->head_stride[0], p->head_stride[1]};
  const void* ptrs[4] = {p->src[0], p->src[1], c->open[0], c->open[1]};
  const int vec = vector_of(c->D, size, strides, 4, ptrs, 4);
  const int chunk = p->max_rows <= 8 ? 1 : kBlock;
  const dim3 grid((p->rows + chunk - 1) / chunk, c->H, 2);
  const size_t smem = kBlock * (c->D | 1) * sizeof(float);
  with_types(c->type, vec, c->code, [&](auto t, auto v, auto k) {
    append_kernel<decltype(t), decltype(v)::value, decltype(k)::value><<<grid, 128, smem, st>>>(*c, *p, chunk);
  });
  return int(cudaGetLastError());
}

int nb_kv8_truncate(const nb_kv8_cache* c, const int* len, cudaStream_t st) {
  using namespace nbk;
  if (bad_cache(c)) return -1;
  const long stride = 0;
  const void* ptrs[2] = {c->open[0], c->open[1]};
  const int vec = vector_of(c->D, c->type == 2 ? 4 : 2, &stride, 1, ptrs, 2);
  const size_t smem = kBlock * (c->D | 1) * sizeof(float);
  with_types(c->type, vec, c->code, [&](auto t, auto v, auto k) {
    truncate_kernel<decltype(t), decltype(v)::value, decltype(k)::value><<<dim3(c->L, c->H, 2), 128, smem, st>>>(*c, len);
  });
  return int(cudaGetLastError());
}

int nb_kv8_read(const nb_kv8_cache* c, const nb_kv8_rows* p, int type, cudaStream_t st) {
  using namespace nbk;
  if (bad_cache(c) || p->rows < 0) return -1;
  if (p->rows == 0) return 0;
  const long stride = 0;
  const void* ptrs[2] = {p->dst[0], p->dst[1]};
  const int vec = vector_of(c->D, type == 2 ? 4 : 2, &stride, 1, ptrs, 2);
  const int chunk = p->max_rows <= 8 ? 1 : kBlock;
  const dim3 grid((p->rows + chunk - 1) / chunk, c->H, 2);
  const size_t smem = kBlock * (c->D | 1) * sizeof(float);
  with_types(type, vec, c->code, [&](auto t, auto v, auto k) {
    read_kernel<decltype(t), decltype(v)::value, decltype(k)::value><<<grid, 128, smem, st>>>(*c, *p, chunk);
  });
  return int(cudaGetLastError());
}

// Bytes of workspace that an attention call over heads of D dims takes for `columns` query columns a list and head.
long nb_kv8_attention_workspace(int D, int columns) {
  using namespace nbk;
  const int U = (D + 7) / 8, nt = tiles_for(U, columns);
  return long(multiprocessors()) * kMaxCtas * kWarps * 2 * slot_floats(U, 8 * nt) * 4 + (kMaxLists + 2) * 8;
}

int nb_kv8_attention(const nb_kv8_cache* c, const nb_kv8_attn* a, void* ws, long ws_bytes, cudaStream_t st) {
  using namespace nbk;
  if (bad_cache(c) || a->rows < 0 || a->group < 1 || long(c->H) * a->group > 65535) return -1;
  // (a list's tasks are counted in 32 bits)
  if (long(c->H) * ((long(a->rows) * a->group + 7) / 8) * c->nb > 0x7fffffffl) return -3;
  if (a->rows == 0) return 0;
  const int sms = multiprocessors();
  const long columns = long(a->max_rows) * a->group;
  const int nt = tiles_for(c->U, columns > 1024 ? 1024 : int(columns)), cols = 8 * nt;
  AttnFn fn = pick(c->U, nt, c->code, a->q_type == 2);
  const int L_smem = c->L < kMaxLists ? c->L : kMaxLists;
  int occ = 1;
  cudaError_t rc = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, fn, kWarps * 32, (L_smem + 1) * sizeof(long));
  if (rc != cudaSuccess) return int(rc);
  occ = occ < 1 ? 1 : (occ > kMaxCtas ? kMaxCtas : occ);
  Attn k;
  k.cum = reinterpret_cast<long*>(ws);
  k.ws = reinterpret_cast<float*>(k.cum + kMaxLists + 2);
  k.min_blocks = 1;
  k.workers = sms * occ * kWarps;
  if (long(k.workers) * 2 * slot_floats(c->U, cols) * 4 + (kMaxLists + 2) * 8 > ws_bytes) return -2;
  for (int l0 = 0; l0 < c->L; l0 += kMaxLists) {      // (more lists than one launch holds: slices, in stream order)
    k.c = *c;
    k.a = *a;
    k.c.L = c->L - l0 < kMaxLists ? c->L - l0 : kMaxLists;
    const long lh = long(l0) * c->H * c->nb;
    for (int i = 0; i < 2; ++i) {
      k.c.codes[i] = reinterpret_cast<uint8_t*>(c->codes[i]) + lh * c->U * 512;
      k.c.scale[i] = c->scale[i] + lh;
    }
    k.a.seg += l0;
    k.a.len += l0;
    const bool last = l0 + k.c.L >= c->L;
    k.a.zero_tail = a->zero_tail && last;
    fn<<<sms * occ, kWarps * 32, (k.c.L + 1) * sizeof(long), st>>>(k);
    attn_join<<<dim3(a->rows, c->H * a->group), kWarps * 32, 0, st>>>(k, cols);
    rc = cudaGetLastError();
    if (rc != cudaSuccess) return int(rc);
  }
  return 0;
}

}  // extern "C"
