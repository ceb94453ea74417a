// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Sequence b has `len` drafted tokens x_0 .. x_{len-1}, drawn from the rows q_i of the draft model (or, without q, each
// the draft's certain choice). Token i is accepted while u_i q_i(x_i) < p_i(x_i); with a accepted tokens the next token
// is drawn from r = max(p_a - q_a, 0) after a refusal (p_a without x_a where there is no q; p_a itself where r is
// empty) and from r = p_len otherwise: the lowest j with r_0 + .. + r_j > w (r_0 + .. + r_{V-1}). Accepted and drawn
// tokens together are distributed as draws from p alone.
//
// Sums are in 64 bits: the running sum has as many steps as the vocabulary has tokens, and a sum in 32 bits would move
// one draw in some fifty across a step. Values below 2^-126 count as zero.
//
// What bounds it: one or two rows of the vocabulary for each sequence, read once from HBM (some KB are read again to find
// the token). A row is cut into spans of 512 entries or more, one warp sums a span, and a cluster of up to 8 CTAs shares a
// row and exchanges the spans' sums through distributed shared memory: one launch, no workspace, a fixed order of additions.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "verify.h"

namespace nbv {
namespace cg = cooperative_groups;

constexpr int kMaxCluster = 8;
constexpr int kMaxSpans = 1024;      // spans of a row: their sums (8 KB) stand in every CTA's shared memory

__device__ __forceinline__ float val(const float* p, long i) { return __ldg(p + i); }
__device__ __forceinline__ float val(const __half* p, long i) { return __half2float(p[i]); }
__device__ __forceinline__ float val(const __nv_bfloat16* p, long i) { return __bfloat162float(p[i]); }

// What vocabulary entry j weighs in the draw. MODE 0: p. 1: max(p - q, 0). 2: p without entry `skip`.
// Weights of the N rows of 32 entries from j0 on, entry j0 + 32 i + lane in w[i]; nothing behind b. Every load is made
// (behind b of the last entry), so that all of them are in flight at once.
template <typename T, int MODE, int N>
__device__ __forceinline__ void load_weights(float (&w)[N], const T* p, const T* q, long skip, int j0, int b) {
  const int lane = threadIdx.x & 31;
  float x[N], y[N];
  const bool whole = j0 + 32 * N <= b;
  if (whole) {
    p += j0 + lane;
    if constexpr (MODE == 1) q += j0 + lane;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i] = val(p, 32 * i);
      if constexpr (MODE == 1) y[i] = val(q, 32 * i);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int j = min(j0 + 32 * i + lane, b - 1);
      x[i] = val(p, j);
      if constexpr (MODE == 1) y[i] = val(q, j);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (MODE == 1) {
      y[i] = fmaxf(y[i], 0.f);      // (a NaN counts as zero)
      w[i] = x[i] > y[i] ? __fsub_rn(x[i], y[i]) : 0.f;
    } else w[i] = x[i] > 0.f && !(MODE == 2 && j0 + 32 * i + lane == skip) ? x[i] : 0.f;
  }
  if (!whole)
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (j0 + 32 * i + lane >= b) w[i] = 0.f;
}

// Sum of entries [a, b), a < b, lane by lane with stride 32.
template <typename T, int MODE>
__device__ __forceinline__ double span_sum(const T* p, const T* q, long skip, int a, int b) {
  double s0 = 0., s1 = 0.;
  for (int j = a; j < b; j += 512) {
    float w[16];
    load_weights<T, MODE>(w, p, q, skip, j, b);
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      s0 += double(w[i]);
      s1 += double(w[i + 1]);
    }
  }
  s0 += s1;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s0 += __shfl_xor_sync(0xffffffffu, s0, d);
  return s0;
}

// The first entry of [a, b) at which `before` plus the running sum passes `goal`; the last one that weighs anything
// where rounding leaves none. Eight rows of 32 entries at a time: their loads and their scans overlap.
template <typename T, int MODE>
__device__ __forceinline__ int find_entry(const T* p, const T* q, long skip, int a, int b, double before, double goal) {
  const int lane = threadIdx.x & 31;
  int last = -1;
  for (int j0 = a; j0 < b; j0 += 256) {
    float w[8];
    double s[8];
    load_weights<T, MODE>(w, p, q, skip, j0, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = w[i];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double up = __shfl_up_sync(0xffffffffu, s[i], d);
        if (lane >= d) s[i] += up;
      }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned has = __ballot_sync(0xffffffffu, w[i] > 0.f);
      const unsigned hit = __ballot_sync(0xffffffffu, w[i] > 0.f && before + s[i] > goal);
      if (hit) return j0 + 32 * i + __ffs(hit) - 1;
      if (has) last = j0 + 32 * i + 31 - __clz(has);
      before += __shfl_sync(0xffffffffu, s[i], 31);
    }
  }
  return last;
}

// Draws from the row; returns false if nothing weighs anything. All CTAs of the cluster call it together. Span i belongs
// to warp i % (warps of the cluster); a CTA keeps the sums of its spans at their places in `all` and copies the others'.
template <typename T, int MODE, int THREADS>
__device__ __forceinline__ bool draw(const nb_verify_args& a, int span, const T* p, const T* q, long skip, float w, int b, double* all) {
  constexpr int kThreads = THREADS, kWarps = THREADS / 32;
  cg::cluster_group cluster = cg::this_cluster();
  const int CL = cluster.num_blocks(), rank = cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, V = a.V;
  const int spans = (V + span - 1) / span, step = CL * kWarps;
  for (int i = rank * kWarps + warp; i < spans; i += step) {
    const double s = span_sum<T, MODE>(p, q, skip, i * span, min(V, (i + 1) * span));
    if (lane == 0) all[i] = s;
  }
  cluster.sync();
  for (int i = threadIdx.x; i < spans; i += kThreads) {
    const int owner = i % step / kWarps;
    if (owner != rank) all[i] = cluster.map_shared_rank(all, owner)[i];
  }
  __syncthreads();
  // running sums over the spans, the same in every warp: each lane over `per` consecutive ones
  const int per = (spans + 31) / 32, first = min(spans, lane * per), end = min(spans, first + per);
  double run = 0.;
  for (int i = first; i < end; ++i) run += all[i];
  double incl = run;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const double up = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += up;
  }
  const double goal = double(w) * __shfl_sync(0xffffffffu, incl, 31);
  // the first span whose running sum passes the goal; failing that the last one that weighs anything
  int hit = kMaxSpans, last = -1;
  double before = incl - run, ahead = 0.;
  for (int i = first; i < end; ++i) {
    const double s = all[i];
    if (s > 0.) {
      if (hit == kMaxSpans && before + s > goal) {
        hit = i;
        ahead = before;
      }
      last = i;
      if (hit == kMaxSpans) ahead = before;
    }
    before += s;
  }
  const int hit_all = __reduce_min_sync(0xffffffffu, hit), last_all = __reduce_max_sync(0xffffffffu, last);
  const int at = hit_all < kMaxSpans ? hit_all : last_all;
  if (at < 0) {
    cluster.sync();      // (the sums are written again by the next draw)
    return false;
  }
  if (at % step == rank * kWarps + warp) {
    ahead = __shfl_sync(0xffffffffu, ahead, at / per);
    const int j = find_entry<T, MODE>(p, q, skip, at * span, min(V, (at + 1) * span), ahead, goal);
    if (lane == 0) a.token[b] = j;
  }
  cluster.sync();        // no CTA leaves while another may read its sums
  return true;
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) verify_kernel(const nb_verify_args a, int span) {
  __shared__ double all[kMaxSpans];
  cg::cluster_group cluster = cg::this_cluster();
  const int b = blockIdx.x / cluster.num_blocks(), lane = threadIdx.x & 31;
  const T* P = reinterpret_cast<const T*>(a.p) + long(b) * a.p_batch;
  const T* Q = a.q ? reinterpret_cast<const T*>(a.q) + long(b) * a.q_batch : nullptr;
  const int len = a.len ? min(max(a.len[b], 0), a.n) : a.n;
  auto token = [&](int i) {
    return a.tokens_64 ? reinterpret_cast<const long long*>(a.tokens)[long(b) * a.n + i] : (long long)(reinterpret_cast<const int*>(a.tokens)[long(b) * a.n + i]);
  };
  // ---- the accepted prefix (every warp for itself; tokens behind `len` are loaded beside it and not looked at)
  int accepted = len;
  for (int i0 = 0; i0 < a.n && i0 < len; i0 += 32) {
    const int i = i0 + lane, at = min(i, a.n - 1);
    const long long x = token(at);
    const float u = a.u[long(b) * a.n + at];
    const bool known = x >= 0 && x < a.V;
    const float px = known ? fmaxf(val(P + at * a.p_row, x), 0.f) : 0.f;      // (a NaN counts as zero)
    const float qx = !Q ? 1.f : (known ? fmaxf(val(Q + at * a.q_row, x), 0.f) : 0.f);
    const bool ok = i >= len || __fmul_rn(u, qx) < px;
    const unsigned refused = ~__ballot_sync(0xffffffffu, ok);
    if (refused) {
      accepted = i0 + __ffs(refused) - 1;
      break;
    }
  }
  // ---- the next token
  const T* p = P + accepted * a.p_row;
  const float w = a.w[b];
  bool done;
  if (accepted == len) done = draw<T, 0, THREADS>(a, span, p, nullptr, -1, w, b, all);
  else {
    done = Q ? draw<T, 1, THREADS>(a, span, p, Q + accepted * a.q_row, -1, w, b, all) : draw<T, 2, THREADS>(a, span, p, nullptr, token(accepted), w, b, all);
    if (!done) done = draw<T, 0, THREADS>(a, span, p, nullptr, -1, w, b, all);
  }
  if (cluster.block_rank() == 0 && threadIdx.x == 0) {
    a.accepted[b] = accepted;
    if (!done) a.token[b] = -1;
  }
}

}  // namespace nbv

extern "C" int nb_verify_draft(const nb_verify_args* a, cudaStream_t st) {
  using namespace nbv;
  if (a->B < 0 || a->n < 0 || a->V < 1 || a->V > (1 << 30) || a->type < 0 || a->type > 2) return -1;
  if (a->B == 0) return 0;
  // Spans that keep the sums within their 8 KB, and no more CTAs a row than there are spans for half of their warps or than
  // fit the GPU at once: a second wave would wait for its first loads while the first one's end idles (256 rows of
  // 100263 in fp32, CTAs a row x warps: 36.4 us for 4 x 4, the whole of one wave; 40.3 for 8 x 4, 60.5 for 1 x 4). Many
  // rows take CTAs of 4 warps instead of 8, which spread evenly (1024 rows of 50257: 54.0 us for 1 x 4, 57.1 for 1 x 8);
  // few rows take 8 (64 rows of 100263: 11.9 us against 12.5).
  int span = 512;
  while ((a->V + span - 1) / span > kMaxSpans) span *= 2;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int threads = long(a->B) * kMaxCluster > 4l * sms ? 128 : 256, warps = threads / 32;
  int cl = 1;
  while (cl < kMaxCluster && long(cl) * warps * span < 2l * a->V && long(a->B) * cl * 2 <= long(1024 / threads) * sms) cl *= 2;
  if (long(a->B) * cl > 0x7fffffffl) return -1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a->B) * cl);
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cl;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  using Fn = void (*)(const nb_verify_args, int);
  const Fn fn = threads == 256 ? (a->type == 0 ? verify_kernel<__nv_bfloat16, 256> : a->type == 1 ? verify_kernel<__half, 256> : verify_kernel<float, 256>)
                               : (a->type == 0 ? verify_kernel<__nv_bfloat16, 128> : a->type == 1 ? verify_kernel<__half, 128> : verify_kernel<float, 128>);
  const cudaError_t rc = cudaLaunchKernelEx(&cfg, fn, *a, span);
  if (rc != cudaSuccess) return int(rc);
  return int(cudaGetLastError());
}
