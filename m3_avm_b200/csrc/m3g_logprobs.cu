// m3g_logprobs.cu -- log probabilities of given tokens, entropy and the most
// probable alternatives of each row of logits, in one pass over the row.
//
// Each thread keeps, in base 2, the running maximum m of its logits, z = sum
// 2^(t - m) and w = sum 2^(t - m) (t - m) with t = x log2(e); they join like
// the partial sums of a softmax:  lse = (m + log2 z) ln 2,  H = (log2 z -
// w / z) ln 2.
//
// The alternatives come out of the same pass.  The CTA's 32 half-warps keep
// running maxima, each of a different element, so the smallest of the 32 is a
// bound that at least 32 elements reach: an element below it is not among the
// best 32 (n_top <= 32).  Elements that reach the bound go to a list in shared
// memory; an element of a later round has a higher id than all of the earlier
// ones, so it must beat the earlier bound, not just reach it.  Of random
// logits about 110 / r of round r's 8192 elements pass.  At the end those that
// reach the last bound are ranked by counting.
//
// A row is read by a cluster of 1 .. 8 CTAs, whose sums and lists join through
// distributed shared memory: 8 while the rows do not fill the SMs.
#include <cmath>

#include <cooperative_groups.h>

#include "m3g_serve.cuh"

namespace cg = cooperative_groups;

namespace m3g {
namespace {

constexpr int kLpThreads = 512;
constexpr int kLpElems = 16;                        // logits per thread and round
constexpr int kLpRound = kLpThreads * kLpElems;
constexpr int kLpMost = 1024;                       // list entries that may wait for the end
constexpr int kLpList = kLpMost + kLpRound;         // a round may add every element
constexpr int kLpTop = 32;

struct LpArgs {
  const void* x;
  long long vocab, stride;
  const int32_t* tokens;
  float* logprob;
  float* entropy;
  int32_t* top_id;
  float* top_lp;
  int n_tokens, n_top;
  int chunk;  // logits per CTA of the cluster
};

struct LpSum {
  float m, z, w;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sums of two disjoint sets (-inf maximum: an empty one, or of probability 0).
__device__ __forceinline__ LpSum join(LpSum a, LpSum b) {
  LpSum r;
  r.m = fmaxf(a.m, b.m);
  const float ref = r.m == -INFINITY ? 0.f : r.m;
  const float da = fmaxf(a.m - ref, -300.f), db = fmaxf(b.m - ref, -300.f);
  const float fa = ex2(a.m - ref), fb = ex2(b.m - ref);
  r.z = fa * a.z + fb * b.z;
  r.w = fa * (a.w + da * a.z) + fb * (b.w + db * b.z);
  return r;
}

// Order of (logit, id) as an integer: larger is better; NaN below -inf, equal
// logits (0 and -0 among them) by the lower id.
__device__ __forceinline__ unsigned long long lp_key(float x, uint32_t id) {
  uint32_t b = __float_as_uint(x + 0.f);
  b = x != x ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return static_cast<unsigned long long>(b) << 32 | (0xFFFFFFFFu - id);
}

// The best min(k, n) of list[0 .. n) in order into best[0 ..]; all threads.
// Up to kLpThreads entries each thread counts what beats its own; longer
// lists (rows of equal logits) give up their best k times.
__device__ void lp_select(const unsigned long long* list, int n, int k, unsigned long long* best,
                          unsigned long long* red) {
  const int tid = threadIdx.x;
  if (n <= kLpThreads) {
    if (tid < n) {
      const unsigned long long mine = list[tid];
      int beaten = 0;
      for (int i = 0; i < n; ++i) beaten += list[i] > mine;
      if (beaten < k) best[beaten] = mine;
    }
    __syncthreads();
    return;
  }
  unsigned long long below = ~0ull;
  for (int r = 0; r < k; ++r) {
    unsigned long long b = 0;
    for (int i = tid; i < n; i += kLpThreads) {
      const unsigned long long e = list[i];
      if (e < below && e > b) b = e;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const unsigned long long e = __shfl_xor_sync(0xFFFFFFFFu, b, o);
      b = e > b ? e : b;
    }
    if ((tid & 31) == 0) red[tid >> 5] = b;
    __syncthreads();
    b = red[0];
#pragma unroll
    for (int i = 1; i < kLpThreads / 32; ++i) b = red[i] > b ? red[i] : b;
    if (tid == 0) best[r] = b;
    below = b;
    __syncthreads();
  }
}

template <class T, bool VEC, bool TOP>
__global__ void __launch_bounds__(kLpThreads) k_token_logprobs(const __grid_constant__ LpArgs a) {
  constexpr int VW = 16 / sizeof(T), NV = kLpElems / VW;
  constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
  extern __shared__ __align__(16) uint8_t smem[];
  unsigned long long* list = reinterpret_cast<unsigned long long*>(smem);  // [kLpList] when TOP
  __shared__ unsigned long long best[kLpTop], red[kLpThreads / 32];
  __shared__ float group_max[2][32];
  __shared__ LpSum sums[kLpThreads / 32];
  __shared__ LpSum total;
  __shared__ int count, kept;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), size = static_cast<int>(cluster.num_blocks());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long row = blockIdx.x / size;
  const T* x = static_cast<const T*>(a.x) + row * a.stride;
  const long long e0 = static_cast<long long>(rank) * a.chunk;
  const long long e1 = min(a.vocab, e0 + a.chunk);
  float given = 0.f;
  const bool asked = rank == 0 && tid < a.n_tokens;
  if (asked) {
    const long long id = a.tokens[row * a.n_tokens + tid];
    given = id >= 0 && id < a.vocab ? Act<T>::to(x[id]) : -INFINITY;
  }
  if (tid == 0) count = 0;
  if (TOP) __syncthreads();
  LpSum s{-INFINITY, 0.f, 0.f};
  float run = -INFINITY, bound = -INFINITY;
  int parity = 0;
  for (long long r0 = e0; r0 < e1; r0 += kLpRound, parity ^= 1) {
    float v[kLpElems];
    float most = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const long long i = r0 + (static_cast<long long>(j) * kLpThreads + tid) * VW;
      float (&w)[VW] = *reinterpret_cast<float(*)[VW]>(&v[j * VW]);
      if (VEC && i + VW <= e1) {
        load_act<T, VW, true>(x + i, w);
      } else {
#pragma unroll
        for (int k = 0; k < VW; ++k) w[k] = i + k < e1 ? Act<T>::to(x[i + k]) : -INFINITY;
      }
    }
#pragma unroll
    for (int k = 0; k < kLpElems; ++k) most = fmaxf(most, v[k]);
    const float t_most = most * kLog2e;
    if (t_most > s.m) {
      const float d = fmaxf(s.m - t_most, -300.f), f = ex2(s.m - t_most);
      s.w = f * (s.w + d * s.z);
      s.z = f * s.z;
      s.m = t_most;
    }
    const float ref = s.m == -INFINITY ? 0.f : s.m;
#pragma unroll
    for (int k = 0; k < kLpElems; ++k) {
      const float t = fmaf(v[k], kLog2e, -ref), e = ex2(t);
      s.z += e;
      s.w = fmaf(e, fmaxf(t, -300.f), s.w);
    }
    if (TOP) {
      run = fmaxf(run, most);
      float g = run;
#pragma unroll
      for (int o = 8; o; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xFFFFFFFFu, g, o));
      if ((lane & 15) == 0) group_max[parity][2 * warp + (lane >> 4)] = g;
      __syncthreads();
      g = group_max[parity][lane];
#pragma unroll
      for (int o = 16; o; o >>= 1) g = fminf(g, __shfl_xor_sync(0xFFFFFFFFu, g, o));
      const bool first = r0 == e0;
      bool full = false;
      if (!(most < g) && (first || !(most <= bound))) {
#pragma unroll
        for (int k = 0; k < kLpElems; ++k) {
          const long long i = r0 + (static_cast<long long>(k / VW) * kLpThreads + tid) * VW + k % VW;
          if (i < e1 && !(v[k] < g) && (first || !(v[k] <= bound))) {
            const int at = atomicAdd(&count, 1);
            list[at] = lp_key(v[k], static_cast<uint32_t>(i));
            full = full || at >= kLpMost;
          }
        }
      }
      bound = g;
      if (__syncthreads_or(full)) {  // keep the best only
        const int n = count;
        lp_select(list, n, a.n_top, best, red);
        if (tid < a.n_top) list[tid] = best[tid];
        if (tid == 0) count = a.n_top;
        __syncthreads();
      }
    }
  }
  // the CTA's sums
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    LpSum b{__shfl_xor_sync(0xFFFFFFFFu, s.m, o), __shfl_xor_sync(0xFFFFFFFFu, s.z, o),
            __shfl_xor_sync(0xFFFFFFFFu, s.w, o)};
    s = join(s, b);
  }
  if (lane == 0) sums[warp] = s;
  if (tid == 0) kept = 0;
  __syncthreads();
  if (warp == 0) {
    s = lane < kLpThreads / 32 ? sums[lane] : LpSum{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = 8; o; o >>= 1) {
      LpSum b{__shfl_xor_sync(0xFFFFFFFFu, s.m, o), __shfl_xor_sync(0xFFFFFFFFu, s.z, o),
              __shfl_xor_sync(0xFFFFFFFFu, s.w, o)};
      s = join(s, b);
    }
    if (lane == 0) total = s;
  }
  int n_best = 0;
  if (TOP) {
    const int n = count;
    lp_select(list, n, a.n_top, best, red);
    n_best = min(n, a.n_top);
    if (tid == 0) kept = n_best;
  }
  cluster.sync();  // every CTA's total and best are in its shared memory
  if (rank == 0) {
    LpSum all = total;
    for (int p = 1; p < size; ++p) all = join(all, *cluster.map_shared_rank(&total, p));
    const float logz = log2f(all.z);
    // a row whose largest logit is not finite has no distribution
    const float lse = fabsf(all.m) < INFINITY ? (all.m + logz) : NAN;
    const float nan = lse - lse + (all.z - all.z);  // 0, or NaN
    if (asked) a.logprob[row * a.n_tokens + tid] = fmaf(given, kLog2e, -lse) * kLn2 + nan;
    if (tid == 0 && a.entropy) a.entropy[row] = (logz - all.w / all.z) * kLn2 + nan;
    if (TOP) {
      if (size > 1) {
        int n = n_best;
        __syncthreads();
        if (tid < n) list[tid] = best[tid];
        for (int p = 1; p < size; ++p) {
          const int np = *cluster.map_shared_rank(&kept, p);
          const unsigned long long* theirs = cluster.map_shared_rank(best, p);
          if (tid < np) list[n + tid] = theirs[tid];
          n += np;
        }
        __syncthreads();
        lp_select(list, n, a.n_top, best, red);
      }
      if (tid < a.n_top) {
        const uint32_t id = 0xFFFFFFFFu - static_cast<uint32_t>(best[tid]);
        a.top_id[row * a.n_top + tid] = static_cast<int32_t>(id);
        a.top_lp[row * a.n_top + tid] = fmaf(Act<T>::to(x[id]), kLog2e, -lse) * kLn2 + nan;
      }
    }
  }
  cluster.sync();  // the others' shared memory stays until rank 0 has read it
}

template <class T, bool VEC, bool TOP>
cudaError_t launch_lp(const LpArgs& a, long long rows, int cluster, cudaStream_t st) {
  const size_t smem = TOP ? sizeof(unsigned long long) * kLpList : 0;
  if (TOP) {
    const cudaError_t e = cudaFuncSetAttribute(k_token_logprobs<T, VEC, TOP>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * cluster));
  cfg.blockDim = dim3(kLpThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k_token_logprobs<T, VEC, TOP>, a);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

template <class T>
cudaError_t launch_lp_t(const LpArgs& a, long long rows, bool vec, int cluster, cudaStream_t st) {
  if (a.n_top) return vec ? launch_lp<T, true, true>(a, rows, cluster, st) : launch_lp<T, false, true>(a, rows, cluster, st);
  return vec ? launch_lp<T, true, false>(a, rows, cluster, st) : launch_lp<T, false, false>(a, rows, cluster, st);
}

}  // namespace
}  // namespace m3g

extern "C" {

M3G_API int m3g_token_logprobs_dev(uint32_t dtype, const void* logits, uint64_t rows, uint64_t vocab,
                                   int64_t row_stride, const int32_t* tokens, uint32_t n_tokens, float* logprob,
                                   float* entropy, uint32_t n_top, int32_t* top_id, float* top_logprob,
                                   void* stream) {
  using namespace m3g;
  const int size = act_size(dtype);
  if (!size) return host_fail(M3G_EINVAL, "logits of dtype %u (F32, F16 and BF16 are supported)", dtype);
  if (!vocab || vocab > (1u << 30)) return host_fail(M3G_EINVAL, "vocabulary of %llu",
                                                    static_cast<unsigned long long>(vocab));
  if (rows > (1u << 27)) return host_fail(M3G_EINVAL, "too many rows");
  if (row_stride < 0) return host_fail(M3G_EINVAL, "negative stride");
  if (n_tokens > static_cast<uint32_t>(kLpThreads)) return host_fail(M3G_EINVAL, "%u tokens per row (at most %d)", n_tokens, kLpThreads);
  if (n_top > static_cast<uint32_t>(kLpTop) || n_top > vocab)
    return host_fail(M3G_EINVAL, "%u alternatives (at most %d, and the vocabulary)", n_top, kLpTop);
  if (!rows) return M3G_OK;
  if (!logits || (n_tokens && (!tokens || !logprob)) || (n_top && (!top_id || !top_logprob)))
    return host_fail(M3G_EINVAL, "null argument");
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return host_fail(M3G_ECUDA, "no CUDA device");
  int cluster = 1;
  while (cluster < 8 && rows * cluster * 2 <= 592 && vocab / (cluster * 2) >= 4096) cluster *= 2;
  LpArgs a{};
  a.x = logits;
  a.vocab = static_cast<long long>(vocab);
  a.stride = row_stride;
  a.tokens = tokens;
  a.logprob = logprob;
  a.entropy = entropy;
  a.top_id = top_id;
  a.top_lp = top_logprob;
  a.n_tokens = static_cast<int>(n_tokens);
  a.n_top = static_cast<int>(n_top);
  a.chunk = static_cast<int>((vocab + cluster - 1) / cluster + 15) / 16 * 16;
  const bool vec = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && row_stride * size % 16 == 0;
  const cudaStream_t st = serve_stream(stream);
  const long long n = static_cast<long long>(rows);
  const cudaError_t e = dtype == M3G_DTYPE_F32   ? launch_lp_t<float>(a, n, vec, cluster, st)
                        : dtype == M3G_DTYPE_F16 ? launch_lp_t<__half>(a, n, vec, cluster, st)
                                                 : launch_lp_t<__nv_bfloat16>(a, n, vec, cluster, st);
  if (e != cudaSuccess) return host_fail(M3G_ECUDA, "k_token_logprobs: %s", cudaGetErrorString(e));
  return M3G_OK;
}

}  // extern "C"
