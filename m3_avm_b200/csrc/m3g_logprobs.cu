// m3g_logprobs.cu -- log probabilities of given tokens, entropy and the most
// probable alternatives of each row of logits, in one pass over the row.
//
// Each thread keeps, in base 2, the running maximum m of its logits, z = sum
// 2^(t - m) and w = sum 2^(t - m) (t - m) with t = x log2(e); they join like
// the partial sums of a softmax:  lse = (m + log2 z) ln 2,  H = (log2 z -
// w / z) ln 2.
//
// The alternatives come out of the same pass.  The CTA's 32 half-warps keep
// running maxima, each of a different element, so the n_top-th largest of the
// 32 is a bound that at least n_top elements reach: an element below it is not
// among the best.  Elements that reach the bound (and are above -inf) go to a
// list in shared memory, and their warp raises the bound.  Maxima and bound
// only grow, so any stale value is a valid bound: after the first round no
// thread waits for another, and a round in which nothing reaches the bound
// costs a load and a vote.  Of random logits some n_top ln(vocab / round)
// elements pass.  At the end those that reach the last bound are ranked by
// counting.  Rows for which the list overflows or stays short (thousands of
// equal logits; fewer finite ones than alternatives) are walked again by
// lp_walk, which is exact for any row.
//
// A row is read by a cluster of 1 .. 8 CTAs, whose sums and lists join through
// distributed shared memory: 8 while the rows do not fill the SMs.
#include <cmath>
#include <type_traits>

#include <cooperative_groups.h>

#include "m3g_serve.cuh"

namespace cg = cooperative_groups;

namespace m3g {
namespace {

constexpr int kLpThreads = 512;
constexpr int kLpVecs = 4;                          // 16-byte loads per thread and round, one round ahead
constexpr int kLpList = 2048;                       // entries of the list of candidates
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

__device__ __forceinline__ LpSum join_lanes(LpSum s, int lanes) {
  for (int o = lanes >> 1; o; o >>= 1) {
    const LpSum b{__shfl_xor_sync(0xFFFFFFFFu, s.m, o), __shfl_xor_sync(0xFFFFFFFFu, s.z, o),
                  __shfl_xor_sync(0xFFFFFFFFu, s.w, o)};
    s = join(s, b);
  }
  return s;
}

// The largest of a round's logits; NaN is left out.
template <class T, int N>
__device__ __forceinline__ float largest(const T (&t)[N]) {
  if constexpr (sizeof(T) == 2) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2 m = *reinterpret_cast<const T2*>(&t[0]);
#pragma unroll
    for (int i = 2; i < N; i += 2) m = __hmax2(m, *reinterpret_cast<const T2*>(&t[i]));
    return fmaxf(Act<T>::to(m.x), Act<T>::to(m.y));
  } else {
    float m = t[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, t[i]);
    return m;
  }
}

// The k-th largest of the 32 lanes' values (ties in lane order).
__device__ __forceinline__ float kth_of_lanes(float g, int k) {
  const int lane = threadIdx.x & 31;
  int above = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const float o = __shfl_sync(0xFFFFFFFFu, g, i);
    above += o > g || (o == g && i < lane);
  }
  return __shfl_sync(0xFFFFFFFFu, g, __ffs(__ballot_sync(0xFFFFFFFFu, above == k - 1)) - 1);
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

// The best min(k, e1 - e0) of x[e0 .. e1) in order into best; any logits.  All
// threads; the list holds what beats the k-th best so far.
template <class T>
__device__ int lp_walk(const T* x, long long e0, long long e1, int k, unsigned long long* list,
                       unsigned long long* best, unsigned long long* red, int* count) {
  constexpr int kStep = kLpList / 2;
  const int tid = threadIdx.x;
  unsigned long long bound = 0;  // every key is above 0
  __syncthreads();
  if (tid == 0) *count = 0;
  __syncthreads();
  for (long long r0 = e0; r0 < e1; r0 += kStep) {
    bool full = false;
    for (int j = tid; j < kStep; j += kLpThreads) {
      if (r0 + j >= e1) break;
      const unsigned long long key = lp_key(Act<T>::to(x[r0 + j]), static_cast<uint32_t>(r0 + j));
      if (key > bound) {
        const int at = atomicAdd(count, 1);
        list[at] = key;
        full = full || at >= kLpList - kStep;
      }
    }
    if (__syncthreads_or(full)) {
      lp_select(list, *count, k, best, red);
      if (tid < k) list[tid] = best[tid];
      bound = best[k - 1];
      if (tid == 0) *count = k;
      __syncthreads();
    }
  }
  __syncthreads();
  const int n = *count;
  lp_select(list, n, k, best, red);
  return min(n, k);
}

template <class T, bool VEC, bool TOP>
__global__ void __launch_bounds__(kLpThreads, 2) k_token_logprobs(const __grid_constant__ LpArgs a) {
  constexpr int VW = 16 / sizeof(T), E = kLpVecs * VW, kRound = kLpThreads * E;
  constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
  __shared__ unsigned long long list[TOP ? kLpList : 1];
  __shared__ unsigned long long best[kLpTop], red[kLpThreads / 32];
  __shared__ float group_max[32];
  __shared__ float shared_bound;
  __shared__ LpSum sums[kLpThreads / 32];
  __shared__ LpSum total;
  __shared__ int count;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), size = static_cast<int>(cluster.num_blocks());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long row = blockIdx.x / size;
  const T* x = static_cast<const T*>(a.x) + row * a.stride;
  const long long e0 = static_cast<long long>(rank) * a.chunk;
  const long long e1 = min(a.vocab, e0 + a.chunk);
  union Raw {  // a round's logits of this thread
    uint4 q[kLpVecs];
    T t[E];
    __device__ Raw() {}
  };
  auto fetch = [&](long long r0, Raw& w) {
#pragma unroll
    for (int j = 0; j < kLpVecs; ++j) {
      const long long i = r0 + (j * kLpThreads + tid) * VW;
      if (VEC && i + VW <= e1) {
        w.q[j] = __ldcs(reinterpret_cast<const uint4*>(x + i));
      } else {
#pragma unroll
        for (int k = 0; k < VW; ++k) w.t[j * VW + k] = i + k < e1 ? x[i + k] : Act<T>::from(-INFINITY);
      }
    }
  };
  LpSum s{-INFINITY, 0.f, 0.f};
  float run = -INFINITY, bound = -INFINITY;
  auto use = [&](long long r0, const Raw& w) {
    const float most = largest<T, E>(w.t);
    const float t_most = most * kLog2e;
    if (t_most > s.m) {
      const float d = fmaxf(s.m - t_most, -300.f), f = ex2(s.m - t_most);
      s.w = f * (s.w + d * s.z);
      s.z = f * s.z;
      s.m = t_most;
    }
    const float ref = s.m == -INFINITY ? 0.f : s.m;
    float z[2] = {0.f, 0.f}, y[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const float t = fmaf(Act<T>::to(w.t[k]), kLog2e, -ref), e = ex2(t);
      z[k & 1] += e;
      y[k & 1] = fmaf(e, fmaxf(t, -300.f), y[k & 1]);
    }
    s.z += z[0] + z[1];
    s.w += y[0] + y[1];
    if (TOP) {
      run = fmaxf(run, most);
      auto raise = [&] {  // this warp's maxima into the shared ones, the bound from all of them
        float g = run;
#pragma unroll
        for (int o = 8; o; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xFFFFFFFFu, g, o));
        if ((lane & 15) == 0) *const_cast<volatile float*>(&group_max[2 * warp + (lane >> 4)]) = g;
        if (r0 == e0) __syncthreads();
        else __syncwarp();
        bound = kth_of_lanes(*const_cast<volatile float*>(&group_max[lane]), a.n_top);
        if (lane == 0) *const_cast<volatile float*>(&shared_bound) = bound;
      };
      if (r0 == e0) raise();
      else bound = fmaxf(bound, *const_cast<volatile float*>(&shared_bound));
      const bool reaches = most >= bound && most > -INFINITY;
      if (__any_sync(0xFFFFFFFFu, reaches)) {
        if (reaches) {
#pragma unroll
          for (int k = 0; k < E; ++k) {
            const float v = Act<T>::to(w.t[k]);
            if (v >= bound && v > -INFINITY) {
              const int at = atomicAdd(&count, 1);
              const long long i = r0 + ((k / VW) * kLpThreads + tid) * VW + k % VW;
              if (at < kLpList) list[at] = lp_key(v, static_cast<uint32_t>(i));
            }
          }
        }
        if (r0 != e0) {
          __syncwarp();
          raise();
        }
      }
    }
  };
  Raw now, next;
  if (e0 < e1) fetch(e0, now);
  float given = 0.f;
  const bool asked = rank == 0 && tid < a.n_tokens;
  if (asked) {
    const long long id = a.tokens[row * a.n_tokens + tid];
    given = id >= 0 && id < a.vocab ? Act<T>::to(x[id]) : -INFINITY;
  }
  if (tid == 0) count = 0;
  if (TOP) __syncthreads();
  for (long long r0 = e0; r0 < e1; r0 += kRound) {
    if (r0 + kRound < e1) fetch(r0 + kRound, next);
    use(r0, now);
    now = next;
  }
  // the CTA's sums
  s = join_lanes(s, 32);
  if (lane == 0) sums[warp] = s;
  __syncthreads();
  if (warp == 0) {
    s = join_lanes(lane < kLpThreads / 32 ? sums[lane] : LpSum{-INFINITY, 0.f, 0.f}, 32);
    if (lane == 0) total = s;
  }
  if (TOP) {
    const int n = count, most = static_cast<int>(min(static_cast<long long>(a.n_top), e1 - e0));
    __syncthreads();
    int got;
    if (n > kLpList || n < most) {
      got = lp_walk(x, e0, e1, a.n_top, list, best, red, &count);
    } else {
      // those that reach the last bound, in place (a thread's entries are read before any is written)
      bound = kth_of_lanes(group_max[lane], a.n_top);
      const unsigned long long least = lp_key(bound, 0xFFFFFFFFu);
      unsigned long long keep[kLpList / kLpThreads];
#pragma unroll
      for (int j = 0; j < kLpList / kLpThreads; ++j) keep[j] = tid + j * kLpThreads < n ? list[tid + j * kLpThreads] : 0;
      if (tid == 0) count = 0;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kLpList / kLpThreads; ++j)
        if (keep[j] >= least) list[atomicAdd(&count, 1)] = keep[j];
      __syncthreads();
      const int left = count;
      lp_select(list, left, a.n_top, best, red);
      got = min(left, a.n_top);
    }
    if (tid >= got && tid < a.n_top) best[tid] = 0;  // below every key
  }
  if (size > 1) cluster.sync();  // every CTA's total and best are in its shared memory
  else __syncthreads();
  if (rank == 0) {
    LpSum all = total;
    if (size > 1) all = join_lanes(lane < size ? *cluster.map_shared_rank(&total, lane) : LpSum{-INFINITY, 0.f, 0.f}, 32);
    if (TOP && size > 1) {
      unsigned long long mine = 0;
      if (tid < size * a.n_top) mine = cluster.map_shared_rank(best, tid / a.n_top)[tid % a.n_top];
      if (tid < size * a.n_top) list[tid] = mine;
      __syncthreads();
      lp_select(list, size * a.n_top, a.n_top, best, red);
    }
    const float logz = log2f(all.z);
    // a row whose largest logit is not finite has no distribution
    const float lse = fabsf(all.m) < INFINITY ? (all.m + logz) : NAN;
    const float nan = lse - lse + (all.z - all.z);  // 0, or NaN
    if (asked) a.logprob[row * a.n_tokens + tid] = fmaf(given, kLog2e, -lse) * kLn2 + nan;
    if (tid == 0 && a.entropy) a.entropy[row] = (logz - all.w / all.z) * kLn2 + nan;
    if (TOP && tid < a.n_top) {
      const uint32_t hi = static_cast<uint32_t>(best[tid] >> 32);  // the key's logit back
      const float v = hi == 0 ? NAN : __uint_as_float(hi & 0x80000000u ? hi & 0x7FFFFFFFu : ~hi);
      a.top_id[row * a.n_top + tid] = static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(best[tid]));
      a.top_lp[row * a.n_top + tid] = fmaf(v, kLog2e, -lse) * kLn2 + nan;
    }
  }
  if (size > 1) cluster.sync();  // the others' shared memory stays until rank 0 has read it
}

template <class T, bool VEC, bool TOP>
cudaError_t launch_lp(const LpArgs& a, long long rows, int cluster, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * cluster));
  cfg.blockDim = dim3(kLpThreads);
  cfg.dynamicSmemBytes = 0;
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
