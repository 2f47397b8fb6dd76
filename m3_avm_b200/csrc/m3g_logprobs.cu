// m3g_logprobs.cu -- log probabilities of given tokens, entropy and the most
// probable alternatives of each row of logits, in one pass over the row.
//
// Each thread keeps, in base 2, the running maximum m of its logits, z = sum
// 2^(t - m) and w = sum 2^(t - m) (t - m) with t = x log2(e); they join like
// the partial sums of a softmax:  lse = (m + log2 z) ln 2,  H = (log2 z -
// w / z) ln 2.
//
// The alternatives come out of the same pass.  The first round's 32 half-warp
// maxima are of different elements, so the n_top-th largest of them is a bound
// that at least n_top elements reach: an element below it is not among the
// best.  A thread with an element that reaches the bound (and is above -inf)
// copies its logits of that round, as they are, to shared memory; what the bound
// leaves of them is ranked by counting once the row has been read.  Some n_top
// threads of each round reach the first bound in a row in no order.  Above kLpRaise
// copies the warps that add some share their running maxima and raise the bound.
// Maxima and bound only grow, so any stale value is a valid bound and no thread
// waits for another after the first round.  Rows with more copies than fit, too many
// equal logits or fewer finite ones than alternatives are walked again by lp_walk,
// which is exact for any row.
//
// The sums take logits below Lp<T>::kLow as that value, which leaves -inf out of
// the products; it matters only in rows without a larger logit.  Those, rows of
// logits above 1e38 (which leave f32 in base 2) and rows without a distribution
// are walked again by lp_extreme: logits that far out are so coarse that all
// but the largest have a probability of 0.
//
// A row is read by a cluster of 1 .. 8 CTAs, whose sums and lists join through
// distributed shared memory: as many as leave no SM with two.
//
// Measured: 1031 BF16 rows of 128256 with 5 alternatives 66 us (4.0 TB/s; without
// alternatives 53).  The exponentials, 16 a cycle and SM, take 36 us by themselves,
// the rest of the loop about as many issue slots; reading takes 41.  One F32 row
// with 20 alternatives 11 us: launch, two loads' latency and the joins in turn.
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
constexpr int kLpCopies = 384;                      // copies of a thread's logits of one round
constexpr int kLpRaise = 96;                        // copies from which the bound is raised
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

// Smallest logit that the sums tell apart, and the smallest of a row's largest
// for which they hold.
template <class T> struct Lp { static constexpr float kLow = -0x1p126f, kRowLow = -0x1p126f; };  // exact in BF16
template <> struct Lp<__half> { static constexpr float kLow = -65504.f, kRowLow = -32768.f; };
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ uint64_t unpack2(__half2 x) {
  const float2 f = __half22float2(x);
  return pair(f.x, f.y);
}
__device__ __forceinline__ uint64_t unpack2(__nv_bfloat162 x) {
  const uint32_t u = *reinterpret_cast<const uint32_t*>(&x);
  return pair(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}

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
#pragma unroll 8
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
// Up to kLpThreads entries 1 .. 32 threads for each count what beats it; longer
// lists (rows of equal logits) give up their best k times.
__device__ __noinline__ void lp_select(const unsigned long long* list, int n, int k, unsigned long long* best,
                                       unsigned long long* red) {
  const int tid = threadIdx.x;
  if (n <= kLpThreads) {
    const int parts = min(32, 1 << (31 - __clz(kLpThreads / max(n, 1)))), c = tid / parts;
    const unsigned long long mine = c < n ? list[c] : 0;
    int beaten = 0;
    if (c < n) {
#pragma unroll 4
      for (int i = tid & (parts - 1); i < n; i += parts) beaten += list[i] > mine;
    }
    for (int o = parts >> 1; o; o >>= 1) beaten += __shfl_xor_sync(0xFFFFFFFFu, beaten, o);
    if (c < n && beaten < k && (tid & (parts - 1)) == 0) best[beaten] = mine;
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
__device__ __noinline__ int lp_walk(const T* x, long long e0, long long e1, int k, unsigned long long* list,
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

// The largest of x[e0 .. e1) as m, how many equal it as z, NaN as w if one is NaN
// (0 otherwise); all threads, the same in each.
template <class T>
__device__ __noinline__ LpSum lp_extreme(const T* x, long long e0, long long e1, LpSum* sums) {
  const int tid = threadIdx.x, lane = tid & 31;
  LpSum s{-INFINITY, 0.f, 0.f};
  auto merge = [](LpSum a, LpSum b) {
    const float m = fmaxf(a.m, b.m);
    return LpSum{m, (a.m == m ? a.z : 0.f) + (b.m == m ? b.z : 0.f), a.w + b.w};
  };
  for (long long i = e0 + tid; i < e1; i += kLpThreads) {
    const float v = Act<T>::to(x[i]);
    s = merge(s, LpSum{v, 1.f, v != v ? v : 0.f});
  }
#pragma unroll
  for (int o = 16; o; o >>= 1)
    s = merge(s, LpSum{__shfl_xor_sync(0xFFFFFFFFu, s.m, o), __shfl_xor_sync(0xFFFFFFFFu, s.z, o),
                       __shfl_xor_sync(0xFFFFFFFFu, s.w, o)});
  __syncthreads();
  if (lane == 0) sums[tid >> 5] = s;
  __syncthreads();
  s = sums[0];
  for (int i = 1; i < kLpThreads / 32; ++i) s = merge(s, sums[i]);
  return s;
}

// Logits lo .. hi-1 of 16 bytes of them, -inf for the others.
template <class T>
__device__ __noinline__ uint4 lp_part(const T* x, int lo, int hi) {
  constexpr int VW = 16 / sizeof(T);
  __align__(16) T t[VW];
#pragma unroll
  for (int k = 0; k < VW; ++k) t[k] = k >= lo && k < hi ? x[k] : Act<T>::from(-INFINITY);
  return *reinterpret_cast<const uint4*>(t);
}

template <class T, bool TOP>
__global__ void __launch_bounds__(kLpThreads, 2) k_token_logprobs(const __grid_constant__ LpArgs a) {
  constexpr int VW = 16 / sizeof(T), E = kLpVecs * VW, kRound = kLpThreads * E;
  __shared__ unsigned long long list[TOP ? kLpList : 1];
  __shared__ uint4 copies[TOP ? kLpCopies : 1][kLpVecs];
  __shared__ int copy_of[TOP ? kLpCopies : 1];  // round * kLpThreads + thread
  __shared__ unsigned long long best[kLpTop], red[kLpThreads / 32];
  __shared__ float group_max[32];
  __shared__ LpSum sums[kLpThreads / 32];
  __shared__ LpSum total, coarse;
  __shared__ int count, n_copies;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), size = static_cast<int>(cluster.num_blocks());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long row = blockIdx.x / size;
  const T* x = static_cast<const T*>(a.x) + row * a.stride;
  // Elements are counted from the 16-byte boundary at or before the row: `lead` are not the row's.
  const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
  const T* base = x - lead;
  const long long e0 = static_cast<long long>(rank) * a.chunk;
  const long long e1 = min(a.vocab + lead, e0 + a.chunk);
  const long long own0 = max(e0 - lead, 0ll), own1 = e1 - lead;  // the CTA's logits
  union Raw {  // a round's logits of this thread
    uint4 q[kLpVecs];
    T t[E];
    __device__ Raw() {}
  };
  uint4 none;  // -inf throughout
  none.x = none.y = none.z = none.w = sizeof(T) == 4 ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
  auto fetch = [&](long long r0, Raw& w) {
    if (r0 >= lead && r0 + kRound <= e1) {
      const uint4* p = reinterpret_cast<const uint4*>(base + r0) + tid;
#pragma unroll
      for (int j = 0; j < kLpVecs; ++j) w.q[j] = __ldcs(p + j * kLpThreads);
      return;
    }
#pragma unroll
    for (int j = 0; j < kLpVecs; ++j) {
      const long long i = r0 + (j * kLpThreads + tid) * VW;
      if (i >= lead && i + VW <= e1) w.q[j] = __ldcs(reinterpret_cast<const uint4*>(base + i));
      else if (i >= e1) w.q[j] = none;
      else w.q[j] = lp_part(base + i, static_cast<int>(max(lead - i, 0ll)), static_cast<int>(min(e1 - i, static_cast<long long>(VW))));
    }
  };
  LpSum s{-INFINITY, 0.f, 0.f};
  float run = -INFINITY, bound = -INFINITY;
  bool again = true;  // the bound is to be raised
  // Lanes to a group whose maximum counts for the bound: a half-warp, fewer where a
  // short row leaves threads without logits, so that 32 groups have some (with 17 of
  // 32 alternatives had no bound, and such rows were read twice: 1031 BF16 rows of
  // 3500 logits with 32 alternatives 176 us, now 55; one row 32.6, now 8.1).
  int group = 16;
  while (group > 1 && e1 - e0 < 32ll * group * VW) group >>= 1;
  auto use = [&](long long r0, const Raw& w) {
    const float most = largest<T, E>(w.t);
    const float t_most = fmaxf(most, Lp<T>::kLow) * kLog2e;
    if (t_most > s.m) {
      const float d = fmaxf(s.m - t_most, -300.f), f = ex2(s.m - t_most);
      s.w = f * (s.w + d * s.z);
      s.z = f * s.z;
      s.m = t_most;
    }
    if constexpr (sizeof(T) == 2) {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      T2 least;
      least.x = least.y = Act<T>::from(Lp<T>::kLow);
      const uint64_t scale = pair(kLog2e, kLog2e), ref = pair(-s.m, -s.m);
      uint64_t z = 0, y = 0;  // pairs of +0
#pragma unroll
      for (int k = 0; k < E; k += 2) {
        const uint64_t t = fma2(unpack2(__hmax2_nan(*reinterpret_cast<const T2*>(&w.t[k]), least)), scale, ref);
        const uint64_t e = pair(ex2(low(t)), ex2(high(t)));
        z = add2(z, e);
        y = fma2(e, t, y);
      }
      s.z += low(z) + high(z);
      s.w += low(y) + high(y);
    } else {
      float z[2] = {0.f, 0.f}, y[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const float t = fmaf(Act<T>::to(w.t[k]), kLog2e, -s.m), e = ex2(t);
        z[k & 1] += e;
        y[k & 1] = fmaf(e, fmaxf(t, -300.f), y[k & 1]);
      }
      s.z += z[0] + z[1];
      s.w += y[0] + y[1];
    }
    if (TOP) {
      run = fmaxf(run, most);
      if (again) {  // this warp's maxima into the shared ones, the bound from all of them
        float g = run;
        for (int o = group >> 1; o; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xFFFFFFFFu, g, o));
        if ((lane & (group - 1)) == 0 && tid < 32 * group) *const_cast<volatile float*>(&group_max[tid / group]) = g;
        if (r0 == e0) __syncthreads();
        else __syncwarp();
        bound = kth_of_lanes(*const_cast<volatile float*>(&group_max[lane]), a.n_top);
        again = false;
      }
      const bool reaches = most >= bound && most > -INFINITY;
      if (__any_sync(0xFFFFFFFFu, reaches)) {
        if (reaches) {
          const int at = atomicAdd(&n_copies, 1);
          if (at < kLpCopies) {
            copy_of[at] = static_cast<int>((r0 - e0) / kRound) * kLpThreads + tid;
#pragma unroll
            for (int j = 0; j < kLpVecs; ++j) copies[at][j] = w.q[j];
          }
        }
        __syncwarp();
        again = __shfl_sync(0xFFFFFFFFu, *const_cast<volatile int*>(&n_copies), 0) >= kLpRaise;
      }
    }
  };
  Raw now, next;
  float given = 0.f;
  const bool asked = rank == 0 && tid < a.n_tokens;
  if (asked) {
    const long long id = a.tokens[row * a.n_tokens + tid];
    given = id >= 0 && id < a.vocab ? Act<T>::to(x[id]) : -INFINITY;
  }
  if (tid == 0) count = n_copies = 0;
  if (TOP) __syncthreads();
  for (long long r0 = e0 - kRound; r0 < e1; r0 += kRound) {
    if (r0 + kRound < e1) fetch(r0 + kRound, next);
    if (r0 >= e0) use(r0, now);
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
    const int most = static_cast<int>(min(static_cast<long long>(a.n_top), own1 - own0));
    const int kept = n_copies;
    for (int c = warp; c < min(kept, kLpCopies); c += kLpThreads / 32) {
      if (lane < E) {
        const float v = Act<T>::to(reinterpret_cast<const T*>(copies[c])[lane]);
        if (v >= bound && v > -INFINITY) {
          const int at = atomicAdd(&count, 1), round = copy_of[c] / kLpThreads, thread = copy_of[c] % kLpThreads;
          const long long i = e0 - lead + static_cast<long long>(round) * kRound + (lane / VW * kLpThreads + thread) * VW + lane % VW;
          if (at < kLpList) list[at] = lp_key(v, static_cast<uint32_t>(i));
        }
      }
    }
    __syncthreads();
    const int n = count;
    int got;
    if (kept > kLpCopies || n > kLpList || n < most) {
      got = lp_walk(x, own0, own1, a.n_top, list, best, red, &count);
    } else {
      lp_select(list, n, a.n_top, best, red);
      got = min(n, a.n_top);
    }
    if (tid >= got && tid < a.n_top) best[tid] = 0;  // below every key
  }
  if (size > 1) cluster.sync();  // every CTA's total and best are in its shared memory
  else __syncthreads();
  LpSum all = total;
  if (size > 1) all = join_lanes(lane < size ? *cluster.map_shared_rank(&total, lane) : LpSum{-INFINITY, 0.f, 0.f}, 32);
  const bool extreme = !(all.m > Lp<T>::kRowLow * kLog2e && all.m < 1e38f * kLog2e);  // the same in the whole cluster
  if (extreme) {
    const LpSum mine = lp_extreme(x, own0, own1, sums);
    if (tid == 0) coarse = mine;
    if (size > 1) cluster.sync();
    else __syncthreads();
    if (rank == 0) {
      all = coarse;
      for (int i = 1; i < size; ++i) {
        const LpSum b = *cluster.map_shared_rank(&coarse, i);
        const float m = fmaxf(all.m, b.m);
        all = LpSum{m, (all.m == m ? all.z : 0.f) + (b.m == m ? b.z : 0.f), all.w + b.w};
      }
    }
  }
  if (rank == 0) {
    if (TOP && size > 1) {
      unsigned long long mine = 0;
      if (tid < size * a.n_top) mine = cluster.map_shared_rank(best, tid / a.n_top)[tid % a.n_top];
      if (tid < size * a.n_top) list[tid] = mine;
      __syncthreads();
      lp_select(list, size * a.n_top, a.n_top, best, red);
    }
    const float logz = log2f(all.z);
    // 0, or NaN in a row without a distribution: a largest logit that is not finite, a NaN
    const float nan = extreme ? (fabsf(all.m) < INFINITY ? all.w : NAN) : all.z - all.z;
    auto log_prob = [&](float v) {  // in halves: v log2(e) may leave f32
      return nan + (extreme ? (v - all.m) - logz * kLn2
                            : (fmaf(0.5f * v, kLog2e, -0.5f * all.m) - 0.5f * logz) * (2.f * kLn2));
    };
    if (asked) a.logprob[row * a.n_tokens + tid] = log_prob(given);
    if (tid == 0 && a.entropy) a.entropy[row] = (extreme ? logz : logz - all.w / all.z) * kLn2 + nan;
    if (TOP && tid < a.n_top) {
      const uint32_t hi = static_cast<uint32_t>(best[tid] >> 32);  // the key's logit back
      const float v = hi == 0 ? NAN : __uint_as_float(hi & 0x80000000u ? hi & 0x7FFFFFFFu : ~hi);
      a.top_id[row * a.n_top + tid] = static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(best[tid]));
      a.top_lp[row * a.n_top + tid] = log_prob(v);
    }
  }
  if (size > 1) cluster.sync();  // the others' shared memory stays until rank 0 has read it
}

template <class T, bool TOP>
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k_token_logprobs<T, TOP>, a);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

template <class T>
cudaError_t launch_lp_t(const LpArgs& a, long long rows, int cluster, cudaStream_t st) {
  return a.n_top ? launch_lp<T, true>(a, rows, cluster, st) : launch_lp<T, false>(a, rows, cluster, st);
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
  if (misaligned(logits, size)) return host_fail(M3G_EINVAL, "logits not aligned to their type");
  for (const void* p : {static_cast<const void*>(tokens), static_cast<const void*>(logprob),
                        static_cast<const void*>(entropy), static_cast<const void*>(top_id),
                        static_cast<const void*>(top_logprob)})
    if (misaligned(p, 4)) return host_fail(M3G_EINVAL, "tokens or results not 4-byte aligned");
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return host_fail(M3G_ECUDA, "no CUDA device");
  // As many CTAs to a row as the SMs hold one each of: clusters that come in a
  // second wave wait for whole ones to end (74 rows of 128256 BF16, 20 alternatives:
  // 15 us with 148 CTAs, 35 with 592; 148 rows 17 us with one CTA each, 35 with four).
  int cluster = 1;
  while (cluster < 8 && rows * cluster * 2 <= 148 && vocab / (cluster * 2) >= 4096) cluster *= 2;
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
  a.chunk = static_cast<int>((vocab + 7 + cluster - 1) / cluster + 15) / 16 * 16;  // 7: the most a row starts behind a boundary
  const cudaStream_t st = serve_stream(stream);
  const long long n = static_cast<long long>(rows);
  const cudaError_t e = dtype == M3G_DTYPE_F32   ? launch_lp_t<float>(a, n, cluster, st)
                        : dtype == M3G_DTYPE_F16 ? launch_lp_t<__half>(a, n, cluster, st)
                                                 : launch_lp_t<__nv_bfloat16>(a, n, cluster, st);
  if (e != cudaSuccess) return host_fail(M3G_ECUDA, "k_token_logprobs: %s", cudaGetErrorString(e));
  return M3G_OK;
}

}  // extern "C"
