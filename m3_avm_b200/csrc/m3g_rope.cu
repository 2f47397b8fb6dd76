// m3g_rope.cu -- rotary positions of q and k rows.
//
// Pair i of a token at position p turns by the angle p * f_i.  The plan holds
// f_i / 2pi as a 64-bit fraction of a turn, so p * f_i modulo one turn is one
// wrapping 64-bit integer product, exact to p * 2^-53 of f_i's own rounding:
// no range reduction, and far positions lose nothing (an f32 product is off by
// 0.06 rad at position 10^6).  sincospif of the top 32 bits gives cos and sin
// once per token; all its heads share them through shared memory.
//
// Bound: HBM (each element read and written once).  One CTA per token; each
// thread loads its first units before the angles are ready, so the angle
// arithmetic hides behind the loads.
#include <cmath>
#include <new>

#include "m3g_serve.cuh"

struct m3g_rope {
  m3g_rope_config cfg;
  unsigned long long turn[128];  // f_i / 2pi, in units of 2^-64 turns
  float magnitude;
};

namespace m3g {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kMaxPairs = 128;

struct RopeArgs {
  const int32_t* positions;
  m3g_rope_rows r[2];
  int heads, heads0;     // rows of both tensors; of the first
  int head_dim, rot;
  int inverse;
  float magnitude;
  unsigned long long turn[kMaxPairs];
};

// A unit is V pairs (two vectors of V values for the half layout, one of 2V
// when interleaved) or, behind rot, one vector of V (2V) values to copy.
template <class T, int V, bool VEC, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) k_rope(const __grid_constant__ RopeArgs a) {
  __shared__ float2 cs[kMaxPairs];
  constexpr int U = 4;       // units a thread holds at once
  constexpr int W = 2 * V;   // values of a unit
  const int t = blockIdx.x, tid = threadIdx.x, half = a.rot / 2;
  const int np = half / V, nt = (a.head_dim - a.rot + (INTER ? W : V) - 1) / (INTER ? W : V);
  const int per = np + nt, units = a.heads * per;
  const int pos = a.positions[t];
  float v[U][W];
  auto place = [&](int u, const T** x, T** y, int* c) {
    const int h = u / per;
    *c = u - h * per;
    const m3g_rope_rows& r = a.r[h >= a.heads0];
    const long long hh = h >= a.heads0 ? h - a.heads0 : h;
    *x = static_cast<const T*>(r.x) + t * r.x_token_stride + hh * r.x_head_stride;
    *y = static_cast<T*>(r.y) + t * r.y_token_stride + hh * r.y_head_stride;
  };
  auto load = [&](int u, float (&w)[W]) {
    const T* x;
    T* y;
    int c;
    place(u, &x, &y, &c);
    if (INTER) {
      if (c < np) load_act<T, W, VEC>(x + c * W, w);
      else if (x != y) load_act<T, W, VEC>(x + a.rot + (c - np) * W, w);
    } else {
      float (&lo)[V] = *reinterpret_cast<float(*)[V]>(&w[0]);
      float (&hi)[V] = *reinterpret_cast<float(*)[V]>(&w[V]);
      if (c < np) {
        load_act<T, V, VEC>(x + c * V, lo);
        load_act<T, V, VEC>(x + half + c * V, hi);
      } else if (x != y) {
        load_act<T, V, VEC>(x + a.rot + (c - np) * V, lo);
      }
    }
  };
  auto finish = [&](int u, float (&w)[W]) {
    const T* x;
    T* y;
    int c;
    place(u, &x, &y, &c);
    if (c >= np) {
      if (x == y) return;
      if (INTER) {
        store_act<T, W, VEC>(y + a.rot + (c - np) * W, w);
      } else {
        store_act<T, V, VEC>(y + a.rot + (c - np) * V, *reinterpret_cast<float(*)[V]>(&w[0]));
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float& p = w[INTER ? 2 * i : i];
      float& q = w[INTER ? 2 * i + 1 : V + i];
      const float2 r = cs[c * V + i];
      const float p0 = p, q0 = q;
      p = p0 * r.x - q0 * r.y;
      q = p0 * r.y + q0 * r.x;
    }
    if (INTER) {
      store_act<T, W, VEC>(y + c * W, w);
    } else {
      store_act<T, V, VEC>(y + c * V, *reinterpret_cast<float(*)[V]>(&w[0]));
      store_act<T, V, VEC>(y + half + c * V, *reinterpret_cast<float(*)[V]>(&w[V]));
    }
  };
#pragma unroll
  for (int k = 0; k < U; ++k)
    if (tid + k * kRopeThreads < units) load(tid + k * kRopeThreads, v[k]);
  if (tid < half) {
    const long long p = a.inverse ? -static_cast<long long>(pos) : static_cast<long long>(pos);
    const unsigned long long turns = static_cast<unsigned long long>(p) * a.turn[tid];
    float s, c;
    // the top 32 bits as a signed fraction of a turn, in half turns
    sincospif(static_cast<float>(static_cast<int>(turns >> 32)) * 0x1p-31f, &s, &c);
    cs[tid] = make_float2(c * a.magnitude, s * a.magnitude);
  }
  __syncthreads();
  for (int u0 = tid; u0 < units; u0 += U * kRopeThreads) {
    if (u0 != tid) {
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (u0 + k * kRopeThreads < units) load(u0 + k * kRopeThreads, v[k]);
    }
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (u0 + k * kRopeThreads < units) finish(u0 + k * kRopeThreads, v[k]);
  }
}

template <class T, bool INTER>
cudaError_t launch_rope_t(const RopeArgs& a, bool vec, unsigned grid, cudaStream_t st) {
  // 16-byte vectors: V pairs are two of them (half layout), or one (interleaved)
  constexpr int V = INTER ? 8 / sizeof(T) : 16 / sizeof(T);
  if (vec) return serve_launch(k_rope<T, V, true, INTER>, dim3(grid), dim3(kRopeThreads), 0, st, false, a);
  return serve_launch(k_rope<T, 1, false, INTER>, dim3(grid), dim3(kRopeThreads), 0, st, false, a);
}

template <class T>
cudaError_t launch_rope(const RopeArgs& a, bool vec, bool inter, unsigned grid, cudaStream_t st) {
  return inter ? launch_rope_t<T, true>(a, vec, grid, st) : launch_rope_t<T, false>(a, vec, grid, st);
}

}  // namespace
}  // namespace m3g

extern "C" {

M3G_API int m3g_rope_create(const m3g_rope_config* cfg, m3g_rope** out) {
  using m3g::host_fail;
  if (!cfg || !out) return host_fail(M3G_EINVAL, "null argument");
  *out = nullptr;
  const m3g_rope_config& c = *cfg;
  if (!c.head_dim || c.head_dim > 512 || c.head_dim % 2)
    return host_fail(M3G_EINVAL, "head_dim %u (even, 2 .. 512)", c.head_dim);
  if (c.rot_dim < 2 || c.rot_dim % 2 || c.rot_dim > c.head_dim || c.rot_dim > 2 * m3g::kMaxPairs)
    return host_fail(M3G_EINVAL, "rot_dim %u (even, 2 .. min(head_dim, 256))", c.rot_dim);
  if (c.interleaved > 1) return host_fail(M3G_EINVAL, "interleaved must be 0 or 1");
  if (c.scaling > M3G_ROPE_LLAMA3) return host_fail(M3G_EINVAL, "unknown scaling %u", c.scaling);
  if (!(c.theta > 1.0) || !std::isfinite(c.theta)) return host_fail(M3G_EINVAL, "theta must be above 1");
  if (!(c.factor >= 1.0) || !std::isfinite(c.factor)) return host_fail(M3G_EINVAL, "factor must be at least 1");
  if (!(c.magnitude >= 0.0) || !std::isfinite(c.magnitude)) return host_fail(M3G_EINVAL, "magnitude must not be negative");
  if (c.scaling == M3G_ROPE_NONE && c.factor != 1.0) return host_fail(M3G_EINVAL, "a factor needs a scaling");
  if (c.scaling == M3G_ROPE_NTK && c.rot_dim < 4) return host_fail(M3G_EINVAL, "NTK scaling needs rot_dim >= 4");
  if (c.scaling == M3G_ROPE_YARN || c.scaling == M3G_ROPE_LLAMA3) {
    if (!c.orig_ctx || c.orig_ctx > (1ull << 40)) return host_fail(M3G_EINVAL, "the scaling needs orig_ctx");
    const double lo = c.scaling == M3G_ROPE_YARN ? c.beta_slow : c.low_freq;
    const double hi = c.scaling == M3G_ROPE_YARN ? c.beta_fast : c.high_freq;
    if (!(lo > 0.0) || !(hi > lo) || !std::isfinite(hi))
      return host_fail(M3G_EINVAL, "the scaling's bounds must be positive and rising");
  }
  auto* r = new (std::nothrow) m3g_rope();
  if (!r) return host_fail(M3G_ENOMEM, "rope plan");
  r->cfg = c;
  const double pi2 = 6.283185307179586476925286766559;
  const double d = c.rot_dim;
  const double theta = c.scaling == M3G_ROPE_NTK ? c.theta * std::pow(c.factor, d / (d - 2.0)) : c.theta;
  double low = 0.0, high = 0.0;
  if (c.scaling == M3G_ROPE_YARN) {
    // pair index at which the original context holds `turns` turns
    auto at = [&](double turns) {
      return d * std::log(static_cast<double>(c.orig_ctx) / (turns * pi2)) / (2.0 * std::log(theta));
    };
    low = std::fmax(std::floor(at(c.beta_fast)), 0.0);
    high = std::fmin(std::ceil(at(c.beta_slow)), d - 1.0);
  }
  for (uint32_t i = 0; i < c.rot_dim / 2; ++i) {
    double f = std::pow(theta, -2.0 * i / d);
    if (c.scaling == M3G_ROPE_LINEAR) {
      f /= c.factor;
    } else if (c.scaling == M3G_ROPE_YARN) {
      const double ramp = std::fmin(1.0, std::fmax(0.0, (i - low) / std::fmax(high - low, 0.001)));
      f = f / c.factor * ramp + f * (1.0 - ramp);
    } else if (c.scaling == M3G_ROPE_LLAMA3) {
      const double turns = static_cast<double>(c.orig_ctx) * f / pi2;
      const double w = std::fmin(1.0, std::fmax(0.0, (turns - c.low_freq) / (c.high_freq - c.low_freq)));
      f = (1.0 - w) * f / c.factor + w * f;
    }
    r->turn[i] = static_cast<unsigned long long>(std::ldexp(f / pi2, 64));  // f <= 1: below 0.16 turns
  }
  r->magnitude = static_cast<float>(c.magnitude > 0.0 ? c.magnitude
                                    : c.scaling == M3G_ROPE_YARN ? 0.1 * std::log(c.factor) + 1.0 : 1.0);
  *out = r;
  return M3G_OK;
}

M3G_API void m3g_rope_destroy(m3g_rope* rope) { delete rope; }

M3G_API int m3g_rope_dev(const m3g_rope* rope, uint32_t dtype, const int32_t* positions, uint64_t n_tokens,
                         const m3g_rope_rows* q, const m3g_rope_rows* k, int inverse, void* stream) {
  using m3g::host_fail;
  if (!rope || !q) return host_fail(M3G_EINVAL, "null argument");
  const int size = m3g::act_size(dtype);
  if (!size) return host_fail(M3G_EINVAL, "rope: dtype %u (F32, F16 and BF16 are supported)", dtype);
  if (n_tokens >= (1ull << 31)) return host_fail(M3G_EINVAL, "too many tokens");
  m3g::RopeArgs a{};
  const int hd = static_cast<int>(rope->cfg.head_dim), rot = static_cast<int>(rope->cfg.rot_dim);
  bool vec = rot * size / 2 % (rope->cfg.interleaved ? 8 : 16) == 0 && (hd - rot) * size % 16 == 0;
  uint64_t heads = 0;
  for (int i = 0; i < (k ? 2 : 1); ++i) {
    const m3g_rope_rows& r = i ? *k : *q;
    if (r.heads > (1u << 20)) return host_fail(M3G_EINVAL, "too many heads");
    if (r.heads && n_tokens && (!r.x || !r.y)) return host_fail(M3G_EINVAL, "null rows");
    if (r.x_token_stride < 0 || r.x_head_stride < 0 || r.y_token_stride < 0 || r.y_head_stride < 0)
      return host_fail(M3G_EINVAL, "negative stride");
    if (r.x == r.y && (r.x_token_stride != r.y_token_stride || r.x_head_stride != r.y_head_stride))
      return host_fail(M3G_EINVAL, "rows turned in place need the same strides");
    if ((n_tokens > 1 && r.heads && r.y_token_stride < hd) || (r.heads > 1 && r.y_head_stride < hd))
      return host_fail(M3G_EINVAL, "result rows overlap");
    vec = vec && m3g::rows_aligned(r.x, r.x_token_stride, r.x_head_stride, size) &&
          m3g::rows_aligned(r.y, r.y_token_stride, r.y_head_stride, size);
    a.r[i] = r;
    heads += r.heads;
  }
  if (!n_tokens || !heads) return M3G_OK;
  if (!positions) return host_fail(M3G_EINVAL, "null positions");
  a.positions = positions;
  a.heads = static_cast<int>(heads);
  a.heads0 = static_cast<int>(q->heads);
  a.head_dim = hd;
  a.rot = rot;
  a.inverse = inverse != 0;
  a.magnitude = rope->magnitude;
  for (int i = 0; i < rot / 2; ++i) a.turn[i] = rope->turn[i];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return host_fail(M3G_ECUDA, "no CUDA device");
  const cudaStream_t st = m3g::serve_stream(stream);
  const bool inter = rope->cfg.interleaved != 0;
  const unsigned grid = static_cast<unsigned>(n_tokens);
  const cudaError_t e = dtype == M3G_DTYPE_F32   ? m3g::launch_rope<float>(a, vec, inter, grid, st)
                        : dtype == M3G_DTYPE_F16 ? m3g::launch_rope<__half>(a, vec, inter, grid, st)
                                                 : m3g::launch_rope<__nv_bfloat16>(a, vec, inter, grid, st);
  if (e != cudaSuccess) return host_fail(M3G_ECUDA, "k_rope: %s", cudaGetErrorString(e));
  return M3G_OK;
}

}  // extern "C"
