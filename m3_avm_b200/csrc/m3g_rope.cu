// m3g_rope.cu -- rotary positions of q and k rows.
//
// Pair i of a token at position p turns by the angle p * f_i.  The plan holds
// f_i / 2pi as a 64-bit fraction of a turn, so p * f_i modulo one turn is one
// wrapping 64-bit integer product without a range reduction.  What it is off by: f_i
// is a double, right to some units (|p| 2^-53 turns); the product's top 32 bits become
// sincospif's f32 argument (2^-26 turns).  An f32 product is off by 0.06 rad at
// position 10^6 already.  cos and sin are worked out once per token; all its heads
// share them through shared memory.
//
// Bound: HBM (each element read and written once; 16384 BF16 tokens of 72 heads of 128
// 116 us, 5.2 TB/s; 4099 F32 tokens of 40 heads of 64 14.5 us, 5.8 TB/s).  A CTA takes a run of tokens.
// Each thread copies its own pieces of the next kRopeDepth tokens into its own
// places in shared memory (cp.async; nobody else reads them, so no barrier), so
// that 3 x 64 bytes a thread are in flight without registers; the angles of as many tokens as there
// are threads for (one thread per pair) are worked out together, between two
// barriers, since that chain of some 1000 cycles is what a token waits for.
#include <algorithm>
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

constexpr int kRopeThreads = 512;  // at most; a token takes as few as hold it in U units a thread
constexpr int kRopeDepth = 3;
constexpr int rope_units(bool inter) { return inter ? 4 : 2; }  // U: four vectors either way
constexpr int kMaxPairs = 128;

struct RopeArgs {
  const int32_t* positions;
  m3g_rope_rows r[2];
  long long n_tokens;
  int batch;             // tokens whose angles are worked out together
  int heads, heads0;     // rows of both tensors; of the first
  int head_dim, rot;
  int inverse;
  float magnitude;
  unsigned long long turn[kMaxPairs];
};

// A unit is two vectors of a head (half layout) or one (interleaved): V pairs,
// or, behind rot, values to copy.  A thread keeps its place in the head, ny
// heads apart; U units of a token are in flight.  What bounds the 16-bit types
// beside HBM is instructions, so loads and stores are the same for turned and
// copied units, and a thread that holds all of its token's units (ONCE, the
// usual case) keeps their addresses.
template <class T, int V, bool VEC, bool INTER, bool ONCE>
__global__ void __launch_bounds__(kRopeThreads, 2) k_rope(const __grid_constant__ RopeArgs a) {
  __shared__ float2 cs[2][kRopeThreads];
  constexpr int U = INTER ? 4 : 2;
  constexpr int S = INTER ? 2 * V : V;  // values of one vector
  struct alignas(VEC ? 16 : sizeof(T)) Vec { T t[S]; };
  const int tid = threadIdx.x, threads = blockDim.x, half = a.rot / 2;
  const int np = half / V, nt = (a.head_dim - a.rot + S - 1) / S;  // units of pairs; vectors behind them
  const int per = np + (INTER ? nt : (nt + 1) / 2);
  // units of a head over the threads, ny heads at once
  const bool fits = ONCE || per <= threads;
  const int ny = fits ? threads / per : 1;
  const int h0 = fits ? tid / per : 0;
  const int c0 = fits ? tid - h0 * per : tid;
  const bool active = h0 < ny && c0 < per;
  // Fields of q's or k's rows picked by value: a reference picked at run time
  // turns every access to the kernel's arguments into a load from memory.
  const int64_t xt0 = a.r[0].x_token_stride, xt1 = a.r[1].x_token_stride, xh0 = a.r[0].x_head_stride,
                xh1 = a.r[1].x_head_stride, yt0 = a.r[0].y_token_stride, yt1 = a.r[1].y_token_stride,
                yh0 = a.r[0].y_head_stride, yh1 = a.r[1].y_head_stride;
  const T *x0 = static_cast<const T*>(a.r[0].x), *x1 = static_cast<const T*>(a.r[1].x);
  T *y0 = static_cast<T*>(a.r[0].y), *y1 = static_cast<T*>(a.r[1].y);
  Vec lo[U], hi[INTER ? 1 : U];
  float2 turn[V];
  // where unit c's vectors lie in a head; the second of a half-layout unit may not exist
  auto lo_at = [&](int c) { return INTER || c < np ? c * S : a.rot + 2 * (c - np) * S; };
  auto hi_at = [&](int c) { return c < np ? half + c * S : a.rot + (2 * (c - np) + 1) * S; };
  auto has_hi = [&](int c) { return !INTER && (c < np || 2 * (c - np) + 1 < nt); };
  auto get = [&](const T* x, int c, int k) {  // x: the head
    lo[k] = *reinterpret_cast<const Vec*>(x + lo_at(c));
    if (has_hi(c)) hi[INTER ? 0 : k] = *reinterpret_cast<const Vec*>(x + hi_at(c));
  };
  auto put = [&](T* y, int c, int k) {
    if (c < np) {
      float p[S], q[S];
      unpack_act<T, S>(lo[k].t, p);
      if (!INTER) unpack_act<T, S>(hi[INTER ? 0 : k].t, q);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float& f = INTER ? p[2 * i < S ? 2 * i : 0] : p[i];
        float& g = INTER ? p[2 * i + 1 < S ? 2 * i + 1 : 0] : q[i];
        const float f0 = f, g0 = g;
        f = f0 * turn[i].x - g0 * turn[i].y;
        g = f0 * turn[i].y + g0 * turn[i].x;
      }
      pack_act<T, S>(lo[k].t, p);
      if (!INTER) pack_act<T, S>(hi[INTER ? 0 : k].t, q);
    }
    *reinterpret_cast<Vec*>(y + lo_at(c)) = lo[k];
    if (has_hi(c)) *reinterpret_cast<Vec*>(y + hi_at(c)) = hi[INTER ? 0 : k];
  };
  auto from = [&](long long tok, int h) {
    return h >= a.heads0 ? x1 + tok * xt1 + (h - a.heads0) * xh1 : x0 + tok * xt0 + h * xh0;
  };
  auto to = [&](long long tok, int h) {
    return h >= a.heads0 ? y1 + tok * yt1 + (h - a.heads0) * yh1 : y0 + tok * yt0 + h * yh0;
  };
  const long long t_end = (blockIdx.x + 1) * a.n_tokens / gridDim.x;
  long long tok = blockIdx.x * a.n_tokens / gridDim.x;
  constexpr bool RING = ONCE && VEC;
  extern __shared__ __align__(16) uint8_t ring[];  // [depth][4][threads] vectors, each thread's its own
  const T* px[U];  // this thread's heads, where it has them at once: of the next token to copy
  T* py[U];        // of the token at hand
  auto slot = [&](int d, int v) { return reinterpret_cast<Vec*>(ring + ((d * 4 + v) * threads + tid) * 16); };
  auto fetch = [&](long long t, int d) {  // the thread's units of token t
    if (active && t < t_end) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int h = h0 + k * ny;
        if (h >= a.heads) break;
        cp16(slot(d, INTER ? k : 2 * k), px[k] + lo_at(c0), 16);
        if (has_hi(c0)) cp16(slot(d, INTER ? k : 2 * k + 1), px[k] + hi_at(c0), 16);
        px[k] += h >= a.heads0 ? xt1 : xt0;
      }
    }
    cp_commit();
  };
  if (ONCE && active) {
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (h0 + k * ny < a.heads) {
        px[k] = from(tok, h0 + k * ny);
        py[k] = to(tok, h0 + k * ny);
        if (!RING) get(px[k], c0, k);
      }
  }
  if (RING) {
#pragma unroll
    for (int d = 0; d < kRopeDepth; ++d) fetch(tok + d, d);
  }
  int depth = 0;
  const int my_token = tid / half, my_pair = tid - my_token * half;  // angle of this thread
  const unsigned long long my_turn = my_token < a.batch ? a.turn[my_pair] : 0;
  auto angle = [&](int pos, unsigned long long per_position) {
    const long long p = a.inverse ? -static_cast<long long>(pos) : static_cast<long long>(pos);
    const unsigned long long turns = static_cast<unsigned long long>(p) * per_position;
    float s, c;
    // the top 32 bits as a signed fraction of a turn, in half turns
    sincospif(static_cast<float>(static_cast<int>(turns >> 32)) * 0x1p-31f, &s, &c);
    return make_float2(c * a.magnitude, s * a.magnitude);
  };
  auto position = [&](long long t) { return my_token < a.batch && t + my_token < t_end ? a.positions[t + my_token] : 0; };
  int pos = position(tok);
  for (int buf = 0; tok < t_end; buf ^= 1) {
    if (my_token < a.batch) cs[buf][tid] = angle(pos, my_turn);
    if (threads < half)  // more pairs than threads (batch 1)
      for (int i = tid + threads; i < half; i += threads) cs[buf][i] = angle(a.positions[tok], a.turn[i]);
    pos = position(tok + a.batch);
    __syncthreads();  // the readers of two batches ago are done with this buffer
    const long long b_end = min(t_end, tok + a.batch);
    if (!active) {
      tok = b_end;
      continue;
    }
    for (int b = 0; tok < b_end; ++tok, ++b) {
      const float2* turns = cs[buf] + b * half;
      if constexpr (ONCE) {
        if (c0 < np) {
#pragma unroll
          for (int i = 0; i < V; ++i) turn[i] = turns[c0 * V + i];
        }
        if (RING) cp_wait<kRopeDepth - 1>();
#pragma unroll
        for (int k = 0; k < U; ++k) {
          const int h = h0 + k * ny;
          if (h >= a.heads) break;
          if (RING) {
            lo[k] = *slot(depth, INTER ? k : 2 * k);
            if (has_hi(c0)) hi[INTER ? 0 : k] = *slot(depth, INTER ? k : 2 * k + 1);
          }
          put(py[k], c0, k);
          py[k] += h >= a.heads0 ? yt1 : yt0;
          if (!RING) {
            px[k] += h >= a.heads0 ? xt1 : xt0;
            if (tok + 1 < t_end) get(px[k], c0, k);
          }
        }
        if (RING) {
          fetch(tok + kRopeDepth, depth);
          depth = depth + 1 == kRopeDepth ? 0 : depth + 1;
        }
      } else {
      for (int c = c0; c < per; c += fits ? per : threads) {
        if (c < np) {
#pragma unroll
          for (int i = 0; i < V; ++i) turn[i] = turns[c * V + i];
        }
        for (int h = h0; h < a.heads; h += U * ny) {
#pragma unroll
          for (int k = 0; k < U; ++k)
            if (h + k * ny < a.heads) get(from(tok, h + k * ny), c, k);
#pragma unroll
          for (int k = 0; k < U; ++k)
            if (h + k * ny < a.heads) put(to(tok, h + k * ny), c, k);
        }
      }
      }
    }
  }
}

template <class Kern>
cudaError_t launch_ring(Kern kern, dim3 grid, unsigned threads, cudaStream_t st, const RopeArgs& a) {
  const size_t smem = static_cast<size_t>(kRopeDepth) * 64 * threads;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRopeDepth * 64 * kRopeThreads);
  return e == cudaSuccess ? serve_launch(kern, grid, dim3(threads), smem, st, false, a) : e;
}

template <class T, bool INTER>
cudaError_t launch_rope_t(RopeArgs a, bool vec, int sms, cudaStream_t st) {
  // 16-byte vectors: V pairs are two of them (half layout), or one (interleaved)
  constexpr int V = INTER ? 8 / sizeof(T) : 16 / sizeof(T);
  const int v = vec ? V : 1, s = INTER ? 2 * v : v;
  const long long tail = (a.head_dim - a.rot + s - 1) / s;
  const long long units = a.rot / 2 / v + (INTER ? tail : (tail + 1) / 2);  // per head
  const long long want = units * ((a.heads + rope_units(INTER) - 1) / rope_units(INTER));
  const unsigned threads = static_cast<unsigned>(std::min<long long>(kRopeThreads, (want + 31) / 32 * 32));
  // as many CTAs as are resident at 64 registers a thread
  const dim3 grid(static_cast<unsigned>(std::min<long long>(a.n_tokens, static_cast<long long>(sms) * (1024 / threads))));
  a.batch = static_cast<int>(std::max<long long>(1, std::min<long long>(threads / (a.rot / 2), a.n_tokens / grid.x)));
  // whether a thread's units are all that it has of a token
  const bool once = units <= threads && rope_units(INTER) * (threads / units) >= a.heads;
  if (vec)
    return once ? launch_ring(k_rope<T, V, true, INTER, true>, grid, threads, st, a)
                : serve_launch(k_rope<T, V, true, INTER, false>, grid, dim3(threads), 0, st, false, a);
  return once ? serve_launch(k_rope<T, 1, false, INTER, true>, grid, dim3(threads), 0, st, false, a)
              : serve_launch(k_rope<T, 1, false, INTER, false>, grid, dim3(threads), 0, st, false, a);
}

template <class T>
cudaError_t launch_rope(const RopeArgs& a, bool vec, bool inter, int sms, cudaStream_t st) {
  return inter ? launch_rope_t<T, true>(a, vec, sms, st) : launch_rope_t<T, false>(a, vec, sms, st);
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
    if (m3g::misaligned(r.x, size) || m3g::misaligned(r.y, size))
      return host_fail(M3G_EINVAL, "rows not aligned to their type");
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
  if (!positions || m3g::misaligned(positions, 4)) return host_fail(M3G_EINVAL, "positions null or not 4-byte aligned");
  a.positions = positions;
  a.heads = static_cast<int>(heads);
  a.heads0 = static_cast<int>(q->heads);
  a.head_dim = hd;
  a.rot = rot;
  a.inverse = inverse != 0;
  a.magnitude = rope->magnitude;
  for (int i = 0; i < rot / 2; ++i) a.turn[i] = rope->turn[i];
  a.n_tokens = static_cast<long long>(n_tokens);
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return host_fail(M3G_ECUDA, "no CUDA device");
  const cudaStream_t st = m3g::serve_stream(stream);
  const bool inter = rope->cfg.interleaved != 0;
  const cudaError_t e = dtype == M3G_DTYPE_F32   ? m3g::launch_rope<float>(a, vec, inter, sms, st)
                        : dtype == M3G_DTYPE_F16 ? m3g::launch_rope<__half>(a, vec, inter, sms, st)
                                                 : m3g::launch_rope<__nv_bfloat16>(a, vec, inter, sms, st);
  if (e != cudaSuccess) return host_fail(M3G_ECUDA, "k_rope: %s", cudaGetErrorString(e));
  return M3G_OK;
}

}  // extern "C"
