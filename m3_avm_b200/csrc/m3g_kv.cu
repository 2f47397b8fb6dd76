// m3g_kv.cu -- the paged, quantised KV cache: writing new rows and reading
// rows back.
//
// A block is 32 consecutive values of a row: d = f16(max|x| / 127) (Q4_0: 7),
// code = round(x / d), halves away from zero, clamped -- the rules of
// quantize_q8_0 / quantize_q4_0 (src/quant.rs:206-264), whose f32 quotient
// x / d is kept to the bit: the quotient from the reciprocal decides unless it
// lies within 2^-12 of a border between two codes, where a correctly rounded
// division does (one value in about 2000).  A block with a value that is not
// finite, or whose scale passes the f16 range, gets the scale NaN and codes
// that stand for 0, so that it reads back as NaN.
//
// Four threads share a block, 8 values each; a thread's 8 values are one
// 16-byte load (two for f32) and its codes one 8-byte store.  Both kernels are
// bound by HBM; a CTA takes kKvTokens tokens, whose places its first threads
// look up in the page table once.
#include "m3g_serve.cuh"

namespace m3g {

int kv_check(const m3g_kv_layout* l) {
  if (!l) return host_fail(M3G_EINVAL, "null cache layout");
  if (l->dtype != M3G_DTYPE_Q8_0 && l->dtype != M3G_DTYPE_Q4_0)
    return host_fail(M3G_EINVAL, "cache dtype %u (Q8_0 and Q4_0 are supported)", l->dtype);
  if (l->head_dim != 64 && l->head_dim != 128)
    return host_fail(M3G_EINVAL, "cache head_dim %u (64 and 128 are supported)", l->head_dim);
  if (!l->n_layers || l->n_layers > 4096 || !l->n_kv_heads || l->n_kv_heads > 1024)
    return host_fail(M3G_EINVAL, "cache of %u layers, %u heads", l->n_layers, l->n_kv_heads);
  if (l->page_size < 16 || l->page_size > 1024 || (l->page_size & (l->page_size - 1)))
    return host_fail(M3G_EINVAL, "page size %u (a power of two, 16 .. 1024)", l->page_size);
  if (!l->n_pages || l->n_pages >= (1ull << 31))
    return host_fail(M3G_EINVAL, "cache of %llu pages", static_cast<unsigned long long>(l->n_pages));
  return M3G_OK;
}

int kv_batch_check(const m3g_kv_layout* l, const m3g_kv_batch* b) {
  if (!b) return host_fail(M3G_EINVAL, "null batch");
  if (b->n_seqs > (1u << 20) || b->n_tokens >= (1u << 31) || b->max_tokens >= (1u << 31) ||
      b->max_len >= (1u << 31) - 2048 || b->max_pages >= (1u << 31))
    return host_fail(M3G_EINVAL, "batch too large");
  if (b->n_seqs && b->n_tokens && (!b->q_start || !b->ctx_len || !b->page_table || !b->max_pages))
    return host_fail(M3G_EINVAL, "null batch array");
  (void)l;
  return M3G_OK;
}

int kv_planes(const m3g_kv_layout* l, const void* pool, uint32_t layer, KvPlanes* out) {
  if (int rc = kv_check(l)) return rc;
  if (layer >= l->n_layers) return host_fail(M3G_EINVAL, "layer %u of %u", layer, l->n_layers);
  if (!pool || reinterpret_cast<uintptr_t>(pool) % 16) return host_fail(M3G_EINVAL, "cache pool null or not 16-byte aligned");
  KvPlanes p{};
  p.kvh = static_cast<int>(l->n_kv_heads);
  p.hd = static_cast<int>(l->head_dim);
  p.cb = l->dtype == M3G_DTYPE_Q8_0 ? p.hd : p.hd / 2;
  p.sb = p.hd / 16;
  p.page_size = static_cast<int>(l->page_size);
  while ((1 << p.page_shift) < p.page_size) ++p.page_shift;
  p.n_pages = static_cast<int>(l->n_pages);
  const uint64_t rows = l->n_pages * l->n_kv_heads * l->page_size;
  uint8_t* base = const_cast<uint8_t*>(static_cast<const uint8_t*>(pool)) + layer * rows * 2 * (p.cb + p.sb);
  p.kc = base;
  p.ks = p.kc + rows * p.cb;
  p.vc = p.ks + rows * p.sb;
  p.vs = p.vc + rows * p.cb;
  *out = p;
  return M3G_OK;
}

namespace {

constexpr int kKvThreads = 256;
constexpr int kKvTokens = 8;  // tokens per CTA

struct KvIoArgs {
  KvPlanes p;
  m3g_kv_batch b;
  m3g_rows k, v;
  long long cap;
};

// round(x / d), halves away from zero, of the f32 quotient; inv = 1 / d.
__device__ __forceinline__ float code_of(float x, float d, float inv) {
  const float t = fabsf(x) * inv;
  float q = floorf(t + 0.5f);
  if (fabsf(t + 0.5f - rintf(t + 0.5f)) < 0x1p-12f) q = roundf(__fdiv_rn(fabsf(x), d));
  return copysignf(q, x);
}

// Places of the CTA's tokens: page * page_size + offset, -1 for none.
__device__ __forceinline__ void find_places(const KvIoArgs& a, int t0, long long (&place)[kKvTokens]) {
  const int tid = threadIdx.x;
  if (tid < kKvTokens) {
    const int t = t0 + tid;
    long long at = -1;
    if (t < static_cast<int>(a.b.n_tokens)) {
      int lo = 0, hi = static_cast<int>(a.b.n_seqs);  // the last s with q_start[s] <= t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.b.q_start[mid] <= t) lo = mid;
        else hi = mid;
      }
      bool bad = false;
      const SeqView s = seq_view(a.b, a.cap, lo, &bad);
      if (t >= s.q0 && t - s.q0 < s.n) {
        const int pos = s.ctx + (t - s.q0);
        const int page = a.b.page_table[static_cast<long long>(lo) * a.b.max_pages + (pos >> a.p.page_shift)];
        if (page >= 0 && page < a.p.n_pages)
          at = kv_row(a.p, page, 0, pos & (a.p.page_size - 1));
        else
          atomicOr(a.p.status, kStatusBadPage);
      }
      if (bad) atomicOr(a.p.status, kStatusBadBatch);
    }
    place[tid] = at;
  }
  __syncthreads();
}

template <class T, bool Q8, bool VEC>
__global__ void __launch_bounds__(kKvThreads) k_kv_write(const __grid_constant__ KvIoArgs a) {
  __shared__ long long place[kKvTokens];
  const int t0 = blockIdx.x * kKvTokens;
  find_places(a, t0, place);
  const int octs = a.p.hd / 8;                      // threads per row
  const int per_token = 2 * a.p.kvh * octs;         // K heads, then V heads
  const int units = kKvTokens * per_token;          // a multiple of 4: the threads of a block stay together
  for (int u = threadIdx.x; u < units; u += kKvThreads) {
    const int ti = u / per_token, w = u - ti * per_token;
    const int row = w / octs, oct = w - row * octs;
    const bool is_v = row >= a.p.kvh;
    const int head = is_v ? row - a.p.kvh : row;
    const unsigned quad = 0xFu << (threadIdx.x & 28);
    if (place[ti] < 0) continue;  // the same for all threads of a block
    const m3g_rows& r = is_v ? a.v : a.k;
    const T* src = static_cast<const T*>(r.p) + (t0 + ti) * r.token_stride + head * r.head_stride + oct * 8;
    float x[8];
    load_act<T, 8, VEC>(src, x);
    float most = 0.f;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      most = fmaxf(most, fabsf(x[i]));
      finite = finite && fabsf(x[i]) <= 3.402823466e38f;
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) most = fmaxf(most, __shfl_xor_sync(quad, most, o));
    finite = (__ballot_sync(quad, finite) & quad) == quad;
    __half dh = __float2half_rn(__fdiv_rn(most, Q8 ? 127.f : 7.f));
    const float d = __half2float(dh);
    const bool ok = finite && d <= 65504.f;
    if (!ok) dh = __ushort_as_half(0x7FFF);
    const float inv = ok && d > 0.f ? __frcp_rn(d) : 0.f;
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float q = inv > 0.f ? code_of(x[i], d, inv) : 0.f;
      q = Q8 ? fminf(fmaxf(q, -127.f), 127.f) + 128.f : fminf(fmaxf(q, -8.f), 7.f) + 8.f;
      c[i] = static_cast<uint32_t>(q);
    }
    const long long at = place[ti] + static_cast<long long>(head) * a.p.page_size;
    uint8_t* codes = is_v ? a.p.vc : a.p.kc;
    if (Q8) {
      const uint32_t w0 = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
      const uint32_t w1 = c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24;
      *reinterpret_cast<uint2*>(codes + at * a.p.cb + oct * 8) = make_uint2(w0, w1);
    } else {
      uint32_t w0 = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
      uint32_t w1 = c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24;
      const uint32_t h0 = __shfl_xor_sync(quad, w0, 2), h1 = __shfl_xor_sync(quad, w1, 2);
      if ((oct & 2) == 0)  // the block's first 16 values are the low nibbles
        *reinterpret_cast<uint2*>(codes + at * a.p.cb + (oct >> 2) * 16 + (oct & 1) * 8) =
            make_uint2(w0 | h0 << 4, w1 | h1 << 4);
    }
    if ((oct & 3) == 0)
      reinterpret_cast<__half*>((is_v ? a.p.vs : a.p.ks) + at * a.p.sb)[oct >> 2] = dh;
  }
}

template <class T, bool Q8, bool VEC>
__global__ void __launch_bounds__(kKvThreads) k_kv_read(const __grid_constant__ KvIoArgs a) {
  __shared__ long long place[kKvTokens];
  const int t0 = blockIdx.x * kKvTokens;
  find_places(a, t0, place);
  const int octs = a.p.hd / 8, per_token = 2 * a.p.kvh * octs, units = kKvTokens * per_token;
  for (int u = threadIdx.x; u < units; u += kKvThreads) {
    const int ti = u / per_token, w = u - ti * per_token;
    const int row = w / octs, oct = w - row * octs;
    const bool is_v = row >= a.p.kvh;
    const int head = is_v ? row - a.p.kvh : row;
    if (place[ti] < 0) continue;
    const long long at = place[ti] + static_cast<long long>(head) * a.p.page_size;
    const uint8_t* codes = (is_v ? a.p.vc : a.p.kc) + at * a.p.cb;
    const float d =
        __half2float(reinterpret_cast<const __half*>((is_v ? a.p.vs : a.p.ks) + at * a.p.sb)[oct >> 2]);
    float x[8];
    uint2 q;
    if (Q8) {
      q = *reinterpret_cast<const uint2*>(codes + oct * 8);
    } else {
      q = *reinterpret_cast<const uint2*>(codes + (oct >> 2) * 16 + (oct & 1) * 8);
      const int sh = (oct & 2) ? 4 : 0;
      q.x = q.x >> sh & 0x0F0F0F0Fu;
      q.y = q.y >> sh & 0x0F0F0F0Fu;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t b = ((i < 4 ? q.x : q.y) >> (8 * (i & 3))) & 0xFFu;
      x[i] = (static_cast<float>(b) - (Q8 ? 128.f : 8.f)) * d;
    }
    const m3g_rows& r = is_v ? a.v : a.k;
    store_act<T, 8, VEC>(static_cast<T*>(r.p) + (t0 + ti) * r.token_stride + head * r.head_stride + oct * 8, x);
  }
}

template <class T, bool Q8>
cudaError_t launch_kv(const KvIoArgs& a, bool vec, bool write, cudaStream_t st) {
  const dim3 grid((a.b.n_tokens + kKvTokens - 1) / kKvTokens), block(kKvThreads);
  if (write)
    return vec ? serve_launch(k_kv_write<T, Q8, true>, grid, block, 0, st, false, a)
               : serve_launch(k_kv_write<T, Q8, false>, grid, block, 0, st, false, a);
  return vec ? serve_launch(k_kv_read<T, Q8, true>, grid, block, 0, st, false, a)
             : serve_launch(k_kv_read<T, Q8, false>, grid, block, 0, st, false, a);
}

int kv_io(const m3g_kv_layout* l, const void* pool, uint32_t layer, const m3g_kv_batch* b, uint32_t dtype,
          const m3g_rows* k, const m3g_rows* v, void* stream, bool write) {
  KvIoArgs a{};
  if (int rc = kv_planes(l, pool, layer, &a.p)) return rc;
  if (int rc = kv_batch_check(l, b)) return rc;
  if (!k || !v) return host_fail(M3G_EINVAL, "null argument");
  const int size = act_size(dtype);
  if (!size) return host_fail(M3G_EINVAL, "cache rows of dtype %u (F32, F16 and BF16 are supported)", dtype);
  bool vec = true;
  for (const m3g_rows* r : {k, v}) {
    if (!r->p && b->n_tokens) return host_fail(M3G_EINVAL, "null rows");
    if (r->token_stride < 0 || r->head_stride < 0) return host_fail(M3G_EINVAL, "negative stride");
    if (!write && ((b->n_tokens > 1 && r->token_stride < a.p.hd) || (a.p.kvh > 1 && r->head_stride < a.p.hd)))
      return host_fail(M3G_EINVAL, "result rows overlap");
    vec = vec && rows_aligned(r->p, r->token_stride, r->head_stride, size);
  }
  if (!b->n_tokens || !b->n_seqs) return M3G_OK;
  int dev = 0;
  if (int rc = serve_device(&dev, &a.p.status)) return rc;
  a.b = *b;
  a.k = *k;
  a.v = *v;
  a.cap = seq_cap(*b, l->page_size);
  const cudaStream_t st = serve_stream(stream);
  const bool q8 = l->dtype == M3G_DTYPE_Q8_0;
  cudaError_t e;
  if (dtype == M3G_DTYPE_F32) e = q8 ? launch_kv<float, true>(a, vec, write, st) : launch_kv<float, false>(a, vec, write, st);
  else if (dtype == M3G_DTYPE_F16) e = q8 ? launch_kv<__half, true>(a, vec, write, st) : launch_kv<__half, false>(a, vec, write, st);
  else e = q8 ? launch_kv<__nv_bfloat16, true>(a, vec, write, st) : launch_kv<__nv_bfloat16, false>(a, vec, write, st);
  if (e != cudaSuccess) return host_fail(M3G_ECUDA, "%s: %s", write ? "k_kv_write" : "k_kv_read", cudaGetErrorString(e));
  return M3G_OK;
}

}  // namespace
}  // namespace m3g

extern "C" {

M3G_API int m3g_kv_bytes(const m3g_kv_layout* l, uint64_t* out) {
  if (!out) return m3g::host_fail(M3G_EINVAL, "null argument");
  *out = 0;
  if (int rc = m3g::kv_check(l)) return rc;
  const uint64_t row = 2ull * ((l->dtype == M3G_DTYPE_Q8_0 ? l->head_dim : l->head_dim / 2) + l->head_dim / 16);
  *out = l->n_layers * l->n_pages * l->n_kv_heads * l->page_size * row;
  if (*out / row / l->page_size / l->n_kv_heads / l->n_layers != l->n_pages || *out >= (1ull << 46)) {
    *out = 0;
    return m3g::host_fail(M3G_EINVAL, "cache too large");
  }
  return M3G_OK;
}

M3G_API int m3g_kv_write_dev(const m3g_kv_layout* layout, void* pool, uint32_t layer, const m3g_kv_batch* batch,
                             uint32_t dtype, const m3g_rows* k, const m3g_rows* v, void* stream) {
  return m3g::kv_io(layout, pool, layer, batch, dtype, k, v, stream, true);
}

M3G_API int m3g_kv_read_dev(const m3g_kv_layout* layout, const void* pool, uint32_t layer, const m3g_kv_batch* batch,
                            uint32_t dtype, const m3g_rows* k, const m3g_rows* v, void* stream) {
  return m3g::kv_io(layout, pool, layer, batch, dtype, k, v, stream, false);
}

}  // extern "C"
