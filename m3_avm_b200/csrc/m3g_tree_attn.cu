// m3g_tree_attn.cu -- attention of drafted tokens over the quantised KV cache.
//
// out = softmax(scale * q K^T + mask) V per (token, query head), positions in
// order with a running maximum and sum.  One CTA per (token, query head); its
// warps take every fourth position, each lane HD / 32 values of the row, and
// their partial results join in shared memory.
#include <cmath>

#include "m3g_device.cuh"
#include "m3g_serve.cuh"

namespace m3g {
namespace {

struct TreeArgs {
  KvPlanes p;
  m3g_kv_batch b;
  m3g_rows q, out;
  const uint32_t* mask;
  long long cap;
  int mask_words, n_heads, group;
  float scale;
};

template <class T, int HD, bool Q8>
__global__ void __launch_bounds__(128) k_tree_attn(const __grid_constant__ TreeArgs a) {
  constexpr int DPL = HD / 32;
  __shared__ float part[4][HD + 2];
  const int t = blockIdx.x, head = blockIdx.y, kvhead = head / a.group;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int lo = 0, hi = static_cast<int>(a.b.n_seqs);
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.b.q_start[mid] <= t) lo = mid;
    else hi = mid;
  }
  bool bad = false;
  const SeqView s = seq_view(a.b, a.cap, lo, &bad);
  if (bad && threadIdx.x == 0) atomicOr(a.p.status, kStatusBadBatch);
  if (t < s.q0 || t - s.q0 >= s.n) return;
  const int j = t - s.q0, len = s.ctx + s.n;
  const T* q = static_cast<const T*>(a.q.p) + t * a.q.token_stride + head * a.q.head_stride;
  float qv[DPL], o[DPL], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < DPL; ++i) {
    qv[i] = Act<T>::to(q[lane * DPL + i]) * a.scale;
    o[i] = 0.f;
  }
  auto value = [&](const uint8_t* codes, const uint8_t* scales, long long row, int e) {
    const float d = __half2float(reinterpret_cast<const __half*>(scales + row * a.p.sb)[e / 32]);
    if (Q8) return (static_cast<float>(codes[row * a.p.cb + e]) - 128.f) * d;
    const uint32_t c = codes[row * a.p.cb + e / 32 * 16 + e % 16];
    return (static_cast<float>(e & 16 ? c >> 4 : c & 15u) - 8.f) * d;
  };
  for (int pos = warp; pos < len; pos += 4) {
    const int i = pos - s.ctx;
    if (i >= 0 && !(a.mask ? a.mask[static_cast<long long>(t) * a.mask_words + (i >> 5)] >> (i & 31) & 1u : i <= j))
      continue;
    const int page = a.b.page_table[static_cast<long long>(lo) * a.b.max_pages + (pos >> a.p.page_shift)];
    const bool there = page >= 0 && page < a.p.n_pages;
    if (!there && lane == 0) atomicOr(a.p.status, kStatusBadPage);
    const long long row = there ? kv_row(a.p, page, kvhead, pos & (a.p.page_size - 1)) : 0;
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < DPL; ++e) dot += there ? qv[e] * value(a.p.kc, a.p.ks, row, lane * DPL + e) : 0.f;
    dot = warp_sum(dot);
    const float mn = fmaxf(m, dot);
    const float f = m == -INFINITY ? 0.f : expf(m - mn), w = expf(dot - mn);
    l = l * f + w;
#pragma unroll
    for (int e = 0; e < DPL; ++e) o[e] = o[e] * f + (there ? w * value(a.p.vc, a.p.vs, row, lane * DPL + e) : 0.f);
    m = mn;
  }
  if (lane == 0) {
    part[warp][HD] = m;
    part[warp][HD + 1] = l;
  }
#pragma unroll
  for (int e = 0; e < DPL; ++e) part[warp][lane * DPL + e] = o[e];
  __syncthreads();
  if (threadIdx.x >= HD) return;
  float M = -INFINITY, L = 0.f, O = 0.f;
  for (int w = 0; w < 4; ++w) M = fmaxf(M, part[w][HD]);
  for (int w = 0; w < 4; ++w) {
    if (part[w][HD + 1] == 0.f) continue;
    const float f = expf(part[w][HD] - M);
    L += f * part[w][HD + 1];
    O += f * part[w][threadIdx.x];
  }
  static_cast<T*>(a.out.p)[t * a.out.token_stride + head * a.out.head_stride + threadIdx.x] =
      Act<T>::from(L == 0.f ? 0.f : O / L);
}

template <class T, int HD, bool Q8>
cudaError_t launch_tree(const TreeArgs& a, cudaStream_t st) {
  return serve_launch(k_tree_attn<T, HD, Q8>, dim3(a.b.n_tokens, a.n_heads), dim3(128), 0, st, false, a);
}
template <class T>
cudaError_t launch_tree_t(const TreeArgs& a, bool q8, cudaStream_t st) {
  if (a.p.hd == 64) return q8 ? launch_tree<T, 64, true>(a, st) : launch_tree<T, 64, false>(a, st);
  return q8 ? launch_tree<T, 128, true>(a, st) : launch_tree<T, 128, false>(a, st);
}

int check_heads(const m3g_kv_layout* l, uint32_t n_heads) {
  if (!n_heads || n_heads > 32768 || n_heads % l->n_kv_heads)
    return host_fail(M3G_EINVAL, "%u query heads over %u KV heads", n_heads, l->n_kv_heads);
  return M3G_OK;
}

}  // namespace
}  // namespace m3g

extern "C" {

M3G_API int m3g_tree_attn_workspace(const m3g_kv_layout* l, uint32_t n_heads, uint64_t* out) {
  if (!out) return m3g::host_fail(M3G_EINVAL, "null argument");
  *out = 0;
  if (int rc = m3g::kv_check(l)) return rc;
  if (int rc = m3g::check_heads(l, n_heads)) return rc;
  *out = 16;
  return M3G_OK;
}

M3G_API int m3g_tree_attn_dev(const m3g_kv_layout* l, const void* pool, uint32_t layer, const m3g_kv_batch* b,
                              uint32_t dtype, const m3g_rows* q, uint32_t n_heads, const uint32_t* mask,
                              uint32_t mask_words, float scale, const m3g_rows* out, void* workspace,
                              uint64_t workspace_bytes, void* stream) {
  using namespace m3g;
  TreeArgs a{};
  if (int rc = kv_planes(l, pool, layer, &a.p)) return rc;
  if (int rc = check_heads(l, n_heads)) return rc;
  if (int rc = kv_batch_check(l, b)) return rc;
  if (!q || !out) return host_fail(M3G_EINVAL, "null argument");
  const int size = act_size(dtype);
  if (!size) return host_fail(M3G_EINVAL, "attention of dtype %u (F32, F16 and BF16 are supported)", dtype);
  for (const m3g_rows* r : {q, out}) {
    if (!r->p && b->n_tokens) return host_fail(M3G_EINVAL, "null rows");
    if (r->token_stride < 0 || r->head_stride < 0) return host_fail(M3G_EINVAL, "negative stride");
  }
  if ((b->n_tokens > 1 && out->token_stride < a.p.hd) || (n_heads > 1 && out->head_stride < a.p.hd))
    return host_fail(M3G_EINVAL, "result rows overlap");
  if (q->p == out->p && (q->token_stride != out->token_stride || q->head_stride != out->head_stride))
    return host_fail(M3G_EINVAL, "results in place of q need the same strides");
  if (!std::isfinite(scale) || scale < 0.f) return host_fail(M3G_EINVAL, "scale must be finite and not negative");
  if (mask && static_cast<uint64_t>(mask_words) * 32 < b->max_tokens)
    return host_fail(M3G_EINVAL, "%u mask words for %u tokens", mask_words, b->max_tokens);
  uint64_t need = 0;
  if (int rc = m3g_tree_attn_workspace(l, n_heads, &need)) return rc;
  if (!b->n_tokens || !b->n_seqs) return M3G_OK;
  if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)
    return host_fail(M3G_EINVAL, "workspace of %llu bytes (16-byte aligned, %llu needed)",
                     static_cast<unsigned long long>(workspace_bytes), static_cast<unsigned long long>(need));
  int dev = 0;
  if (int rc = serve_device(&dev, &a.p.status)) return rc;
  a.b = *b;
  a.q = *q;
  a.out = *out;
  a.mask = mask;
  a.mask_words = static_cast<int>(mask_words);
  a.cap = seq_cap(*b, l->page_size);
  a.n_heads = static_cast<int>(n_heads);
  a.group = static_cast<int>(n_heads / l->n_kv_heads);
  a.scale = scale > 0.f ? scale : 1.f / sqrtf(static_cast<float>(a.p.hd));
  const cudaStream_t st = serve_stream(stream);
  const bool q8 = l->dtype == M3G_DTYPE_Q8_0;
  const cudaError_t e = dtype == M3G_DTYPE_F32   ? launch_tree_t<float>(a, q8, st)
                        : dtype == M3G_DTYPE_F16 ? launch_tree_t<__half>(a, q8, st)
                                                 : launch_tree_t<__nv_bfloat16>(a, q8, st);
  if (e != cudaSuccess) return host_fail(M3G_ECUDA, "k_tree_attn: %s", cudaGetErrorString(e));
  return M3G_OK;
}

}  // extern "C"
