// m3g_kv.cu -- the paged, quantised KV cache: writing new rows and reading
// rows back.
//
// A block is 32 consecutive values of a row: d = f16(max|x| / 127) (Q4_0: 7),
// code = round(x / d), halves away from zero, clamped -- the rules of
// quantize_q8_0 / quantize_q4_0 (src/quant.rs:206-264), whose f32 quotients
// are kept to the bit.  x times an approximate reciprocal of d is off by 2^-22
// of the quotient, so it decides unless it lies within 2^-14 (Q4_0: 2^-18) of a
// border between two codes or d is subnormal in f16 (codes_near_borders then).  max|x| / 127 is a product with the rounded reciprocal and one
// residual step (Markstein's theorem; equal to the division for every f32).  A block with a value that is not
// finite, or whose scale passes the f16 range, gets the scale NaN and codes
// that stand for 0, so that it reads back as NaN.
//
// Four threads share a block, 8 values each; a thread's 8 values are one
// 16-byte load (two for f32) and its codes one 8-byte store.  A CTA takes an even
// share of the tokens, 64 at a time, whose places its threads look up first, one
// token each.
//
// Measured: 20954 BF16 tokens of 8 + 8 heads of 128 (5 ragged prompts) to Q4_0, written
// 39.2 us (110 MB, 2.8 TB/s), read back 24.5 us (4.5 TB/s); 23918 tokens to Q8_0
// 34.8 us (150 MB, 4.3 TB/s) and back 33.0 us (4.6 TB/s).  Issue slots are 70 % used
// in writing (125 instructions for a thread's 8 values to Q8_0, 167 to Q4_0, where 29 %
// of the warps hold a value near a border), 64 % in reading (87).
#include <algorithm>

#include "m3g_device.cuh"
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
  if (misaligned(b->q_start, 4) || misaligned(b->ctx_len, 4) || misaligned(b->page_table, 4))
    return host_fail(M3G_EINVAL, "batch array not 4-byte aligned");
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
constexpr int kKvTokens = 64;    // tokens looked up at once
constexpr int kKvStarts = 1024;  // starts of sequences held in shared memory

struct KvIoArgs {
  KvPlanes p;
  m3g_kv_batch b;
  m3g_rows k, v;
  long long cap;
};

// A thread's 8 codes, in the bytes of two words (two's complement), by the
// rule.  F32: the quotient of a correctly rounded division.  16-bit values: no
// quotient but an exact half rounds to one (11-bit numbers: the others are off
// by 2^-12 at least), so the nearest code is found from the exact residual
// x - q d; these ties are common (wherever max|x| / 127 is an 11-bit number).
template <class T>
__device__ __forceinline__ uint2 codes_near_borders(const float (&v)[8], float d, float inv, float least, float most) {
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float q;
    if (sizeof(T) == 4) {
      q = roundf(__fdiv_rn(v[i], d));
    } else {
      q = rintf(v[i] * inv);
      const float e = fmaf(-q, d, v[i]);
      // away from zero at a tie: where the residual still points away
      if (e * v[i] > 0.f ? 2.f * fabsf(e) >= d : 2.f * fabsf(e) > d) q += copysignf(1.f, e);
    }
    q = d > 0.f ? fminf(fmaxf(q, least), most) : 0.f;
    w[i >> 2] |= (static_cast<uint32_t>(static_cast<int>(q)) & 0xFFu) << (8 * (i & 3));
  }
  return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN where one is NaN
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The largest magnitude of the 8 values of each of a block's four threads, NaN
// where one is NaN; 16-bit values two at a time.
template <class T>
__device__ __forceinline__ float block_max(const T (&x)[8], unsigned lanes) {
  if constexpr (sizeof(T) == 2) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* w = reinterpret_cast<const T2*>(x);
    T2 m = __hmax2_nan(__hmax2_nan(__habs2(w[0]), __habs2(w[1])), __hmax2_nan(__habs2(w[2]), __habs2(w[3])));
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) m = __hmax2_nan(m, __shfl_xor_sync(lanes, m, o));
    return max_nan(Act<T>::to(m.x), Act<T>::to(m.y));
  } else {
    float m = max_nan(fabsf(x[0]), fabsf(x[1]));
#pragma unroll
    for (int i = 2; i < 8; i += 2) m = max_nan(m, fabsf(x[i]), fabsf(x[i + 1]));
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) m = max_nan(m, __shfl_xor_sync(lanes, m, o));
    return m;
  }
}

// Places of the CTA's tokens: byte offsets of head 0's row in a plane of codes, -1 for none.  One
// thread looks up one token, by bisection over the starts of the sequences (in
// shared memory where they fit).
__device__ __forceinline__ void find_places(const KvIoArgs& a, int t0, int n_tok, long long* place, int32_t* starts) {
  const int tid = threadIdx.x, n_seqs = static_cast<int>(a.b.n_seqs);
  const bool held = n_seqs <= kKvStarts;
  if (tid >= n_tok && tid < kKvTokens) place[tid] = -1;
  if (tid < n_tok) {
    const int t = t0 + tid;
    int lo = 0, hi = n_seqs;  // the last s with q_start[s] <= t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((held ? starts[mid] : a.b.q_start[mid]) <= t) lo = mid;
      else hi = mid;
    }
    long long at = -1;
    bool bad = false;  // hold_starts reports it
    const SeqView s = seq_view(a.b, a.cap, lo, &bad);
    if (t >= s.q0 && t - s.q0 < s.n) {
      const int pos = s.ctx + (t - s.q0);
      const int page = a.b.page_table[static_cast<long long>(lo) * a.b.max_pages + (pos >> a.p.page_shift)];
      if (page >= 0 && page < a.p.n_pages)
        at = kv_row(a.p, page, 0, pos & (a.p.page_size - 1)) * a.p.cb;
      else
        atomicOr(a.p.status, kStatusBadPage);
    }
    place[tid] = at;
  }
  __syncthreads();
}

// The starts into shared memory, where they fit.  The first CTA (all, where they
// do not) looks the sequences over and reports those outside the call's limits,
// also ones that no token leads to.
__device__ __forceinline__ void hold_starts(const KvIoArgs& a, int32_t* starts) {
  const int n_seqs = static_cast<int>(a.b.n_seqs), tid = threadIdx.x;
  bool bad = false;
  if (n_seqs > kKvStarts) {
    for (long long s = static_cast<long long>(blockIdx.x) * kKvThreads + tid; s < n_seqs; s += gridDim.x * kKvThreads)
      seq_view(a.b, a.cap, static_cast<int>(s), &bad);
  } else if (blockIdx.x == 0) {
    for (int s = tid; s < n_seqs; s += kKvThreads) {
      const SeqView v = seq_view(a.b, a.cap, s, &bad);
      starts[s] = v.q0;
    }
  } else {
    for (int s = tid; s < n_seqs; s += kKvThreads) starts[s] = a.b.q_start[s];
  }
  if (bad) atomicOr(a.p.status, kStatusBadBatch);
  __syncthreads();
}

// How a CTA's threads share the 8-value pieces of its tokens: thread -> one
// piece of a token (K heads, then V heads) and every `ny`-th token; tokens
// with more pieces than threads (not FITS) are walked piece by piece.
template <bool FITS>
struct KvShare {
  int octs, per, ny, y0, w0;
  __device__ __forceinline__ explicit KvShare(const KvPlanes& p) {
    octs = p.hd / 8;
    per = 2 * p.kvh * octs;  // a multiple of 16: the four threads of a block stay together
    ny = FITS ? kKvThreads / per : 1;
    y0 = FITS ? static_cast<int>(threadIdx.x) / per : 0;
    w0 = FITS ? static_cast<int>(threadIdx.x) - y0 * per : static_cast<int>(threadIdx.x);
  }
};

template <class T, bool VEC>
struct alignas(VEC ? 16 : sizeof(T)) Oct {
  T t[8];
};

// Where a thread's piece of a token goes.
struct KvPiece {
  uint8_t *codes, *scales;  // at a place of 0
  int64_t stride, offset;   // of the activations: between tokens; of the piece in a token
  int oct;
  bool is_v;
  __device__ __forceinline__ KvPiece(const KvIoArgs& a, bool q8, int octs, int w) {
    // picked by value: a reference picked at run time would make every access a load from memory
    const int row = w / octs;
    oct = w - row * octs;
    is_v = row >= a.p.kvh;
    const int head = is_v ? row - a.p.kvh : row;
    const long long rows = static_cast<long long>(head) * a.p.page_size;
    codes = (is_v ? a.p.vc : a.p.kc) + rows * a.p.cb + (q8 ? oct * 8 : (oct >> 2) * 16 + (oct & 1) * 8);
    scales = (is_v ? a.p.vs : a.p.ks) + rows * a.p.sb + (oct >> 2) * 2;
    stride = is_v ? a.v.token_stride : a.k.token_stride;
    offset = head * (is_v ? a.v.head_stride : a.k.head_stride) + oct * 8;
  }
};

// Codes of 8 values (four neighbouring threads hold their block) into their
// place; `lanes` call together, those with a negative place store nothing.
template <class T, bool Q8>
__device__ __forceinline__ void write_piece(const KvPiece& w, long long place, const T (&x)[8],
                                            unsigned lanes) {
  float v[8];
  unpack_act<T, 8>(x, v);
  const float most = block_max<T>(x, lanes);
  constexpr float kMost = Q8 ? 127.f : 7.f, kInv = 1.f / kMost;
  const float q0 = most * kInv;
  __half dh = __float2half_rn(fmaf(fmaf(-kMost, q0, most), kInv, q0));
  const float d = __half2float(dh);
  const bool ok = d <= 65504.f;  // else a value that is not finite, or a scale past the f16 range
  if (!ok) dh = __ushort_as_half(0x7FFF);
  // nearest integers by the sum with 1.5 * 2^23; at |x / d| <= 127 (1 + 2^-11) none needs a clamp
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(d));
  float far = 0.f;  // the largest distance from the nearest integer
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint64_t t = mul2(pair(v[i], v[i + 1]), pair(inv, inv)), u = add2(t, pair(12582912.f, 12582912.f));
    const uint64_t e = fma2(add2(u, pair(-12582912.f, -12582912.f)), pair(-1.f, -1.f), t);
    far = max3(far, fabsf(low(e)), fabsf(high(e)));
    c[i] = __float_as_uint(low(u));
    c[i + 1] = __float_as_uint(high(u));
  }
  const bool near = d < 0x1p-14f || far > 0.5f - (Q8 ? 0x1p-14f : 0x1p-18f);
  uint32_t w0 = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
  uint32_t w1 = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
  if (near) {
    const uint2 e = codes_near_borders<T>(v, ok ? d : 0.f, inv, Q8 ? -127.f : -8.f, Q8 ? 127.f : 7.f);
    w0 = e.x;
    w1 = e.y;
  }
  if (!ok) w0 = w1 = 0u;
  const bool store = place >= 0;
  if (Q8) {
    if (store) *reinterpret_cast<uint2*>(w.codes + place) = make_uint2(w0 ^ 0x80808080u, w1 ^ 0x80808080u);
  } else {
    w0 = (w0 & 0x0F0F0F0Fu) ^ 0x08080808u;
    w1 = (w1 & 0x0F0F0F0Fu) ^ 0x08080808u;
    const uint32_t g0 = __shfl_xor_sync(lanes, w0, 2), g1 = __shfl_xor_sync(lanes, w1, 2);
    if (store && (w.oct & 2) == 0)  // the block's first 16 values are the low nibbles
      *reinterpret_cast<uint2*>(w.codes + place) = make_uint2(w0 | g0 << 4, w1 | g1 << 4);
  }
  // a scale of 2 bytes for 32 (Q4_0: 16) bytes of codes
  if (store && (w.oct & 3) == 0) *reinterpret_cast<__half*>(w.scales + (place >> (Q8 ? 4 : 3))) = dh;
}

// RING (a thread has one piece of a token, 16-byte aligned): its pieces of the
// next tokens come by cp.async into its own places in shared memory, 128 bytes
// a thread in flight.
template <class T, bool Q8, bool VEC, bool FITS>
__global__ void __launch_bounds__(kKvThreads, 4) k_kv_write(const __grid_constant__ KvIoArgs a) {
  constexpr bool RING = VEC && FITS;
  constexpr int PB = 8 * sizeof(T), D = 128 / PB;  // bytes of a piece; pieces in flight
  __shared__ long long place[kKvTokens];
  __shared__ int32_t starts[kKvStarts];
  __shared__ __align__(16) uint8_t ring[RING ? kKvThreads * 128 : 16];
  const int tid = threadIdx.x;
  const int t_begin = static_cast<int>(static_cast<long long>(blockIdx.x) * a.b.n_tokens / gridDim.x);
  const int t_end = static_cast<int>((blockIdx.x + 1ll) * a.b.n_tokens / gridDim.x);
  const unsigned quad = 0xFu << (tid & 28);
  const KvShare<FITS> sh(a.p);
  const bool active = sh.y0 < sh.ny && sh.w0 < sh.per;
  const KvPiece mine(a, Q8, sh.octs, active ? sh.w0 : 0);
  const T* from = static_cast<const T*>(mine.is_v ? a.v.p : a.k.p) + mine.offset + (t_begin + sh.y0) * mine.stride;
  const int64_t step = sh.ny * mine.stride;
  auto slot = [&](int d, int h) { return ring + ((d * (PB / 16) + h) * kKvThreads + tid) * 16; };
  auto fetch = [&](int t, int d) {
    if (active && t < t_end) {
#pragma unroll
      for (int h = 0; h < PB / 16; ++h) cp16(slot(d, h), from + h * (16 / sizeof(T)), 16);
      from += step;
    }
    cp_commit();
  };
  if (RING) {
#pragma unroll
    for (int d = 0; d < D; ++d) fetch(t_begin + sh.y0 + d * sh.ny, d);
  }
  int depth = 0;
  hold_starts(a, starts);
  const int batch = kKvTokens / sh.ny * sh.ny;  // a thread's tokens are ny apart across batches too
  for (int t0 = t_begin; t0 < t_end; t0 += batch) {
    const int n_tok = min(batch, t_end - t0);
    find_places(a, t0, n_tok, place, starts);
    if constexpr (RING) {
      for (int k = 0; k < n_tok; k += sh.ny) {  // whole warps: shuffles of a part of one cost more than a block
        const int ti = k + sh.y0;
        cp_wait<D - 1>();
        alignas(16) T x[8];
#pragma unroll
        for (int h = 0; h < PB / 16; ++h)
          reinterpret_cast<uint4*>(x)[h] = *reinterpret_cast<const uint4*>(slot(depth, h));
        fetch(t0 + ti + D * sh.ny, depth);
        depth = depth + 1 == D ? 0 : depth + 1;
        write_piece<T, Q8>(mine, active ? place[ti] : -1, x, 0xFFFFFFFFu);
      }
    } else {
      for (int w = active ? sh.w0 : sh.per; w < sh.per; w += FITS ? sh.per : kKvThreads) {
        const KvPiece piece(a, Q8, sh.octs, w);
        const T* src = static_cast<const T*>(piece.is_v ? a.v.p : a.k.p) + t0 * piece.stride + piece.offset;
        for (int ti = sh.y0; ti < n_tok; ti += sh.ny) {
          if (place[ti] < 0) continue;
          const Oct<T, VEC> x = *reinterpret_cast<const Oct<T, VEC>*>(src + ti * piece.stride);
          write_piece<T, Q8>(piece, place[ti], x.t, quad);
        }
      }
    }
    __syncthreads();  // the places are read
  }
}

template <class T, bool Q8, bool VEC, bool FITS>
__global__ void __launch_bounds__(kKvThreads, 4) k_kv_read(const __grid_constant__ KvIoArgs a) {
  constexpr int U = 8;  // tokens in flight
  __shared__ long long place[kKvTokens];
  __shared__ int32_t starts[kKvStarts];
  const int t_begin = static_cast<int>(static_cast<long long>(blockIdx.x) * a.b.n_tokens / gridDim.x);
  const int t_end = static_cast<int>((blockIdx.x + 1ll) * a.b.n_tokens / gridDim.x);
  const KvShare<FITS> sh(a.p);
  hold_starts(a, starts);
  for (int t0 = t_begin; t0 < t_end; t0 += kKvTokens) {
    const int n_tok = min(kKvTokens, t_end - t0);
    find_places(a, t0, n_tok, place, starts);
    for (int w = sh.y0 < sh.ny ? sh.w0 : sh.per; w < sh.per; w += FITS ? sh.per : kKvThreads) {
      const KvPiece piece(a, Q8, sh.octs, w);
      const int down = (piece.oct & 2) ? 4 : 0;
      T* dst = static_cast<T*>(piece.is_v ? a.v.p : a.k.p) + t0 * piece.stride + piece.offset;
      for (int ti0 = sh.y0; ti0 < n_tok; ti0 += U * sh.ny) {
        uint2 q[U];
        __half d[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
          const int ti = ti0 + k * sh.ny;
          if (ti < n_tok && place[ti] >= 0) {
            q[k] = *reinterpret_cast<const uint2*>(piece.codes + place[ti]);
            d[k] = *reinterpret_cast<const __half*>(piece.scales + (place[ti] >> (Q8 ? 4 : 3)));
          }
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
          const int ti = ti0 + k * sh.ny;
          if (ti >= n_tok || place[ti] < 0) continue;
          if (!Q8) {
            q[k].x = q[k].x >> down & 0x0F0F0F0Fu;
            q[k].y = q[k].y >> down & 0x0F0F0F0Fu;
          }
          const float f = __half2float(d[k]);
          Oct<T, VEC> y;
          float v[8];
          v[0] = byte_2p23<0>(q[k].x); v[1] = byte_2p23<1>(q[k].x);
          v[2] = byte_2p23<2>(q[k].x); v[3] = byte_2p23<3>(q[k].x);
          v[4] = byte_2p23<0>(q[k].y); v[5] = byte_2p23<1>(q[k].y);
          v[6] = byte_2p23<2>(q[k].y); v[7] = byte_2p23<3>(q[k].y);
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            constexpr float kZero = -(k2p23 + (Q8 ? 128.f : 8.f));
            const uint64_t x = mul2(add2(pair(v[i], v[i + 1]), pair(kZero, kZero)), pair(f, f));
            v[i] = low(x);
            v[i + 1] = high(x);
          }
          pack_act<T, 8>(y.t, v);
          *reinterpret_cast<Oct<T, VEC>*>(dst + ti * piece.stride) = y;
        }
      }
    }
    __syncthreads();  // the places are read
  }
}

template <class T, bool Q8, bool VEC>
cudaError_t launch_kv(const KvIoArgs& a, bool write, int sms, cudaStream_t st) {
  const dim3 grid(std::min<uint32_t>(a.b.n_tokens, 4u * static_cast<uint32_t>(sms))), block(kKvThreads);
  const bool fits = 2 * a.p.kvh * (a.p.hd / 8) <= kKvThreads;
  if (write)
    return fits ? serve_launch(k_kv_write<T, Q8, VEC, true>, grid, block, 0, st, false, a)
                : serve_launch(k_kv_write<T, Q8, VEC, false>, grid, block, 0, st, false, a);
  return fits ? serve_launch(k_kv_read<T, Q8, VEC, true>, grid, block, 0, st, false, a)
              : serve_launch(k_kv_read<T, Q8, VEC, false>, grid, block, 0, st, false, a);
}
template <class T>
cudaError_t launch_kv_t(const KvIoArgs& a, bool q8, bool vec, bool write, int sms, cudaStream_t st) {
  if (q8) return vec ? launch_kv<T, true, true>(a, write, sms, st) : launch_kv<T, true, false>(a, write, sms, st);
  return vec ? launch_kv<T, false, true>(a, write, sms, st) : launch_kv<T, false, false>(a, write, sms, st);
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
    if (misaligned(r->p, size)) return host_fail(M3G_EINVAL, "rows not aligned to their type");
    if (r->token_stride < 0 || r->head_stride < 0) return host_fail(M3G_EINVAL, "negative stride");
    if (!write && ((b->n_tokens > 1 && r->token_stride < a.p.hd) || (a.p.kvh > 1 && r->head_stride < a.p.hd)))
      return host_fail(M3G_EINVAL, "result rows overlap");
    vec = vec && rows_aligned(r->p, r->token_stride, r->head_stride, size);
  }
  if (!b->n_tokens || !b->n_seqs) return M3G_OK;
  int dev = 0, sms = 0;
  if (int rc = serve_device(&dev, &a.p.status)) return rc;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return host_fail(M3G_ECUDA, "device attributes");
  a.b = *b;
  a.k = *k;
  a.v = *v;
  a.cap = seq_cap(*b, l->page_size);
  const cudaStream_t st = serve_stream(stream);
  const bool q8 = l->dtype == M3G_DTYPE_Q8_0;
  const cudaError_t e = dtype == M3G_DTYPE_F32   ? launch_kv_t<float>(a, q8, vec, write, sms, st)
                        : dtype == M3G_DTYPE_F16 ? launch_kv_t<__half>(a, q8, vec, write, sms, st)
                                                 : launch_kv_t<__nv_bfloat16>(a, q8, vec, write, sms, st);
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
