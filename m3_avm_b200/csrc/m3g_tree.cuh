// m3g_tree.cuh -- what the two forms of tree attention share: arguments, the
// even cut of the work over the CTAs, and the join of pieces.
//
// Sequences' lengths are only known on the device.  A unit is one (sequence, KV
// head, row tile), cut into chunks of positions; each CTA adds up all chunks
// from the lengths and takes an equal, contiguous share, whatever unit borders
// lie in it.  A unit inside one CTA is written out there; pieces of a cut one go
// to the workspace, and k_tree_join adds them up in CTA order, so the bits do
// not depend on timing.  One token of one long sequence is thus spread over all
// SMs, and a ragged batch is balanced to one chunk.
#pragma once
#include "m3g_device.cuh"
#include "m3g_serve.cuh"

namespace m3g {

constexpr int kTreeMaxCtas = 3 * 160;  // CTAs that the workspace is sized for

struct TreeArgs {
  KvPlanes p;
  m3g_kv_batch b;
  m3g_rows q, out;
  const uint32_t* mask;
  float* parts;  // [2 * CTAs] pieces: a tile's results, then its maxima and sums
  int4* desc;    // [CTAs] the cut unit that starts in the CTA: sequence (-1: none), KV head, tile, its last CTA
  long long cap;
  int mask_words, n_heads, group;
  int vec, vec_out;  // q, result rows are 16-byte aligned
  float scale;
  uint32_t wait_polls, wait_ns;  // of the 128-row form's waits: polls, and the longest that each takes
};

template <int HD, int TILE>
struct Part {
  static constexpr int kFloats = TILE * HD + 2 * TILE;
};

__device__ __forceinline__ float tex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The factor that turns raw scores into base-2 exponents.  Never 0: -inf, the score
// of what a row does not see, times 0 is NaN.  (Raw scores stay below 2^42, so
// that with factors up to this one all seen scores are 0 to 2^-84.)
__device__ __forceinline__ float score_factor(float f) { return fmaxf(f, 0x1p-126f); }

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t x) {
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}

// Low n bits set, n clamped to 0 .. 32.
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

// A sequence's work in chunks of CHUNK positions and tiles of TILE rows.
// kTreeMost: chunks that a batch may come to.  The host refuses what its tokens and
// bounds could exceed; tree_share looks at what the arrays really say (sequences
// that overlap can come to more), so that every sum of chunks fits an int.
constexpr long long kTreeMost = (1ll << 31) - 1024;
template <int CHUNK, int TILE>
struct SeqWork {
  SeqView v;
  int chunks, tiles;  // chunks per unit, row tiles per KV head
  __device__ __forceinline__ SeqWork(const TreeArgs& a, int s, bool* bad) : v(seq_view(a.b, a.cap, s, bad)) {
    chunks = v.n ? (v.ctx + v.n + CHUNK - 1) / CHUNK : 0;
    tiles = (v.n * a.group + TILE - 1) / TILE;
  }
  __device__ __forceinline__ int total(int kvh) const { return chunks * tiles * kvh; }
  __device__ __forceinline__ long long total64(int kvh) const { return static_cast<long long>(chunks) * tiles * kvh; }
};

// A CTA's share of all chunks and where it starts: G CTAs have work, the first
// `more` of them each + 1 chunks, the others `each`.
struct TreeShare {
  int G, each, more;
  int first, last;  // this CTA's chunks
  int before;       // chunks of the sequences before `seq`
  int seq;          // sequence of the first chunk
};

struct ShareScratch {
  int red[32], red2[32], found[2];
};

// All threads of the CTA (THREADS, whole warps); false: nothing to do.  LEAST:
// chunks that a CTA takes at least while there are so many.
template <int CHUNK, int TILE, int THREADS, int LEAST>
__device__ __forceinline__ bool tree_share(const TreeArgs& a, ShareScratch& sc, TreeShare& out) {
  constexpr int WARPS = THREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n_seqs = static_cast<int>(a.b.n_seqs), kvh = a.p.kvh;
  using Work = SeqWork<CHUNK, TILE>;
  bool bad = false;
  long long mine = 0, own0 = 0;
#pragma unroll 1
  for (int s = tid; s < n_seqs; s += THREADS) {
    const long long own = min(Work(a, s, &bad).total64(kvh), kTreeMost + 1);
    if (s == tid) own0 = own;
    mine += own;
  }
  mine = min(mine, kTreeMost + 1);  // added up in two parts, of 24 bits and of the others
  const int lo = __reduce_add_sync(0xFFFFFFFFu, static_cast<int>(mine & 0xFFFFFF));
  const int hi = __reduce_add_sync(0xFFFFFFFFu, static_cast<int>(mine >> 24));
  if (lane == 0) {
    sc.red[warp] = lo;
    sc.red2[warp] = hi;
  }
  __syncthreads();
  const int part = lane < WARPS ? sc.red[lane] : 0, above = lane < WARPS ? sc.red2[lane] : 0;
  const long long all = __reduce_add_sync(0xFFFFFFFFu, part & 0xFFFFFF) +
                        (static_cast<long long>(__reduce_add_sync(0xFFFFFFFFu, above + (part >> 24))) << 24);
  if (all > kTreeMost) bad = true;  // the batch as a whole: nothing is done
  if (bad && blockIdx.x == 0) atomicOr(a.p.status, kStatusBadBatch);
  const int W = all > kTreeMost ? 0 : static_cast<int>(all);
  const int b = blockIdx.x, G = min(static_cast<int>(gridDim.x), (W + LEAST - 1) / LEAST);
  if (tid == 0) a.desc[b].x = -1;
  if (b >= G) return false;
  out.G = G;
  out.each = W / G;
  out.more = W - out.each * G;
  out.first = b * out.each + min(b, out.more);
  out.last = out.first + out.each + (b < out.more);
  int before = 0;
#pragma unroll 1
  for (int s0 = 0; s0 < n_seqs; s0 += THREADS) {
    int own = static_cast<int>(own0);
    if (s0) own = s0 + tid < n_seqs ? Work(a, s0 + tid, &bad).total(kvh) : 0;
    int up = own;  // inclusive scan
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xFFFFFFFFu, up, o);
      if (lane >= o) up += x;
    }
    __syncthreads();
    if (lane == 31) sc.red[warp] = up;
    __syncthreads();
    const int w = lane < WARPS ? sc.red[lane] : 0;
    up += __reduce_add_sync(0xFFFFFFFFu, lane < warp ? w : 0);
    const int begin = before + up - own;
    if (out.first >= begin && out.first < begin + own) {
      sc.found[0] = s0 + tid;
      sc.found[1] = begin;
    }
    before += __reduce_add_sync(0xFFFFFFFFu, w);
    if (out.first < before) break;  // the same for all threads
  }
  __syncthreads();
  out.seq = sc.found[0];
  out.before = sc.found[1];
  return true;
}

// The CTA that holds a unit's last chunk; `end`: the chunks up to the unit's end.
__device__ __forceinline__ int tree_last_cta(const TreeShare& s, int end) {
  const int x = end - 1, y = x - s.more * (s.each + 1);
  return y < 0 ? x / (s.each + 1) : s.more + y / s.each;
}

// The new tokens of its sequence, and positions before them, that token number
// `token` (in the sequence; `q0` its first) sees among positions p0 .. p0 + 31,
// one bit each.
__device__ __forceinline__ uint32_t tree_sees(const TreeArgs& a, int q0, int token, int ctx, int len, int p0) {
  const int i0 = p0 - ctx;  // the first position as a new token's number
  uint32_t vis;
  if (!a.mask) {
    vis = low_bits(token + 1 - i0);
  } else {
    const uint32_t* row = a.mask + static_cast<long long>(q0 + token) * a.mask_words;
    const int wd = i0 >> 5;  // floor: negative while context positions come first
    const uint32_t lo = wd >= 0 && wd < a.mask_words ? row[wd] : 0u;
    const uint32_t hi = wd + 1 >= 0 && wd + 1 < a.mask_words ? row[wd + 1] : 0u;
    vis = __funnelshift_r(lo, hi, i0 & 31) | low_bits(-i0);
  }
  return vis & low_bits(len - p0);
}

// The pieces of the units that were cut, in CTA order: a row of CTAs per main
// CTA, ROWS rows of the tile per warp (their loads in flight together).
constexpr int kJoinWarps = 16;
template <class T, int HD, int TILE, int ROWS>
__global__ void __launch_bounds__(32 * kJoinWarps) k_tree_join(const __grid_constant__ TreeArgs a) {
  constexpr int DPL = HD / 32;
  grid_dep_wait();
  const int4 u = a.desc[blockIdx.x];
  if (u.x < 0) return;
  const int lane = threadIdx.x & 31, row0 = (blockIdx.y * kJoinWarps + (threadIdx.x >> 5)) * ROWS;
  bool bad = false;
  const SeqView s = seq_view(a.b, a.cap, u.x, &bad);
  const int rows = min(TILE, s.n * a.group - u.z * TILE);  // of the tile
  if (row0 >= rows) return;
  const int n = u.w - static_cast<int>(blockIdx.x) + 1;  // pieces
  auto part = [&](int i) {  // this CTA's piece starts the unit, the others continue it
    return a.parts + static_cast<long long>(i ? 2 * (blockIdx.x + i) : 2 * blockIdx.x + 1) * Part<HD, TILE>::kFloats;
  };
  float M[ROWS], L[ROWS], O[ROWS][DPL];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    M[r] = -INFINITY;
    L[r] = 0.f;
#pragma unroll
    for (int d = 0; d < DPL; ++d) O[r][d] = 0.f;
  }
  for (int i = lane; i < n; i += 32) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (row0 + r < rows) M[r] = fmaxf(M[r], part(i)[TILE * HD + row0 + r]);
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
#pragma unroll
    for (int o = 16; o; o >>= 1) M[r] = fmaxf(M[r], __shfl_xor_sync(0xFFFFFFFFu, M[r], o));
    if (M[r] == -INFINITY) M[r] = 0.f;
  }
#pragma unroll 8 / ROWS
  for (int i = 0; i < n; ++i) {
    const float* p = part(i);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (row0 + r >= rows) continue;
      const float f = tex2(p[TILE * HD + row0 + r] - M[r]);
      L[r] += f * p[TILE * HD + TILE + row0 + r];
      float v[DPL];
      load_act<float, DPL, true>(p + (row0 + r) * HD + lane * DPL, v);
#pragma unroll
      for (int d = 0; d < DPL; ++d) O[r][d] += f * v[d];
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (row0 + r >= rows) continue;
    const int row = u.z * TILE + row0 + r;
    T* y = static_cast<T*>(a.out.p) + (s.q0 + row / a.group) * a.out.token_stride +
           (u.y * a.group + row % a.group) * a.out.head_stride;
    const float inv = L[r] == 0.f ? 0.f : 1.f / L[r];
#pragma unroll
    for (int d = 0; d < DPL; ++d) y[lane * DPL + d] = Act<T>::from(L[r] == 0.f ? 0.f : O[r][d] * inv);
  }
}

// A tile's join: 1 row per warp for tiles of 16, 4 for larger ones.
template <class T, int HD, int TILE>
cudaError_t launch_join(const TreeArgs& a, int grid, cudaStream_t st) {
  constexpr int ROWS = TILE > kJoinWarps ? 4 : 1;
  return serve_launch(k_tree_join<T, HD, TILE, ROWS>, dim3(grid, TILE / (kJoinWarps * ROWS)), dim3(32 * kJoinWarps), 0,
                      st, true, a);
}

// The form on the fifth-generation tensor cores (m3g_tree_umma.cu): 16-bit
// types, units of 128 rows.
constexpr int kUmmaTile = 128, kUmmaChunk = 64;  // rows, positions
cudaError_t launch_tree_umma(const TreeArgs& a, uint32_t dtype, bool q8, int sms, cudaStream_t st);

}  // namespace m3g
