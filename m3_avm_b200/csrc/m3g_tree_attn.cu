// m3g_tree_attn.cu -- attention of drafted tokens over the quantised KV cache.
//
// out = softmax(scale * q K^T + mask) V with a running maximum and sum, the
// cached codes multiplied as they are.
//
// Rows.  The query heads that share a KV head and the new tokens of a sequence
// are the rows of one product (row = token * group + head in group), 16 to a
// tile; every tile reads its sequence's K and V of one KV head.
//
// Products.  mma.sync m16n8k16 in f16 with f32 sums.  A code (c - 128, or
// n - 8) is an integer that f16 holds exactly: one PRMT puts it behind the
// exponent of 1024 and one HADD2 takes the offset off.  Scores: 32 products per
// block, then f32 scores += d * sum, so nothing of K is rounded.  Values: the
// weight times V's scale, p * d, is the f16 operand and V's codes the exact
// other one.  q is an exact f16 operand for F16 and BF16 (its rows are scaled by
// a power of two); for F32 q and p * d are two f16 parts, hi + lo, 22 bits.
// So that p * d stays in f16's normal range whatever V's scale, d is taken
// relative to a power of two dref >= every |d| seen by the warp; when it grows,
// the sums are rescaled (rare).
//
// Inside a CTA each of 4 warps owns every fourth group of 32 positions and a
// ring of stages filled by 16-byte cp.async; it keeps its own maximum, sum and
// 16 x HD results in registers, so the warps meet only at the end of a piece.
// The stages are swizzled so that the fragment loads touch all banks.
//
// Split.  The chunks of all sequences, heads and tiles form one line that the
// CTAs cut evenly, whatever the lengths; a unit that is cut leaves its parts
// (maximum, sum, results) in the workspace for k_tree_join.
//
// Bound.  With few rows HBM: 48 ragged contexts of up to 16000 positions, 4 rows
// a KV head, BF16 over Q8_0: 239 us in a graph, 4.75 TB/s (one call after another from
// Python 268); the same loads without the arithmetic take 181 us, the rest is ALU
// work (unpacking, softmax) beside them.  One context of 1024 positions: 9.2 to 9.6 us,
// of which a launch, the loads' latency and the join each take 2 to 3.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "m3g_tree.cuh"

namespace m3g {
namespace {

constexpr int kTreeWarps = 4;
constexpr int kTreeThreads = 32 * kTreeWarps;
constexpr int kGroup = 32;                      // positions per warp and step
constexpr int kChunk = kGroup * kTreeWarps;     // positions per unit of work
constexpr int kTile = 16;                       // rows per tile
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same into a new sum.
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// Bytes SEL picks of w (two of them), less `off`, as exact f16 values.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t codes2(uint32_t w, __half2 off) {
  const uint32_t x = __byte_perm(w, 0x64646464u, SEL);  // 1024 + byte
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), off);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// CTAs per SM: what their registers leave room for without spills in the loop.
// With 64 values a row three (12 warps of 168 registers; 8 contexts of 8000
// positions and 16 tokens: 27.0 us, with two 28.0; F32, 256 tokens: 195 us, with two
// 214).  With 128 values two: three need 26 KB of stages instead of 48 and gain
// nothing, since the ALU pipe is what is short and not warps to issue from (48
// ragged contexts of up to 16000 positions: 246 us, with three 249).
template <int HD>
struct Ctas {
  static constexpr int kPerSm = HD == 128 ? 2 : 3;
};

// Geometry of a warp's stage: K codes, V codes, K scales, V scales of 32 rows.
template <int HD, bool Q8, int CTAS>
struct Stage {
  static constexpr int CB = Q8 ? HD : HD / 2, SB = HD / 16, NB = HD / 32;
  static constexpr int CPR = CB / 16;   // 16-byte pieces per row
  static constexpr int RPL = 128 / CB;  // rows per 128-byte line
  static constexpr int kCodes = kGroup * CB, kScales = kGroup * SB;
  static constexpr int kBytes = 2 * (kCodes + kScales);
  static constexpr int kRoom = CTAS == 2 ? 26112 : 18432;  // shared memory of a warp
  static constexpr int NS = kRoom / kBytes < 8 ? kRoom / kBytes : 8;
  static constexpr int kWarpBytes = NS * kBytes;
  // Byte offset of 16-byte piece `col` of `row`.  K fragments read one block of
  // 8 rows at once, V fragments one block of rows 2t (t = 0..3).
  static __device__ __forceinline__ int k_at(int row, int col) {
    int slot = (row % RPL) * CPR + col;
    if (Q8) slot ^= HD == 128 ? (row & 3) << 1 : ((row >> 1) & 1) << 1;
    else slot ^= HD == 128 ? (row >> 1) & 3 : (row >> 2) & 1;
    return (row / RPL) * 128 + slot * 16;
  }
  static __device__ __forceinline__ int v_at(int row, int col) {
    int slot = (row % RPL) * CPR + col;
    if (Q8) slot ^= ((row >> 1) & 3) << 1;
    else slot ^= HD == 128 ? (row >> 1) & 3 : (row >> 2) & 1;
    return (row / RPL) * 128 + slot * 16;
  }
};

template <int HD, bool Q8, int CTAS>
constexpr size_t tree_smem() {
  const size_t ring = static_cast<size_t>(kTreeWarps) * Stage<HD, Q8, CTAS>::kWarpBytes;
  const size_t join = sizeof(float) * kTreeWarps * kTile * (HD + 4 + 2);
  return ring > join ? ring : join;
}

template <class T, int HD, bool Q8>
__global__ void __launch_bounds__(kTreeThreads, (Ctas<HD>::kPerSm)) k_tree_attn(const __grid_constant__ TreeArgs a) {
  using St = Stage<HD, Q8, Ctas<HD>::kPerSm>;
  constexpr bool SPLIT = std::is_same<T, float>::value;
  constexpr int NB = St::NB, NT = kGroup / 8, NO = HD / 8, KS = HD / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ ShareScratch scratch;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = lane >> 2, t = lane & 3;
  const int kvh = a.p.kvh;
  TreeShare share;
  if (!tree_share<kChunk, kTile, kTreeThreads, 1>(a, scratch, share)) return;
  bool bad = false;
  int seq = share.seq;
  SeqWork<kChunk, kTile> sw(a, seq, &bad);
  int base_chunk = share.before;  // chunks of the sequences before this one
  int at = share.first;           // the next chunk
  const int last = share.last;

  uint8_t* ring = smem + warp * St::kWarpBytes;
  const __half2 off = __half2half2(__ushort_as_half(Q8 ? 0x6480 : 0x6408));  // 1152, 1032

  while (at < last) {
    while (at >= base_chunk + sw.total(kvh)) {
      base_chunk += sw.total(kvh);
      sw = SeqWork<kChunk, kTile>(a, ++seq, &bad);
    }
    const int in_seq = (at - base_chunk) / sw.chunks;  // unit of the sequence
    const int c0 = at - base_chunk - in_seq * sw.chunks;
    const int c1 = min(sw.chunks, c0 + (last - at));
    const int head = in_seq / sw.tiles, tile = in_seq % sw.tiles;
    const int ctx = sw.v.ctx, len = sw.v.ctx + sw.v.n, rows = sw.v.n * a.group;
    const int32_t* table = a.b.page_table + static_cast<long long>(seq) * a.b.max_pages;

    // ---------------------------------------------------------------- copies
    int pg[2];  // pages of the next step's two groups of 16 positions
    auto pages_of = [&](int c) {
      const int p0 = c * kChunk + warp * kGroup;
#pragma unroll
      for (int h = 0; h < 2; ++h) pg[h] = c < c1 && p0 + 16 * h < len ? table[(p0 + 16 * h) >> a.p.page_shift] : 0;
    };
    auto issue = [&](int c) {
      if (c < c1) {
        const int p0 = c * kChunk + warp * kGroup, valid = min(kGroup, len - p0);
        uint8_t* st = ring + ((c - c0) % St::NS) * St::kBytes;
        long long row[2];
        int have[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool there = pg[h] >= 0 && pg[h] < a.p.n_pages;
          if (!there && valid > 16 * h && lane == 0) atomicOr(a.p.status, kStatusBadPage);
          row[h] = there ? kv_row(a.p, pg[h], head, (p0 + 16 * h) & (a.p.page_size - 1)) : 0;
          have[h] = there ? min(16, valid - 16 * h) : 0;
        }
#pragma unroll
        for (int i = 0; i < St::CPR; ++i) {
          const int x = i * 32 + lane, rw = x / St::CPR, col = x % St::CPR, h = i * 32 / (16 * St::CPR);
          const long long off16 = row[h] * St::CB + (x % (16 * St::CPR)) * 16;
          const int bytes = (rw & 15) < have[h] ? 16 : 0;
          cp16(st + St::k_at(rw, col), a.p.kc + off16, bytes);
          cp16(st + St::kCodes + St::v_at(rw, col), a.p.vc + off16, bytes);
        }
        constexpr int SP = 16 / St::SB, PPG = 16 / SP;  // rows per 16 bytes of scales; pieces per group
        if (lane < 4 * PPG) {
          const int v = lane / (2 * PPG), x = lane % (2 * PPG), h = x / PPG, rw = x % PPG * SP;
          const int bytes = max(0, min(16, (have[h] - rw) * St::SB));
          const uint8_t* src = (v ? a.p.vs : a.p.ks) + (row[h] + rw) * St::SB;
          cp16(st + 2 * St::kCodes + v * St::kScales + x * 16, src, bytes);
        }
      }
      cp_commit();
      pages_of(c + 1);
    };
    pages_of(c0);
#pragma unroll
    for (int i = 0; i < St::NS - 1; ++i) issue(c0 + i);

    // ---------------------------------------------------------------- q
    const T* qp[2];
    int token[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = tile * kTile + r + 8 * i;
      token[i] = row / a.group;
      qp[i] = row < rows ? static_cast<const T*>(a.q.p) + (sw.v.q0 + token[i]) * a.q.token_stride +
                               (head * a.group + row % a.group) * a.q.head_stride
                         : nullptr;
      if (row >= rows) token[i] = 0;
    }
    uint32_t qh[KS][4], ql[SPLIT ? KS : 1][4];
    float row_scale[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float x[KS][4];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        // the 8 values of block b that this thread's fragments hold
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          float (&w)[4] = x[2 * b + s];
          const int d = Q8 ? 32 * b + 8 * t + 4 * s : 32 * b + 16 * s + 4 * t;
          if (!qp[i]) w[0] = w[1] = w[2] = w[3] = 0.f;
          else if (a.vec) load_act<T, 4, true>(qp[i] + d, w);
          else load_act<T, 4, false>(qp[i] + d, w);
        }
      }
      float most = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(x[k][e]));
      most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
      // times a power of two that puts the largest into [2^10, 2^11)
      const int e = max(60, min(254, static_cast<int>(__float_as_uint(most) >> 23)));
      const float up = __uint_as_float(static_cast<uint32_t>(264 - e) << 23);
      row_scale[i] = score_factor(a.scale * 1.4426950408889634f * __uint_as_float(static_cast<uint32_t>(e - 10) << 23));
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float v0 = x[k][2 * h] * up, v1 = x[k][2 * h + 1] * up;
          const uint32_t hi = pack_f16(v0, v1);
          qh[k][2 * h + i] = hi;
          if (SPLIT) {
            const float2 f = unpack_f16(hi);
            ql[k][2 * h + i] = pack_f16(v0 - f.x, v1 - f.y);
          }
        }
    }

    // ---------------------------------------------------------------- the piece's positions
    float o[NO][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float dref = 0x1p-24f;
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

    for (int c = c0; c < c1; ++c) {
      cp_wait<St::NS - 2>();
      __syncwarp();
      issue(c + St::NS - 1);
      const int p0 = c * kChunk + warp * kGroup;
      if (p0 >= len) continue;
      const uint8_t* st = ring + ((c - c0) % St::NS) * St::kBytes;
      const uint8_t* kcodes = st;
      const uint8_t* vcodes = st + St::kCodes;
      const uint8_t* kscales = st + 2 * St::kCodes;
      const uint8_t* vscales = kscales + St::kScales;

      uint64_t s2[NT][2];  // raw scores of positions 8nt + 2t, + 1; of rows r, r + 8
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int row = 8 * nt + r;
        uint32_t dk[NB];  // scales of positions 8nt + 2t and + 1: block pairs of the one, then of the other
        if (NB == 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(kscales + (8 * nt + 2 * t) * St::SB);
          dk[0] = x.x; dk[1] = x.y; dk[NB - 2] = x.z; dk[NB - 1] = x.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(kscales + (8 * nt + 2 * t) * St::SB);
          dk[0] = x.x; dk[1] = x.y;
        }
        uint64_t dd[NB];  // of the two positions
#pragma unroll
        for (int h = 0; h < NB / 2; ++h) {
          const float2 x = unpack_f16(dk[h]), y = unpack_f16(dk[NB / 2 + h]);
          dd[2 * h] = pair(x.x, y.x);
          dd[2 * h + 1] = pair(x.y, y.y);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          uint32_t w[2];
          if (Q8) {
            const uint2 x = *reinterpret_cast<const uint2*>(kcodes + St::k_at(row, 2 * b + (t >> 1)) + (t & 1) * 8);
            w[0] = x.x;
            w[1] = x.y;
          } else {
            const uint32_t x = *reinterpret_cast<const uint32_t*>(kcodes + St::k_at(row, b) + t * 4);
            w[0] = x & 0x0F0F0F0Fu;
            w[1] = (x >> 4) & 0x0F0F0F0Fu;
          }
          float acc[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t b0 = codes2<0x4140>(w[h], off), b1 = codes2<0x4342>(w[h], off);
            if (h) mma_f16(acc, qh[2 * b + h], b0, b1);
            else mma_f16_first(acc, qh[2 * b], b0, b1);
            if (SPLIT) mma_f16(acc, ql[SPLIT ? 2 * b + h : 0], b0, b1);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint64_t x = pair(acc[2 * i], acc[2 * i + 1]);
            s2[nt][i] = b ? fma2(dd[b], x, s2[nt][i]) : mul2(dd[b], x);
          }
        }
      }

      // ------------------------------------------------------------ mask
      const bool tail = p0 + kGroup > ctx;  // new tokens, or positions behind the sequence
      if (tail) {
        uint32_t vis[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) vis[i] = tree_sees(a, sw.v.q0, token[i], ctx, len, p0);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t v = vis[i] >> (8 * nt + 2 * t);
            s2[nt][i] = pair(v & 1u ? low(s2[nt][i]) : -INFINITY, v & 2u ? high(s2[nt][i]) : -INFINITY);
          }
      }

      // ------------------------------------------------------------ softmax
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) top[i] = max3(top[i], low(s2[nt][i]), high(s2[nt][i]));
      float ref[2], grow[2];
      bool grew = false;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xFFFFFFFFu, top[i], 1));
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xFFFFFFFFu, top[i], 2));
        const float mn = fmaxf(m[i], top[i] * row_scale[i]);
        ref[i] = mn == -INFINITY ? 0.f : mn;
        grow[i] = tex2(m[i] - ref[i]);
        grew = grew || mn > m[i];
        m[i] = mn;
      }
      // V's scales: the largest magnitude of this step against dref (another writer's pool may hold scales below zero)
      uint32_t dv[NT][NB];
      __half2 big = __half2half2(__ushort_as_half(0));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (NB == 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(vscales + (8 * nt + 2 * t) * St::SB);
          dv[nt][0] = x.x; dv[nt][1] = x.y; dv[nt][NB - 2] = x.z; dv[nt][NB - 1] = x.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(vscales + (8 * nt + 2 * t) * St::SB);
          dv[nt][0] = x.x; dv[nt][1] = x.y;
        }
      }
      if (tail) {
        // A scale that is not finite among them (0 times it is NaN): the rows that see
        // its position get NaN in its block of values, however small their weights, and
        // the others are not to meet it.
        const __half2 most = __half2half2(__ushort_as_half(0x7BFF));  // 65504
        bool odd = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < NB; ++h) odd = odd || !__hble2(__habs2(*reinterpret_cast<const __half2*>(&dv[nt][h])), most);
        if (__any_sync(0xFFFFFFFFu, odd)) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t vis = tree_sees(a, sw.v.q0, token[i], ctx, len, p0);
            uint32_t blocks = 0u;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int h = 0; h < 2 * NB; ++h) {  // position h / NB of the two, block h % NB
                const uint32_t d = dv[nt][h / NB * (NB / 2) + h % NB / 2] >> (16 * (h & 1)) & 0x7FFFu;
                if (d > 0x7BFFu && (vis >> (8 * nt + 2 * t + h / NB) & 1u)) blocks |= 1u << (h % NB);
              }
            blocks |= __shfl_xor_sync(0xFFFFFFFFu, blocks, 1);
            blocks |= __shfl_xor_sync(0xFFFFFFFFu, blocks, 2);
#pragma unroll
            for (int b = 0; b < NO; ++b)
              if (blocks >> (b / 4) & 1u) o[b][2 * i] = o[b][2 * i + 1] = NAN;
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < NB; ++h) {
              if ((dv[nt][h] & 0x7FFFu) > 0x7BFFu) dv[nt][h] &= 0xFFFF0000u;
              if ((dv[nt][h] >> 16 & 0x7FFFu) > 0x7BFFu) dv[nt][h] &= 0x0000FFFFu;
            }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int h = 0; h < NB; ++h) big = __hmax2(big, __habs2(*reinterpret_cast<const __half2*>(&dv[nt][h])));
      }
#pragma unroll
      for (int x = 1; x < 4; x <<= 1) big = __hmax2(big, __shfl_xor_sync(0xFFFFFFFFu, big, x));
      const float dmax = fminf(fmaxf(__low2float(big), __high2float(big)), 65504.f);  // an infinite one spoils its block alone
      float shrink = 1.f;
      if (dmax > dref) {  // the same for all lanes
        const float up = __uint_as_float((__float_as_uint(dmax) + 0x7FFFFFu) & 0x7F800000u);
        shrink = dref / up;
        dref = up;
      }
      if (__any_sync(0xFFFFFFFFu, grew) || shrink != 1.f) {
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][e] *= grow[e >> 1] * shrink;
      }
      // Weights times 2^14 / dref, a power of two, so that times V's scales they are
      // at most 2^14.
      const int lift = 14 + 127 - static_cast<int>(__float_as_uint(dref) >> 23);
      const float unlift = dref * 0x1p-14f;
      uint64_t sum2[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float c0 = static_cast<float>(lift) - ref[i];
        const uint64_t rs2 = pair(row_scale[i], row_scale[i]), c2 = pair(c0, c0);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint64_t x = fma2(s2[nt][i], rs2, c2);
          s2[nt][i] = pair(tex2(low(x)), tex2(high(x)));
          sum2[i] = add2(sum2[i], s2[nt][i]);
        }
        l[i] = l[i] * grow[i] + (low(sum2[i]) + high(sum2[i])) * unlift;
      }

      // ------------------------------------------------------------ values
#pragma unroll
      for (int kk = 0; kk < kGroup / 16; ++kk) {
        uint32_t vw[NB][4];  // codes of positions 16kk + {2t, 2t + 1, 2t + 8, 2t + 9}, four dims of each block
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int row = 16 * kk + 2 * t + (k & 1) + 8 * (k >> 1);
            const uint32_t x = *reinterpret_cast<const uint32_t*>(vcodes + St::v_at(row, Q8 ? 2 * b + (r >> 2) : b) + (r & 3) * 4);
            vw[b][k] = Q8 ? x : (x >> (r & 4)) & 0x0F0F0F0Fu;
          }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          uint32_t ph[4], pl[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // positions 16kk + 8h + 2t, + 1
            const int nt = 2 * kk + h;
            const float2 x = unpack_f16(dv[nt][b / 2]), y = unpack_f16(dv[nt][NB / 2 + b / 2]);
            const uint64_t e = b & 1 ? pair(x.y, y.y) : pair(x.x, y.x);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint64_t w = mul2(s2[nt][i], e);
              const float w0 = low(w), w1 = high(w);
              const uint32_t hi = pack_f16(w0, w1);
              ph[2 * h + i] = hi;
              if (SPLIT) {
                const float2 f = unpack_f16(hi);
                pl[2 * h + i] = pack_f16(w0 - f.x, w1 - f.y);
              }
            }
          }
          const uint32_t a01 = __byte_perm(vw[b][0], vw[b][1], 0x5140), a23 = __byte_perm(vw[b][0], vw[b][1], 0x7362);
          const uint32_t b01 = __byte_perm(vw[b][2], vw[b][3], 0x5140), b23 = __byte_perm(vw[b][2], vw[b][3], 0x7362);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t x = i < 2 ? a01 : a23, y = i < 2 ? b01 : b23;
            const uint32_t b0 = i & 1 ? codes2<0x4342>(x, off) : codes2<0x4140>(x, off);
            const uint32_t b1 = i & 1 ? codes2<0x4342>(y, off) : codes2<0x4140>(y, off);
            mma_f16(o[4 * b + i], ph, b0, b1);
            if (SPLIT) mma_f16(o[4 * b + i], pl, b0, b1);
          }
        }
      }
    }
    cp_wait<0>();

    // ---------------------------------------------------------------- join the warps
    constexpr int LD = HD + 4;
    float* jo = reinterpret_cast<float*>(smem);            // [warps][16][LD]
    float* jm = jo + kTreeWarps * kTile * LD;              // [warps][16] maxima, then sums
    float* jl = jm + kTreeWarps * kTile;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 1);
      l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 2);
    }
    __syncthreads();  // every warp is done with its ring
    const float back = dref * 0x1p-14f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float* dst = jo + (warp * kTile + r + 8 * i) * LD;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          const int n = 2 * t + cc;  // column of the fragment
          const int d = Q8 ? 32 * b + 4 * n : 32 * b + 4 * (n & 3) + 16 * (n >> 2);
          const int e = 2 * i + cc;
          *reinterpret_cast<float4*>(dst + d) = make_float4(o[4 * b][e] * back, o[4 * b + 1][e] * back,
                                                            o[4 * b + 2][e] * back, o[4 * b + 3][e] * back);
        }
      if (t == 0) {
        jm[warp * kTile + r + 8 * i] = m[i];
        jl[warp * kTile + r + 8 * i] = l[i];
      }
    }
    __syncthreads();
    {
      constexpr int DPT = HD / 8;  // dims per thread, 8 threads to a row
      const int row = tid >> 3, d0 = (tid & 7) * 4;
      float M = -INFINITY, L = 0.f, O[DPT], f[kTreeWarps];
#pragma unroll
      for (int w = 0; w < kTreeWarps; ++w) M = fmaxf(M, jm[w * kTile + row]);
      const float rf = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int d = 0; d < DPT; ++d) O[d] = 0.f;
#pragma unroll
      for (int w = 0; w < kTreeWarps; ++w) {
        f[w] = tex2(jm[w * kTile + row] - rf);
        L += f[w] * jl[w * kTile + row];
#pragma unroll
        for (int d = 0; d < DPT; d += 4) {
          const float4 x = *reinterpret_cast<const float4*>(jo + (w * kTile + row) * LD + d0 + 8 * d);
          O[d] += f[w] * x.x;
          O[d + 1] += f[w] * x.y;
          O[d + 2] += f[w] * x.z;
          O[d + 3] += f[w] * x.w;
        }
      }
      const int grow_row = tile * kTile + row;
      if (c0 == 0 && c1 == sw.chunks) {
        if (grow_row < rows) {
          T* y = static_cast<T*>(a.out.p) + (sw.v.q0 + grow_row / a.group) * a.out.token_stride +
                 (head * a.group + grow_row % a.group) * a.out.head_stride;
          const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
          for (int d = 0; d < DPT; d += 4)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[d0 + 8 * d + e] = Act<T>::from(L == 0.f ? 0.f : O[d + e] * inv);
        }
      } else {
        float* part = a.parts + static_cast<long long>(2 * blockIdx.x + (c0 == 0)) * Part<HD, kTile>::kFloats;
#pragma unroll
        for (int d = 0; d < DPT; d += 4)
          *reinterpret_cast<float4*>(part + row * HD + d0 + 8 * d) = make_float4(O[d], O[d + 1], O[d + 2], O[d + 3]);
        if ((tid & 7) == 0) {
          part[kTile * HD + row] = M;
          part[kTile * HD + kTile + row] = L;
        }
        if (tid == 0 && c0 == 0) {
          const int end = base_chunk + (in_seq + 1) * sw.chunks;  // the unit's end
          a.desc[blockIdx.x] = make_int4(seq, head, tile, tree_last_cta(share, end));
        }
      }
    }
    __syncthreads();  // the join buffer becomes the ring again
    at += c1 - c0;
  }
  grid_dep_launch();
}

template <class T, int HD, bool Q8>
cudaError_t launch_tree(const TreeArgs& a, int sms, cudaStream_t st) {
  constexpr size_t smem = tree_smem<HD, Q8, Ctas<HD>::kPerSm>();
  cudaError_t e = cudaFuncSetAttribute(k_tree_attn<T, HD, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  const int grid = std::min(kTreeMaxCtas, Ctas<HD>::kPerSm * sms);
  e = serve_launch(k_tree_attn<T, HD, Q8>, dim3(grid), dim3(kTreeThreads), smem, st, false, a);
  if (e != cudaSuccess || a.cap <= kChunk) return e;  // one chunk per unit: none is cut
  return launch_join<T, HD, kTile>(a, grid, st);
}
template <class T>
cudaError_t launch_tree_t(const TreeArgs& a, bool q8, int sms, cudaStream_t st) {
  if (a.p.hd == 64) return q8 ? launch_tree<T, 64, true>(a, sms, st) : launch_tree<T, 64, false>(a, sms, st);
  return q8 ? launch_tree<T, 128, true>(a, sms, st) : launch_tree<T, 128, false>(a, sms, st);
}

// Which form: the one of 128-row tiles (m3g_tree_umma.cu) for 16-bit types where a
// KV head has rows enough and there are 8 chunks for each of its CTAs.  F16 takes
// more rows: K and the weights go into that form in two parts.  Measured, that form
// against this one (32 query over 8 KV heads, Q8_0, 8 sequences of 2700 to 8000
// positions): BF16 of 128 values, 32 rows 66 against 56 us, 48 rows 68 against 75,
// 56 rows 69 against 100, 256 rows 102 against 343; of 64 values, 48 rows 54
// against 50, 64 rows 56 against 62, 128 rows 58 against 114; F16 of 128, 56 rows 85
// against 99, 80 rows 88 against 119, 96 rows 89 against 139; of 64, 64 rows 64
// against 62, 80 rows 65 against 75, 128 rows 66 against 114.  So it is ahead from one
// or two tiles of 16 rows below the borders; they lie where they do since it also
// rounds cached values to f16, which this one takes exactly.  With fewer chunks (BF16, 2
// sequences of 8000, 128 rows, 2000 chunks) 69 against 58 us, with 3000 63 against 80;
// one sequence of 2000 positions, 256 rows, 29 against 28.
constexpr uint64_t kUmmaChunks = 8 * 296;
bool can_use_umma(const m3g_kv_layout* l, uint32_t dtype, uint32_t n_heads, uint32_t max_tokens) {
  const uint64_t least = dtype == M3G_DTYPE_F16 ? 81 : l->head_dim == 128 ? 49 : 65;
  return dtype != M3G_DTYPE_F32 && static_cast<uint64_t>(max_tokens) * (n_heads / l->n_kv_heads) >= least;
}

int check_heads(const m3g_kv_layout* l, uint32_t n_heads) {
  if (!n_heads || n_heads > 32768 || n_heads % l->n_kv_heads)
    return host_fail(M3G_EINVAL, "%u query heads over %u KV heads", n_heads, l->n_kv_heads);
  return M3G_OK;
}

}  // namespace
}  // namespace m3g

extern "C" {

M3G_API int m3g_tree_attn_workspace(const m3g_kv_layout* l, uint32_t dtype, uint32_t n_heads, uint32_t max_tokens,
                                    uint64_t* out) {
  if (!out) return m3g::host_fail(M3G_EINVAL, "null argument");
  *out = 0;
  if (int rc = m3g::kv_check(l)) return rc;
  if (int rc = m3g::check_heads(l, n_heads)) return rc;
  if (!m3g::act_size(dtype)) return m3g::host_fail(M3G_EINVAL, "attention of dtype %u (F32, F16 and BF16 are supported)", dtype);
  const uint64_t tile = m3g::can_use_umma(l, dtype, n_heads, max_tokens) ? m3g::kUmmaTile : m3g::kTile;
  *out = m3g::kTreeMaxCtas * (sizeof(int4) + 2 * sizeof(float) * tile * (l->head_dim + 2));
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
    if (misaligned(r->p, size)) return host_fail(M3G_EINVAL, "rows not aligned to their type");
    if (r->token_stride < 0 || r->head_stride < 0) return host_fail(M3G_EINVAL, "negative stride");
  }
  if ((b->n_tokens > 1 && out->token_stride < a.p.hd) || (n_heads > 1 && out->head_stride < a.p.hd))
    return host_fail(M3G_EINVAL, "result rows overlap");
  if (q->p == out->p && (q->token_stride != out->token_stride || q->head_stride != out->head_stride))
    return host_fail(M3G_EINVAL, "results in place of q need the same strides");
  if (!std::isfinite(scale) || scale < 0.f) return host_fail(M3G_EINVAL, "scale must be finite and not negative");
  if (misaligned(mask, 4)) return host_fail(M3G_EINVAL, "mask not 4-byte aligned");
  if (mask && static_cast<uint64_t>(mask_words) * 32 < b->max_tokens)
    return host_fail(M3G_EINVAL, "%u mask words for %u tokens", mask_words, b->max_tokens);
  uint64_t need = 0;
  if (int rc = m3g_tree_attn_workspace(l, dtype, n_heads, b->max_tokens, &need)) return rc;
  if (!b->n_tokens || !b->n_seqs) return M3G_OK;
  if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)
    return host_fail(M3G_EINVAL, "workspace of %llu bytes (16-byte aligned, %llu needed)",
                     static_cast<unsigned long long>(workspace_bytes), static_cast<unsigned long long>(need));
  a.cap = seq_cap(*b, l->page_size);
  a.n_heads = static_cast<int>(n_heads);
  a.group = static_cast<int>(n_heads / l->n_kv_heads);
  const uint64_t most_rows = static_cast<uint64_t>(b->max_tokens) * a.group;  // of a sequence's KV head
  const uint64_t tiles = (most_rows + kUmmaTile - 1) / kUmmaTile;
  const bool umma = can_use_umma(l, dtype, n_heads, b->max_tokens) &&
                    b->n_seqs * l->n_kv_heads * tiles * ((static_cast<uint64_t>(a.cap) + 63) / 64) >= kUmmaChunks;
  // Chunks that the batch can come to in this form: no sequence has more than
  // max_tokens, all together no more than n_tokens.
  const uint64_t tile = umma ? kUmmaTile : kTile, chunk = umma ? kUmmaChunk : kChunk;
  const uint64_t units = l->n_kv_heads * std::min(b->n_seqs * ((most_rows + tile - 1) / tile),
                                                  static_cast<uint64_t>(b->n_tokens) * a.group / tile + b->n_seqs);
  if (most_rows >= (1ull << 31) || units * ((static_cast<uint64_t>(a.cap) + chunk - 1) / chunk) > kTreeMost)
    return host_fail(M3G_EINVAL, "batch too large (sequences x heads x tokens x length)");
  int dev = 0, sms = 0;
  if (int rc = serve_device(&dev, &a.p.status)) return rc;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return host_fail(M3G_ECUDA, "device attributes");
  a.desc = static_cast<int4*>(workspace);
  a.parts = reinterpret_cast<float*>(a.desc + kTreeMaxCtas);
  a.vec = rows_aligned(q->p, q->token_stride, q->head_stride, size);
  a.vec_out = rows_aligned(out->p, out->token_stride, out->head_stride, size);
  a.b = *b;
  a.q = *q;
  a.out = *out;
  a.mask = mask;
  a.mask_words = static_cast<int>(mask_words);
  a.scale = scale > 0.f ? scale : 1.f / sqrtf(static_cast<float>(a.p.hd));
  const uint64_t wait_us = attn_wait_us();
  a.wait_ns = static_cast<uint32_t>(std::min<uint64_t>(2000, 1000 * wait_us));
  a.wait_polls = static_cast<uint32_t>(std::max<uint64_t>(1, wait_us / 2));
  const cudaStream_t st = serve_stream(stream);
  const bool q8 = l->dtype == M3G_DTYPE_Q8_0;
  const cudaError_t e = umma ? launch_tree_umma(a, dtype, q8, sms, st)
                        : dtype == M3G_DTYPE_F32 ? launch_tree_t<float>(a, q8, sms, st)
                        : dtype == M3G_DTYPE_F16 ? launch_tree_t<__half>(a, q8, sms, st)
                                                 : launch_tree_t<__nv_bfloat16>(a, q8, sms, st);
  if (e != cudaSuccess) return host_fail(M3G_ECUDA, "k_tree_attn: %s", cudaGetErrorString(e));
  return M3G_OK;
}

}  // extern "C"
