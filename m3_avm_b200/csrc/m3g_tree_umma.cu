// m3g_tree_umma.cu -- attention of larger drafted trees on the fifth-generation
// tensor cores (16-bit types; units of 128 rows).
//
// With 128 rows to a tile every cached position costs 128 x HD x 4 flops, which
// mma.sync (16 rows at a time, each tile unpacking the codes anew) turns into
// some ten times the time the cache takes to read.  Here a CTA unpacks a chunk
// of 64 positions once, into f16 tiles in shared memory, and tcgen05.mma
// (M = 128, accumulators in tensor memory) does both products:
//   S[128][64]  = Q[128][HD] K^T       Q, K tiles in shared memory, K-major
//   O[128][HD] += P[128][64] V         P in tensor memory, V tile MN-major
// One thread owns one row: it reads its 64 scores from tensor memory, keeps the
// running maximum and sum in registers without any exchange, and writes its
// weights back over the scores as the next product's operand.  O is rescaled
// only when a row's maximum grows by more than 2^11 over the one its weights
// refer to; all weights carry a factor 2^4, so that small ones stay in f16's
// normal range.
//
// Roundings.  Cached values enter as f16 products code * d (2^-11), or, for F16
// activations, whose own step is as fine, K as two f16 parts (hi + lo, exact)
// in two MMAs and the weights as two (with one, a result was off by 1.6 times what
// rounding it to f16 costs, with two 1.35 times, for 12 % of the time); otherwise
// weights as f16.  A group of 16 positions with a scale past +-500 (a
// value could pass the f16 range) is taken at 2^-7, which its scores or weights
// get back.
//
// Roles (16 warps, two CTAs to an SM, so that one CTA's products and waits
// overlap the other's softmax): a warpgroup for the softmax; one that unpacks K
// and one that unpacks V, each warp 16 positions of the chunk; and four warps
// that only issue: the scores, the results, and the bulk copies that bring K's
// and V's codes and scales (rows of a page are contiguous) two chunks ahead (F16
// over Q8_0 with 128 values has room for one stage: there a copy starts when the chunk
// before it is unpacked).
// Measured: 8 trees of up to 64 tokens over contexts of up to 8190 (256 rows a KV
// head, BF16 over Q8_0) 100 us, 12 trees of 13 over contexts of up to 30011 (104 rows,
// F16 over Q4_0) 280 us.  Neither HBM nor the products bound it (their floors are
// 21 and 44 us): a chunk's softmax and unpacking follow one another, issue slots are
// 60 % used, and waits for tensor memory, barriers and instructions share the rest.
// Polls that hold a waiting thread for 2 us at most are part of that: with the
// hardware's own limit the two cases took 114 and 333 us.
// Scores run one chunk ahead of the weights.  Every role's chain of waits,
// fences and issues is some 1000 cycles a chunk, so each has warps of its own: a
// clock64 trace showed 5100 cycles a chunk with one issuing thread for both
// products, 4700 with the issuing done by the unpacking warps.  Registers go
// from the other groups to the softmax.  256 TMEM columns: two score buffers
// (weights written over them) and O.
//
// Every wait is bounded (wait_polls polls of wait_ns at most).  A role whose wait
// gives up raises the attention-timeout bit and the CTA's abort word, which ends the
// others' waits, and neither issues nor arrives any more: a phase that a barrier
// completes is always one whose work was done.  At the end of the piece the issuing
// warps wait (bounded too) for their products and copies in flight; the rows of
// this piece and of the CTA's later ones become NaN.
#include <type_traits>

#include "m3g_tcgen05.cuh"
#include "m3g_tree.cuh"

namespace m3g {
namespace {

constexpr int kUChunk = kUmmaChunk;
constexpr int kUThreads = 512;                       // softmax, K, V and issuing warpgroups
constexpr int kUCols = 256;                          // TMEM columns of a CTA
constexpr int kOCol = 2 * kUChunk;                   // O behind the two score buffers
constexpr uint32_t kSettlePolls = 1u << 20, kSettleNs = 2000;  // for work in flight when a wait gave up
// log2 of the factor that all weights carry, and of the growth of a row's maximum
// that is let pass: weights stay below 2^15.  Where V's groups at 2^-7 get their
// factor back in the weights, less growth passes.  (A rescaling costs its warp
// some 4000 cycles, and with it the CTA: at a lag of 4 a third of all time.)
constexpr float kLift = 4.f, kLag = 11.f, kLagOddV = 4.f;

// B operand with N contiguous ("MN-major"): bit 16 of the instruction descriptor.
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool b_mn) {
  return idesc_f16_m128(n) | (b_mn ? 1u << 16 : 0u);
}

__device__ __forceinline__ void tc_ld16(uint32_t ta, uint32_t (&x)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]), "=r"(x[8]),
        "=r"(x[9]), "=r"(x[10]), "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15])
      : "r"(ta)
      : "memory");
}

// The load without its wait, and the wait: the values are only used behind it.
__device__ __forceinline__ void tc_ld16_start(uint32_t ta, uint32_t (&x)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]), "=r"(x[8]),
        "=r"(x[9]), "=r"(x[10]), "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15])
      : "r"(ta)
      : "memory");
}
__device__ __forceinline__ void tc_ld_wait(uint32_t (&x)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(x[0]), "+r"(x[1]), "+r"(x[2]), "+r"(x[3]), "+r"(x[4]), "+r"(x[5]), "+r"(x[6]), "+r"(x[7]),
                 "+r"(x[8]), "+r"(x[9]), "+r"(x[10]), "+r"(x[11]), "+r"(x[12]), "+r"(x[13]), "+r"(x[14]), "+r"(x[15])
               :
               : "memory");
}

template <int HD, bool Q8, bool SPLIT>
struct UGeo {
  static constexpr int CB = Q8 ? HD : HD / 2, SB = HD / 16, NB = HD / 32, CPR = CB / 16;
  // Tiles: 16 bytes (8 values of a row) at (dim / 8) * stride + row * 16.  The
  // stride of K and V tiles is 16 bytes off a multiple of 128, so that stores of
  // neighbouring pieces of a row lie in different banks.
  static constexpr int kQStride = 128 * 16, kStride = kUChunk * 16 + 16;
  static constexpr int kQ = HD / 8 * kQStride, kK = HD / 8 * kStride;  // bytes of the Q tile; of a K part or the V tile
  // Stages of 4 x 16 rows: K codes, K scales, V scales each; V codes, V scales each.
  static constexpr int kRawK = 16 * (CB + 2 * SB), kRawV = 16 * (CB + SB);
  static constexpr int NST = SPLIT && Q8 && HD == 128 ? 1 : 2;
  static constexpr int off_k = kQ, off_v = off_k + (SPLIT ? 2 : 1) * kK, off_raw_k = off_v + kK;
  static constexpr int off_raw_v = off_raw_k + 4 * NST * kRawK, kBytes = off_raw_v + 4 * NST * kRawV;
};

struct UBars {
  // Of score buffers: scores there, weights there, weights used.  One barrier per
  // buffer, since softmax and products may be a chunk apart and a wait by parity
  // only tells a phase from the one before it.
  uint64_t s_full[2], p_ready[2], s_free[2];
  uint64_t q_ready, k_ready, k_free, v_ready, pv_done;
  uint64_t raw[2][2], raw_free[2][2];  // [K, V][stage]
};

// A CTA's piece of a unit.
struct UPiece {
  int seq, q0, ctx, len, rows, head, tile, c0, n, whole, last_cta;
};

// The two 16-bit values of a word.
template <class T>
__device__ __forceinline__ float2 two(uint32_t w) {
  if (std::is_same<T, __half>::value) return unpack_f16(w);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

// A value that all lanes of the warp share, in a form that the compiler knows to
// be uniform.  tcgen05 instructions take uniform operands: of values that only
// happen to be equal they are made by a loop over the lanes, some 90
// instructions for each MMA.
template <class T>
__device__ __forceinline__ T uniform(T v) { return __shfl_sync(0xFFFFFFFFu, v, 0); }

__device__ __forceinline__ bool not_finite(__half d) { return (__half_as_ushort(d) & 0x7FFFu) > 0x7BFFu; }

// One lane of a converged warp.
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

template <int R>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }

// 16 codes as 8 f16 pairs, times d; lo: what the rounding left (exact).
template <bool Q8, bool LO>
__device__ __forceinline__ void unpack16(const uint32_t (&w)[4], __half2 d, uint4 (&hi)[2], uint4 (&lo)[2]) {
  const __half2 off = __half2half2(__ushort_as_half(Q8 ? 0x6480 : 0x6408));  // 1152, 1032
  uint32_t h[8], l[8];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t x = __byte_perm(w[i], 0x64646464u, j ? 0x4342 : 0x4140);  // 1024 + code
      const __half2 c = __hsub2(*reinterpret_cast<const __half2*>(&x), off);
      const __half2 p = __hmul2(c, d);
      h[2 * i + j] = *reinterpret_cast<const uint32_t*>(&p);
      if (LO) {
        const __half2 q = __hfma2(c, d, __hneg2(p));
        l[2 * i + j] = *reinterpret_cast<const uint32_t*>(&q);
      }
    }
  hi[0] = make_uint4(h[0], h[1], h[2], h[3]);
  hi[1] = make_uint4(h[4], h[5], h[6], h[7]);
  if (LO) {
    lo[0] = make_uint4(l[0], l[1], l[2], l[3]);
    lo[1] = make_uint4(l[4], l[5], l[6], l[7]);
  }
}

// Which 16-byte piece of a warp's 16 rows lane `lane` takes in step `j`: eight
// neighbouring lanes read 128 different bytes mod 128, and with the tiles' odd
// stride store into different banks (4-bit rows of 64 bytes: two by two).
template <int CPR>
__device__ __forceinline__ void piece_of(int j, int lane, int& key, int& col) {
  if (CPR == 8) {
    const int b = (lane >> 2) & 1;  // four pieces of one row, the other four of the next
    key = 2 * ((lane >> 3) + 4 * (j >> 1)) + b;
    col = (lane & 3) + 4 * (b ^ (j & 1));
  } else {
    key = (j * 32 + lane) / CPR;
    col = (j * 32 + lane) % CPR;
  }
}

// A warp's 16 rows into rows trow0 .. of the tiles.
template <class G, bool Q8, bool LO>
__device__ __forceinline__ void unpack_rows(const uint8_t* codes, const __half (&d)[G::CPR / 2], uint8_t* tile_hi,
                                            uint8_t* tile_lo, int trow0, int lane) {
#pragma unroll
  for (int j = 0; j < G::CPR / 2; ++j) {
    int key, col;
    piece_of<G::CPR>(j, lane, key, col);
    const uint4 x = *reinterpret_cast<const uint4*>(codes + key * G::CB + col * 16);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int q = 0; q < (Q8 ? 1 : 2); ++q) {  // 4 bits: the low nibbles are the block's first 16 values
      uint32_t y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = Q8 ? w[i] : (w[i] >> (4 * q)) & 0x0F0F0F0Fu;
      uint4 hi[2], lo[2];
      unpack16<Q8, LO>(y, __half2half2(d[j]), hi, lo);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int o = (Q8 ? 2 * col + h : 4 * col + 2 * q + h) * G::kStride + (trow0 + key) * 16;
        *reinterpret_cast<uint4*>(tile_hi + o) = hi[h];
        if (LO) *reinterpret_cast<uint4*>(tile_lo + o) = lo[h];
      }
    }
  }
}

template <class T, int HD, bool Q8, bool SPLIT>
__global__ void __launch_bounds__(kUThreads, 2) k_tree_umma(const __grid_constant__ TreeArgs a) {
  using G = UGeo<HD, Q8, SPLIT>;
  constexpr int NB = G::NB, CPR = G::CPR, PPL = CPR / 2, NST = G::NST;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ ShareScratch scratch;
  __shared__ UBars bar;
  __shared__ UPiece pc;
  __shared__ uint32_t tslot;
  __shared__ int abort_word;
  // Of a chunk's groups of 16 positions: 1 K, 2 V at 2^-7, 4 a scale of V that is not
  // finite in a tail; and of a tail chunk's positions the blocks of V with such scales.  Four chunks
  // deep: K is unpacked at most three ahead of a softmax that still reads.
  __shared__ __align__(16) int odd[4][4];
  __shared__ uint32_t v_nan[4][kUChunk];
  __shared__ int held[2][2][4];  // [K, V][stage]: positions that each group of 16 has (0: behind the end, bad page)
  const int tid = threadIdx.x, lane = tid & 31, warp = uniform(tid >> 5), group = warp >> 2, gw = warp & 3;
  volatile int* abort_flag = &abort_word;
  TreeShare share;
  if (!tree_share<kUChunk, kUmmaTile, kUThreads, 4>(a, scratch, share)) return;
  if (tid == 0) {
    mbar_init(&bar.q_ready, 4);
    mbar_init(&bar.k_ready, 4);
    mbar_init(&bar.k_free, 1);
    mbar_init(&bar.v_ready, 4);
    mbar_init(&bar.pv_done, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.s_full[i], 1);
      mbar_init(&bar.p_ready[i], 4);
      mbar_init(&bar.s_free[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bar.raw[i >> 1][i & 1], 4);
      mbar_init(&bar.raw_free[i >> 1][i & 1], 4);
    }
    abort_word = 0;
    fence_mbar_init();
  }
  if (warp == 4) {
    tc_alloc(&tslot, kUCols);
    tc_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = uniform(tslot);
  // Short: with 16 warps in four roles the kernel's loops have to stay within the
  // instruction caches (with everything unrolled and inlined waits for instructions
  // were the largest stall).
  auto wait_one = [&](uint64_t* b, uint32_t parity) -> bool {  // by one lane; false: gave up
    uint32_t polls = 0;
    while (!mbar_try_wait_for(b, parity, a.wait_ns)) {
      if (++polls < a.wait_polls && !*abort_flag) continue;
      if (!*abort_flag) atomicOr(a.p.status, kStatusAttnTimeout);
      *abort_flag = 1;
      return false;
    }
    return true;
  };
  auto wait = [&](uint64_t* b, uint32_t parity) -> bool {  // by a warp, the same for all lanes
    return __all_sync(0xFFFFFFFFu, wait_one(b, parity));
  };
  auto aborted = [&]() -> bool { return __any_sync(0xFFFFFFFFu, *abort_flag); };
  // The first thread of the V group finds the CTA's pieces.
  int at_seq = share.seq, at = share.first, before = share.before;
  auto next_piece = [&] {
    pc.n = 0;
    if (at >= share.last) return;
    bool bad = false;
    SeqWork<kUChunk, kUmmaTile> w(a, at_seq, &bad);
#pragma unroll 1
    while (at >= before + w.total(a.p.kvh)) {
      before += w.total(a.p.kvh);
      w = SeqWork<kUChunk, kUmmaTile>(a, ++at_seq, &bad);
    }
    const int unit = (at - before) / w.chunks;
    pc.c0 = at - before - unit * w.chunks;
    pc.n = min(w.chunks - pc.c0, share.last - at);
    pc.seq = at_seq;
    pc.q0 = w.v.q0;
    pc.ctx = w.v.ctx;
    pc.len = w.v.ctx + w.v.n;
    pc.rows = w.v.n * a.group;
    pc.head = unit / w.tiles;
    pc.tile = unit - pc.head * w.tiles;
    pc.whole = pc.n == w.chunks;
    pc.last_cta = tree_last_cta(share, before + (unit + 1) * w.chunks);
    at += pc.n;
  };

  // Chunks are counted through the pieces: chunk `it + c` has that phase of every barrier.
  if (group == 0) {
    // -------------------------------------------------------------- q, softmax, result: one row per thread
    regs_up<112>();
    uint32_t it = 0;
#pragma unroll 1
    for (int pn = 0;; ++pn) {
      __syncthreads();
      const int n = uniform(pc.n);
      if (!n) break;
      const int row = pc.tile * kUmmaTile + tid;
      const bool live = row < pc.rows;
      const int token = live ? row / a.group : 0, hq = pc.head * a.group + row % a.group;
      bool dead = aborted();  // the rows of this piece become NaN
      float cs = 0.f;         // factor of the raw scores, in base 2
      if (!dead) {
        // This thread's row, read for its largest value and read again, times a power of two that puts its largest into
        // [2^4, 2^5): room for K's f16 range in the f32 sums.
        const T* q = static_cast<const T*>(a.q.p) + (pc.q0 + token) * a.q.token_stride + hq * a.q.head_stride;
        constexpr int PART = 8;  // 16-byte loads in flight
        if (!(live && a.vec)) {  // rows that are not aligned go through their place in the tile
#pragma unroll 1
          for (int i = 0; i < HD; ++i)
            reinterpret_cast<T*>(smem + (i / 8) * G::kQStride + tid * 16)[i % 8] = live ? q[i] : Act<T>::from(0.f);
        }
        auto load = [&](int i) {
          return live && a.vec ? reinterpret_cast<const uint4*>(q)[i]
                               : *reinterpret_cast<const uint4*>(smem + i * G::kQStride + tid * 16);
        };
        uint4 x[PART];
        float most = 0.f;
#pragma unroll 1
        for (int i0 = 0; i0 < HD / 8; i0 += PART) {
#pragma unroll
          for (int i = 0; i < PART; ++i) x[i] = load(i0 + i);
#pragma unroll
          for (int i = 0; i < PART; ++i) {
            const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 v = two<T>(w[k]);
              most = max3(most, fabsf(v.x), fabsf(v.y));
            }
          }
        }
        const int e = max(60, min(254, static_cast<int>(__float_as_uint(most) >> 23)));
        const float up = __uint_as_float(static_cast<uint32_t>(258 - e) << 23);
        cs = score_factor(a.scale * 1.4426950408889634f * __uint_as_float(static_cast<uint32_t>(e - 4) << 23));
#pragma unroll 1
        for (int i0 = 0; i0 < HD / 8; i0 += PART) {
#pragma unroll
          for (int i = 0; i < PART; ++i) x[i] = load(i0 + i);
#pragma unroll
          for (int i = 0; i < PART; ++i) {
            uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 v = two<T>(w[k]);
              w[k] = pack_f16(v.x * up, v.y * up);
            }
            *reinterpret_cast<uint4*>(smem + (i0 + i) * G::kQStride + tid * 16) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.q_ready);
      }
      const uint32_t tl = tbase + (static_cast<uint32_t>(32 * warp) << 16);
      float m = -INFINITY, l = 0.f;
      uint32_t nan_blocks = 0u;
#pragma unroll 1
      for (int c = 0; c < n && !dead; ++c) {
        const uint32_t ph = it + c;
        const int buf = ph & 1, p0 = (pc.c0 + c) * kUChunk;
        const bool tail = p0 + kUChunk > pc.ctx;
        uint32_t vis[2] = {~0u, ~0u};
        if (tail) {
          vis[0] = tree_sees(a, pc.q0, token, pc.ctx, pc.len, p0);
          vis[1] = tree_sees(a, pc.q0, token, pc.ctx, pc.len, p0 + 32);
        }
        if (!wait(&bar.s_full[buf], (ph >> 1) & 1)) {
          dead = true;
          break;
        }
        tc_fence_after();
        const int4 od = *reinterpret_cast<const int4*>(odd[ph & 3]);
        const int flags[4] = {od.x, od.y, od.z, od.w};
        const float lag = (od.x | od.y | od.z | od.w) & 2 ? kLagOddV : kLag;
        // Some row of the warp refers to a larger maximum from now on; false: a wait gave up.
        auto rescale = [&](float mx, bool grows) -> bool {
          const float f = grows ? tex2(m - mx) : 1.f;
          if (grows) {
            m = mx;
            l *= f;
          }
          if (c > 0) {
            if (!wait(&bar.s_free[buf ^ 1], ((ph - 1) >> 1) & 1)) return false;  // the results so far are there
            tc_fence_after();
#pragma unroll 1
            for (int h = 0; h < HD / 16; ++h) {
              uint32_t x[16];
              tc_ld16(tl + kOCol + 16 * h, x);
#pragma unroll
              for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * f);
              tc_st16(tl + kOCol + 16 * h, x);
            }
          }
          return true;
        };
        // The scores of a group of 16 positions, read while the one before is worked on.
        uint32_t x[2][16];
        auto scores = [&](int h) -> uint32_t(&)[16] {
          uint32_t(&s)[16] = x[h & 1];
          tc_ld_wait(s);
          if (h + 1 < kUChunk / 16) tc_ld16_start(tl + buf * kUChunk + 16 * (h + 1), x[(h + 1) & 1]);
          if (tail) {
#pragma unroll
            for (int j = 0; j < 16; ++j) s[j] = vis[h >> 1] >> (16 * (h & 1) + j) & 1u ? s[j] : 0xFF800000u;  // -inf
          }
          return s;
        };
        float sum = 0.f;
        if constexpr (SPLIT) {  // the maximum first, then the weights, each group's in the place of its scores
          float mx = -INFINITY;
          tc_ld16_start(tl + buf * kUChunk, x[0]);
#pragma unroll
          for (int h = 0; h < kUChunk / 16; ++h) {
            const uint32_t(&s)[16] = scores(h);
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 16; j += 2) top = max3(top, __uint_as_float(s[j]), __uint_as_float(s[j + 1]));
            mx = fmaxf(mx, top * (flags[h] & 1 ? 128.f * cs : cs));
          }
          const bool grows = mx > m + lag || (m == -INFINITY && mx > -INFINITY);
          if (__any_sync(0xFFFFFFFFu, grows) && !rescale(mx, grows)) {
            dead = true;
            break;
          }
          const float ref = m == -INFINITY ? 0.f : m - kLift;
          tc_ld16_start(tl + buf * kUChunk, x[0]);
#pragma unroll
          for (int h = 0; h < kUChunk / 16; ++h) {
            const float csk = flags[h] & 1 ? 128.f * cs : cs, refv = flags[h] & 2 ? ref - 7.f : ref;
            const uint64_t cs2 = pair(csk, csk), ref2 = pair(-refv, -refv);
            const uint32_t(&s)[16] = scores(h);
            uint32_t p[16];
            uint64_t part = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const uint64_t t = fma2(pair(__uint_as_float(s[2 * j]), __uint_as_float(s[2 * j + 1])), cs2, ref2);
              const float w0 = tex2(low(t)), w1 = tex2(high(t));
              part = add2(part, pair(w0, w1));
              p[j] = pack_f16(w0, w1);
              const float2 hi = unpack_f16(p[j]);
              p[8 + j] = pack_f16(w0 - hi.x, w1 - hi.y);
            }
            sum += (low(part) + high(part)) * (flags[h] & 2 ? 0x1p-7f : 1.f);
            tc_st16(tl + buf * kUChunk + 16 * h, p);
          }
        } else {
          // One pass takes the maximum and, with the reference so far, the weights;
          // where a row's maximum grows past the lag they are taken again.
          uint32_t p[32];
#pragma unroll 1
          for (;;) {
            const float ref = m == -INFINITY ? 0.f : m - kLift;
            float mx = -INFINITY;
            sum = 0.f;
            tc_ld16_start(tl + buf * kUChunk, x[0]);
#pragma unroll
            for (int h = 0; h < kUChunk / 16; ++h) {
              // a group at 2^-7: its scores, or its weights, get it back
              const float csk = flags[h] & 1 ? 128.f * cs : cs, refv = flags[h] & 2 ? ref - 7.f : ref;
              const uint64_t cs2 = pair(csk, csk), ref2 = pair(-refv, -refv);
              const uint32_t(&s)[16] = scores(h);
              float top = -INFINITY;
              uint64_t part = 0;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float s0 = __uint_as_float(s[2 * j]), s1 = __uint_as_float(s[2 * j + 1]);
                top = max3(top, s0, s1);
                const uint64_t t = fma2(pair(s0, s1), cs2, ref2);
                const float w0 = tex2(low(t)), w1 = tex2(high(t));
                part = add2(part, pair(w0, w1));
                p[8 * h + j] = pack_f16(w0, w1);
              }
              mx = fmaxf(mx, top * csk);
              sum += (low(part) + high(part)) * (flags[h] & 2 ? 0x1p-7f : 1.f);
            }
            const bool grows = mx > m + lag || (m == -INFINITY && mx > -INFINITY);
            if (!__any_sync(0xFFFFFFFFu, grows)) break;
            if (!rescale(mx, grows)) {
              dead = true;
              break;
            }
          }
          if (dead) break;
          tc_st16(tl + buf * kUChunk, *reinterpret_cast<uint32_t(*)[16]>(&p[0]));
          tc_st16(tl + buf * kUChunk + 16, *reinterpret_cast<uint32_t(*)[16]>(&p[16]));
        }
        l += sum;
        if ((od.x | od.y | od.z | od.w) & 4) {
#pragma unroll 1
          for (int j = 0; j < kUChunk; ++j)
            if ((odd[ph & 3][j / 16] & 4) && (vis[j / 32] >> (j & 31) & 1u)) nan_blocks |= v_nan[ph & 3][j];
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.p_ready[buf]);
      }
      if (!dead) dead = !wait(&bar.s_free[(it + n - 1) & 1], ((it + n - 1) >> 1) & 1);
      tc_fence_after();
      if (dead) {  // a NaN sum makes what is joined from this piece NaN too
        m = 0.f;
        l = NAN;
      }
      {
        const bool whole = pc.whole;
        float* part = a.parts + static_cast<long long>(2 * blockIdx.x + (pc.c0 == 0)) * Part<HD, kUmmaTile>::kFloats;
        T* y = static_cast<T*>(a.out.p) + (pc.q0 + token) * a.out.token_stride + hq * a.out.head_stride;
        const float f = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
#pragma unroll 1
        for (int h = 0; h < HD / 16; ++h) {
          uint32_t x[16];
          if (dead) {
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = 0x7FC00000u;
          } else {
            tc_ld16(tl + kOCol + 16 * h, x);
          }
          if (live) {
#pragma unroll
            for (int q = 0; q < 16; q += 8) {
              float o[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                o[j] = __uint_as_float(x[q + j]) * f;
                if (nan_blocks >> (h >> 1) & 1u) o[j] = NAN;
                if (l == 0.f) o[j] = 0.f;  // sees nothing
              }
              if (!whole) store_act<float, 8, true>(part + tid * HD + 16 * h + q, o);
              else if (a.vec_out) store_act<T, 8, true>(y + 16 * h + q, o);
              else store_act<T, 8, false>(y + 16 * h + q, o);
            }
          }
          __syncwarp();
        }
        if (!whole && live) {
          part[kUmmaTile * HD + tid] = m;
          part[kUmmaTile * HD + kUmmaTile + tid] = l;
        }
        if (tid == 0 && !whole && pc.c0 == 0) a.desc[blockIdx.x] = make_int4(pc.seq, pc.head, pc.tile, pc.last_cta);
      }
      tc_fence_before();
      it += n;
      __syncthreads();
    }
  } else if (group < 3) {
    // -------------------------------------------------------------- K (group 1) and V: 16 positions of each chunk
    regs_down<56>();
    const bool is_v = group == 2;
    const uint8_t* raw = smem + (is_v ? G::off_raw_v + gw * G::kRawV : G::off_raw_k + gw * G::kRawK);
    const int raw_stage = 4 * (is_v ? G::kRawV : G::kRawK);
    uint32_t it = 0;
#pragma unroll 1
    for (int pn = 0;; ++pn) {
      if (tid == 256) next_piece();
      __syncthreads();
      const int n = uniform(pc.n);
      if (!n) break;
      const int first_tail = (pc.ctx / kUChunk) - pc.c0;  // the first chunk with new tokens
      const int todo = aborted() ? 0 : n;
#pragma unroll 1
      for (int c = 0; c < todo; ++c) {
        const uint32_t ph = it + c, rs = ph % NST;
        const uint8_t* st = raw + rs * raw_stage;
        if (!wait(&bar.raw[is_v][rs], (ph / NST) & 1)) break;
        const int have = held[is_v][rs][gw];
        // scales of this lane's pieces, and (K's warps) of its share of the group's V blocks
        __half d[PPL];
        bool plain = true;
        const __half lim = __float2half_rn(500.f);
        const __half* sc = reinterpret_cast<const __half*>(st + 16 * G::CB);
#pragma unroll
        for (int j = 0; j < PPL; ++j) {
          int key, col;
          piece_of<CPR>(j, lane, key, col);
          const int at16 = key * NB + (Q8 ? col >> 1 : col);
          d[j] = key < have ? sc[at16] : __ushort_as_half(0);
          const __half dv = is_v ? d[j] : key < have ? sc[16 * NB + at16] : __ushort_as_half(0);
          plain = plain && __habs(d[j]) <= lim && __habs(dv) <= lim;  // NaN: not plain
        }
        int flags = 0;
        if (!__all_sync(0xFFFFFFFFu, plain)) {
          int odd_k = 0, odd_v = 0;
#pragma unroll 1
          for (int b = lane; b < 16 * NB; b += 32) {
            if (b / NB >= have) continue;
            const __half dv = sc[is_v ? b : 16 * NB + b];
            odd_k |= !is_v && __habs(sc[b]) > lim;
            odd_v |= (__habs(dv) > lim ? 1 : 0) | (not_finite(dv) ? 2 : 0);
          }
          flags = (__any_sync(0xFFFFFFFFu, odd_k) ? 1 : 0) | (__any_sync(0xFFFFFFFFu, odd_v & 1) ? 2 : 0) |
                  (__any_sync(0xFFFFFFFFu, odd_v & 2) && c >= first_tail ? 4 : 0);
        }
        // K's tile is free once the last chunk's scores are done, V's once its results are.
        if (c > 0 && !wait(is_v ? &bar.pv_done : &bar.k_free, (ph - 1) & 1)) break;
        if (!is_v && lane == 0) odd[ph & 3][gw] = flags;
        if (flags & (is_v ? 2 : 1)) {
#pragma unroll
          for (int j = 0; j < PPL; ++j) d[j] = __hmul(d[j], __float2half_rn(0x1p-7f));
        }
        if (flags & 4) {  // a row that does not see a position must not meet 0 times it: NaN is put back at the end
          if (is_v) {
#pragma unroll
            for (int j = 0; j < PPL; ++j)
              if (not_finite(d[j])) d[j] = __ushort_as_half(0);
          } else if (lane < 16) {
            uint32_t blocks = 0u;
#pragma unroll 1
            for (int b = 0; b < NB; ++b)
              if (lane < have && not_finite(sc[(16 + lane) * NB + b]))
                blocks |= 1u << b;
            v_nan[ph & 3][16 * gw + lane] = blocks;
          }
          __syncwarp();
        }
        if constexpr (SPLIT) {
          if (is_v) unpack_rows<G, Q8, false>(st, d, smem + G::off_v, nullptr, 16 * gw, lane);
          else unpack_rows<G, Q8, true>(st, d, smem + G::off_k, smem + G::off_k + G::kK, 16 * gw, lane);
        } else {
          unpack_rows<G, Q8, false>(st, d, smem + (is_v ? G::off_v : G::off_k), nullptr, 16 * gw, lane);
        }
        fence_proxy_async_smem();  // the tile's writes before the product reads it; the stage's reads before it is refilled
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(is_v ? &bar.v_ready : &bar.k_ready);
          mbar_arrive(&bar.raw_free[is_v][rs]);
        }
      }
      it += n;
      __syncthreads();
    }
  } else {
    // -------------------------------------------------------------- the issuing warps
    regs_down<32>();
    uint32_t it = 0;
    const uint64_t policy = l2_evict_first_policy();
#pragma unroll 1
    for (int pn = 0;; ++pn) {
      __syncthreads();
      const int n = uniform(pc.n);
      if (!n) break;
      const int todo = aborted() ? 0 : n;
      int c = 0;  // chunks that this lane has issued
      if (gw == 0) {
        if (todo && elect()) {
        // S = Q K^T, into the buffer whose weights are used
        // (a descriptor's low 14 bits are the address in 16-byte units: steps are added to it)
        const uint64_t q0 = smem_desc(smem_addr(smem), G::kQStride, 128);
        const uint64_t k0 = smem_desc(smem_addr(smem + G::off_k), G::kStride, 128);
        const bool ready = wait_one(&bar.q_ready, pn & 1);
#pragma unroll 1
        for (; ready && c < todo; ++c) {
          const uint32_t ph = it + c, buf = ph & 1;
          if (!wait_one(&bar.k_ready, ph & 1)) break;
          if (c >= 2 && !wait_one(&bar.s_free[buf], ((ph >> 1) - 1) & 1)) break;
          tc_fence_after();
#pragma unroll
          for (int part = 0; part < (SPLIT ? 2 : 1); ++part)
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
              tc_mma_ss(tbase + buf * kUChunk, q0 + k * 2 * G::kQStride / 16,
                        k0 + (part * G::kK + k * 2 * G::kStride) / 16, idesc_f16(kUChunk, false), part || k);
          tc_commit(&bar.s_full[buf]);
          tc_commit(&bar.k_free);
        }
        }
      } else if (gw == 1) {
        if (todo && elect()) {
        // O += P V
        const uint64_t v0 = smem_desc(smem_addr(smem + G::off_v), 128, G::kStride);
#pragma unroll 1
        for (; c < todo; ++c) {
          const uint32_t ph = it + c, buf = ph & 1;
          if (!wait_one(&bar.v_ready, ph & 1)) break;
          if (!wait_one(&bar.p_ready[buf], (ph >> 1) & 1)) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < kUChunk / 16; ++k)
#pragma unroll
            for (int part = 0; part < (SPLIT ? 2 : 1); ++part)
              tc_mma_ts(tbase + kOCol, tbase + buf * kUChunk + (SPLIT ? 16 : 8) * k + 8 * part, v0 + k * 256 / 16,
                        idesc_f16(HD, true), c > 0 || k > 0 || part > 0);
          tc_commit(&bar.s_free[buf]);
          tc_commit(&bar.pv_done);
        }
        }
      } else if (lane < 4) {
        // K's (V's) codes and scales; lane g: positions 16g .. of each chunk
        const bool is_v = gw == 3;
        const int first = pc.c0 * kUChunk + 16 * lane;
        const int32_t* table = a.b.page_table + static_cast<long long>(pc.seq) * a.b.max_pages;
        auto page_of = [&](int c) {
          const int p0 = first + c * kUChunk;
          return c < n && p0 < pc.len ? table[p0 >> a.p.page_shift] : 0;
        };
        int page = page_of(0);
#pragma unroll 1
        for (; c < todo; ++c) {
          const uint32_t ph = it + c, rs = ph % NST;
          const int ahead = page_of(c + 1), p0 = first + c * kUChunk;
          // all four lanes or none, so that a stage that one has copies for completes
          if (!__all_sync(0xFu, ph < NST || wait_one(&bar.raw_free[is_v][rs], (ph / NST - 1) & 1))) break;
          const bool there = page >= 0 && page < a.p.n_pages;
          const int have = there ? max(0, min(16, pc.len - p0)) : 0;
          held[is_v][rs][lane] = have;
          uint64_t* full = &bar.raw[is_v][rs];
          if (have) {
            const long long r0 = kv_row(a.p, page, pc.head, p0 & (a.p.page_size - 1));
            const int bytes = is_v ? G::kRawV : G::kRawK;
            uint8_t* dst = smem + (is_v ? G::off_raw_v : G::off_raw_k) + (rs * 4 + lane) * bytes;
            mbar_arrive_expect_tx(full, bytes);
            bulk_g2s(dst, (is_v ? a.p.vc : a.p.kc) + r0 * G::CB, 16 * G::CB, full, policy);
            dst += 16 * G::CB;
            if (!is_v) {
              bulk_g2s(dst, a.p.ks + r0 * G::SB, 16 * G::SB, full, policy);
              dst += 16 * G::SB;
            }
            bulk_g2s(dst, a.p.vs + r0 * G::SB, 16 * G::SB, full, policy);
          } else {
            if (!there && p0 < pc.len && !is_v) atomicOr(a.p.status, kStatusBadPage);
            mbar_arrive(full);
          }
          page = ahead;
        }
      }
      __syncwarp();
      it += n;
      __syncthreads();
      if (*abort_flag && c > 0) {  // products and copies in flight: of the last phases issued
        const uint32_t last = it - n + c - 1;
        auto settle = [&](uint64_t* b, uint32_t parity) {
          for (uint32_t i = 0; i < kSettlePolls && !mbar_try_wait_for(b, parity, kSettleNs); ++i) {
          }
        };
        if (gw < 2) {
          settle(gw ? &bar.pv_done : &bar.k_free, last & 1);
        } else {
#pragma unroll 1
          for (uint32_t k = 0; k < NST && k <= last; ++k)
            settle(&bar.raw[gw == 3][(last - k) % NST], ((last - k) / NST) & 1);
        }
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) tc_dealloc(tbase, kUCols);
  grid_dep_launch();
}

template <class T, int HD, bool Q8>
cudaError_t launch_umma(const TreeArgs& a, int sms, cudaStream_t st) {
  constexpr bool SPLIT = std::is_same<T, __half>::value;
  constexpr int smem = UGeo<HD, Q8, SPLIT>::kBytes;
  static_assert(2 * (smem + 4096) <= 228 * 1024, "two CTAs per SM");
  const auto kern = k_tree_umma<T, HD, Q8, SPLIT>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const int grid = 2 * sms < kTreeMaxCtas ? 2 * sms : kTreeMaxCtas;
  e = serve_launch(kern, dim3(grid), dim3(kUThreads), smem, st, false, a);
  if (e != cudaSuccess || a.cap <= kUChunk) return e;  // one chunk per unit: none is cut
  return launch_join<T, HD, kUmmaTile>(a, grid, st);
}

template <class T>
cudaError_t launch_umma_t(const TreeArgs& a, bool q8, int sms, cudaStream_t st) {
  if (a.p.hd == 64) return q8 ? launch_umma<T, 64, true>(a, sms, st) : launch_umma<T, 64, false>(a, sms, st);
  return q8 ? launch_umma<T, 128, true>(a, sms, st) : launch_umma<T, 128, false>(a, sms, st);
}

}  // namespace

cudaError_t launch_tree_umma(const TreeArgs& a, uint32_t dtype, bool q8, int sms, cudaStream_t st) {
  return dtype == M3G_DTYPE_F16 ? launch_umma_t<__half>(a, q8, sms, st) : launch_umma_t<__nv_bfloat16>(a, q8, sms, st);
}

}  // namespace m3g
