// kernels_paged_attn.h -- attention of a sequence's newest tokens over a cache in pages.
//
//   s_p = scale (q . k_p) for p <= the row's position;  w = softmax(s);  o = sum_p w_p v_p
//
// Bound: the cache's bytes (4 hd per position and KV head, against 4 hd flop per position and row),
// so the kernel's work is to keep HBM busy whatever the batch looks like.  Heads of 128:
//   4 sequences of 65536, 32 + 8 heads: 165 + 5 us (split + join), 6.5 TB/s in the split
//   64 of up to 4001, 24 + 8 heads: 90 + 5 us, 6.0 TB/s
//   1 of 8199, 32 + 8 heads: 9.4 + 4.3 us for 34 MB: latency (launch 1, plan 1.2, pages 0.6, K and V and
//     the query operands 2, products and softmax 1.4, states joined and written 1.3, then the join's launch)
//   16 of up to 1100, up to 5 new tokens, weights kept: 16.8 + 6.4 us for 39 MB: the same, two tiles a wave
//
// Split.  A segment is (sequence, KV head, block of 16 NR query rows); its tiles are 32 positions.
// The query rows are the new tokens times the KV head's query heads, so K and V are read once for
// all of them.  A segment is cut into pieces of about equal size, none above `target` tiles, which
// comes from the batch's tiles altogether; a workgroup does one piece.  Every wave of every workgroup
// works the plan out from lens (a captured graph follows growing caches).  A segment of one piece is
// finished there; of the others each piece writes its part (maximum, sum, unnormalised rows), and
// k_pa_join joins them.
//
// Inside a workgroup the 4 waves take a segment's tiles in turn, each with a softmax state of its own,
// joined through LDS at the segment's end.  A wave reads its K and V granules (16 bytes: 8 dims of a
// position, 8 positions of a dim) straight into the operand layout of v_mfma_f32_16x16x32:
//   S^T = K Q^T, two 16-position products whose rows are the positions 8 (r / 4) + r % 4 and + 4, so
//   that lane group l / 16 ends up with the 8 consecutive positions of one V granule, which is what
//   O^T = V^T P^T reads as its second operand: P never leaves the lane.
// K of the next tile is in flight from the moment the scores are done, V of the next from the
// moment the products are: about 16 KB a wave outstanding.
//
// Numbers.  f32 queries are the sum of two f16 (22 bits) or of three bf16, a row scaled by a power of two
// into their range, 16-bit queries are used as they are; the weights exp2(s - max) are the sum of
// two f16 (22 bits) or of three bf16 (all 24 of them).  f16 weights carry a factor 2^14: a term's steps are
// 2^-39 of the row's largest weight at least.  bf16 weights carry 2^-24: the sum over 2^24 positions at most
// of values near the largest f32 stays below it (products below f32's subnormals vanish: 2^-126 of an output).
#pragma once
#include <type_traits>
#include "kernels_paged.h"

namespace cm {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int PA_NT = 256;
constexpr uint32_t PA_TILE = 32;
constexpr float PA_LOWEST = -3.402823466e38f;
constexpr float PA_LOG2E = 1.4426950408889634f;

struct PaArgs {
  Paged g;
  const void* q;
  const uint32_t* new_lens;
  const uint16_t* kc;
  const uint16_t* vc;
  void* out;
  float* scores;   // [seq][kv head][row][cap], log2 domain; null: no weights kept
  float* stats;    // [seq][kv head][row][2]: maximum and sum of the rows of uncut segments
  uint2* cuts;     // [seq][kv head][block]: a segment's first slot and its pieces
  float* part_ml;  // [slot][row of the block][2]
  float* part_o;   // [slot][row of the block][hd]
  float* weights;
  float scale;
  float p_bits;    // weights are held times 2^p_bits
  uint32_t q_stride, out_stride, n_new, n_heads;
  uint32_t at_once;   // pieces that run at the same time
  uint32_t blocks;    // row blocks of a sequence with n_new new tokens
  uint32_t part_rows; // rows of a slot
  uint32_t group;       // query heads of a KV head
  uint32_t group_magic; // ceil(2^32 / group), 0 for group = 1: row / group for row * group < 2^32
};

// 16-bit operand vectors
template <int T>
struct Op16;
template <>
struct Op16<TY_F16> {
  typedef f16x8 v8;
  typedef _Float16 e;
  static __device__ __forceinline__ f32x4 mfma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Op16<TY_BF16> {
  typedef bf16x8 v8;
  typedef __bf16 e;
  static __device__ __forceinline__ f32x4 mfma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

// Maximum / sum over the 4 lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float pa_max4(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  x = fmaxf(u2f(a[0]), u2f(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
  return fmaxf(u2f(b[0]), u2f(b[1]));
}
__device__ __forceinline__ float pa_sum4(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  x = u2f(a[0]) + u2f(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
  return u2f(b[0]) + u2f(b[1]);
}

// Lanes' values by data-parallel moves (a few clocks each; a shuffle goes through LDS).
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t pa_dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
// Inclusive prefix sum over the wave.
__device__ __forceinline__ uint32_t pa_scan(uint32_t x) {
  x += pa_dpp<0x111>(x);  // from 1, 2, 4, 8 lanes below in the row of 16
  x += pa_dpp<0x112>(x);
  x += pa_dpp<0x114>(x);
  x += pa_dpp<0x118>(x);
  x += pa_dpp<0x142, 0xa>(x);  // rows 1 and 3: the end of the row below
  x += pa_dpp<0x143, 0xc>(x);  // rows 2 and 3: the end of row 1
  return x;
}
// Maximum of |.| (bits of a nonnegative float) over aligned groups of N = 8, 16 or 32 lanes.
template <int N>
__device__ __forceinline__ uint32_t pa_group_max(uint32_t x) {
  x = max(x, pa_dpp<0xb1>(x));   // lane ^ 1
  x = max(x, pa_dpp<0x4e>(x));   // lane ^ 2
  x = max(x, pa_dpp<0x141>(x));  // mirrored in 8
  if (N > 8) x = max(x, pa_dpp<0x140>(x));  // mirrored in 16
  if (N > 16) {
    auto b = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max((uint32_t)b[0], (uint32_t)b[1]);
  }
  return x;
}

__device__ __forceinline__ uint32_t pa_token(const PaArgs& a, uint32_t row) {
  return a.group_magic ? __umulhi(row, a.group_magic) : row;
}

// ---- the plan
struct PaSeq {
  uint32_t len, first, rows, tiles, blocks;  // blocks: row blocks of the sequence
};
template <int NR, uint32_t TILE = PA_TILE>
__device__ __forceinline__ PaSeq pa_seq(const PaArgs& a, uint32_t s, bool flag) {
  PaSeq q;
  const uint32_t L = a.g.lens[s], m = a.new_lens ? a.new_lens[s] : a.n_new;
  const bool ok = (uint64_t)L <= ((uint64_t)a.g.stride << a.g.shift) && m <= a.n_new && m <= L;
  if (!ok && flag) paged_flag(a.g, PG_BAD_LENGTH);
  q.len = L;
  q.first = L - m;
  q.rows = ok ? m * a.group : 0u;
  q.tiles = q.rows ? (L + TILE - 1) / TILE : 0u;
  q.blocks = (q.rows + 16 * NR - 1) / (16 * NR);
  return q;
}

// Tiles of a piece at most, for `total` of the batch.  Small batches: one tile per wave, or as many as
// bring the pieces below what the chip holds at once (a second generation of workgroups costs its
// whole latency again), the same for every wave (16x1100 with 5 drafts: 22.9 us at 8 tiles, 24.0 at 5).
// Large ones: 16, so that workgroups ending early make room for others, and
// more once that makes over 2048 pieces.
struct PaTarget {
  template <typename F>
  __device__ __forceinline__ uint32_t operator()(const PaArgs& a, uint32_t total, F) const {
    const uint32_t one = (total + a.at_once - 1) / a.at_once;
    return one <= 16 ? max(4u, (one + 3) & ~3u) : max(16u, (total + 2047) / 2048);
  }
};

struct PaPiece {
  uint32_t s, h, rb, t0, t1, n, slot;  // n: the segment's pieces; slot: this piece's (n > 1)
  uint32_t at, slots;                  // index among the sequence's pieces, the sequence's first slot
  PaSeq q;
  bool any;
  // Piece `piece` of segment (h, rb).
  __device__ __forceinline__ void place(uint32_t piece) {
    const uint32_t even = q.tiles / n, more = q.tiles - even * n;  // the first `more` pieces take one tile more
    t0 = piece * even + min(piece, more);
    t1 = t0 + even + (piece < more ? 1u : 0u);
    slot = slots + (h * q.blocks + rb) * n + piece;
  }
};

// Piece `index` of the batch (pieces in the order sequence, KV head, block, tiles).  Each wave works
// it out by itself: a lane for every 64th part of the sequences.
template <int NR, uint32_t TILE = PA_TILE, typename Target = PaTarget>
__device__ __forceinline__ PaPiece pa_piece(const PaArgs& a, uint32_t index, bool flag) {
  const uint32_t lane = threadIdx.x & 63u, n = a.g.n_seqs, per = (n + 63) / 64;
  const uint32_t s0 = min(n, lane * per), s1 = min(n, s0 + per);
  uint32_t total = 0;
  PaSeq q{};
  for (uint32_t s = s0; s < s1; ++s) {
    q = pa_seq<NR, TILE>(a, s, flag);
    total += q.tiles * q.blocks * a.g.n_kv;
  }
  total = __builtin_amdgcn_readlane(pa_scan(total), 63);
  const uint32_t target = Target{}(a, total, [&](auto of) {  // the sum over all segments of what `of` says of theirs
    uint32_t k = 0;
    for (uint32_t s = s0; s < s1; ++s) {
      if (per > 1) q = pa_seq<NR, TILE>(a, s, false);
      k += of(q) * q.blocks * a.g.n_kv;
    }
    return (uint32_t)__builtin_amdgcn_readlane(pa_scan(k), 63);
  });
  const auto count = [&](const PaSeq& z) { return (z.tiles + target - 1) / target; };
  uint32_t mine = 0, cut = 0;
  for (uint32_t s = s0; s < s1; ++s) {
    if (per > 1) q = pa_seq<NR, TILE>(a, s, false);
    const uint32_t c = count(q), k = c * q.blocks * a.g.n_kv;
    mine += k;
    if (c > 1) cut += k;
  }
  const uint32_t x = pa_scan(mine), y = pa_scan(cut);
  PaPiece p;
  const uint64_t here = __ballot(index < x);
  p.any = here != 0;
  if (!p.any) return p;
  const int owner = __builtin_ctzll(here);
  uint32_t before = __builtin_amdgcn_readlane(x - mine, owner), slots = __builtin_amdgcn_readlane(y - cut, owner);
  uint32_t s = owner * per;
  for (;; ++s) {
    q = pa_seq<NR, TILE>(a, s, false);
    const uint32_t c = count(q), k = c * q.blocks * a.g.n_kv;
    if (index - before < k) break;
    before += k;
    if (c > 1) slots += k;
  }
  p.s = s;
  p.q = q;
  p.n = count(q);
  p.slots = slots;
  p.at = index - before;
  const uint32_t seg = p.at / p.n;
  p.h = q.blocks == 1 ? seg : seg / q.blocks;
  p.rb = seg - p.h * q.blocks;
  p.place(p.at - seg * p.n);
  return p;
}

// A granule's page of the tile at pos0: the table entry of position pos0 + 8 gran.
__device__ __forceinline__ uint32_t pa_page(const PaArgs& a, const uint32_t* tab, uint32_t pos, uint32_t len) {
  return pos < len ? tab[pos >> a.g.shift] : 0u;
}

// N granules, `step` apart; STREAM: without keeping them in the caches.
template <bool STREAM, int N, typename V>
__device__ __forceinline__ void pa_load(const V* p, size_t step, V* to) {
#pragma unroll
  for (int i = 0; i < N; ++i) to[i] = STREAM ? __builtin_nontemporal_load(p + i * step) : p[i * step];
}

// Four outputs to elements from dst on.
template <int QT>
__device__ __forceinline__ void pa_store4(void* out, size_t dst, f32x4 z) {
  if constexpr (QT == TY_F32) {
    *reinterpret_cast<f32x4*>(static_cast<float*>(out) + dst) = z;
  } else {
    ushort4 b;
    b.x = to_bits16<QT>(z[0]);
    b.y = to_bits16<QT>(z[1]);
    b.z = to_bits16<QT>(z[2]);
    b.w = to_bits16<QT>(z[3]);
    *reinterpret_cast<ushort4*>(static_cast<uint16_t*>(out) + dst) = b;
  }
}

// Workgroups of a CU, by registers and LDS.
constexpr int pa_per_cu(int hd, int nr) { return hd == 64 ? 5 - nr : hd == 128 ? 4 - nr : 2; }

// One piece per workgroup.  STREAM: the batch's K and V are beyond what the memory-side cache holds and
// pass the caches by.
template <int HD, int KT, int QT, int NR, bool STREAM>
__global__ __launch_bounds__(PA_NT, pa_per_cu(HD, NR)) void k_pa_split(PaArgs a) {
  typedef typename Op16<KT>::v8 v8;
  typedef typename Op16<KT>::e e16;
  constexpr int NQ = QT != TY_F32 ? 1 : KT == TY_F16 ? 2 : 3;  // 16-bit terms of a query
  constexpr int NP = KT == TY_F16 ? 2 : 3;                     // ... of a weight
  constexpr int KS = HD / 32, DS = HD / 16;
  constexpr int ROWS = 16 * NR, PITCH = HD + 4;
  extern __shared__ float smem[];  // [4][ROWS][PITCH] rows, [4][ROWS][2] states, [ROWS]
  float* s_ml = smem + 4 * ROWS * PITCH;
  float* s_c = s_ml + 4 * ROWS * 2;  // [ROWS] scale log2(e) / the row's power of two
  float* s_q = smem;                 // [NR][NQ][KS][64] operands of 16 bytes
  const uint32_t tid = threadIdx.x, lane = tid & 63u, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t col = lane & 15u, grp = lane >> 4;
  const Paged& g = a.g;
  const uint32_t group = a.group, cap = g.stride << g.shift;

  const PaPiece pc = pa_piece<NR>(a, blockIdx.x, blockIdx.x == 0);
  if (!pc.any) return;
  const PaSeq& sq = pc.q;
  const uint32_t s = pc.s, h = pc.h, rb = pc.rb, t0 = pc.t0, t1 = pc.t1;
  {
    const uint32_t* tab = g.table + (size_t)s * g.stride;
    const uint32_t len = sq.len, first = sq.first;

    f32x4 o[NR][DS];
    float m[NR], l[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.0f;
#pragma unroll
      for (int d = 0; d < DS; ++d) o[r][d] = f32x4{0, 0, 0, 0};
    }

    // ---- tiles t0 + w, t0 + w + 4, ...: the first one's pages, then its K and V, are on their way before
    // the query rows are made ready
    const uint32_t ta = t0 + w;
    const uint32_t kpos = 8 * (col >> 2), ko = kpos + (col & 3u);  // this lane's K row in a tile
    const size_t head_elems = (size_t)HD << g.shift;
    const uint32_t pmask = (1u << g.shift) - 1u;
    v8 kf[2][KS], vf[DS];
    uint32_t odd_tile = ~0u;  // the tile whose infinities and NaN were set aside (a wave has one at most)
    const auto load_k = [&](uint32_t pos0, uint32_t page) {
      if (page >= g.n_pages) page = 0;
      const uint16_t* p = a.kc + ((size_t)page * g.n_kv + h) * head_elems +
                          (((size_t)grp << g.shift) + ((pos0 + ko) & pmask)) * 8;
      const size_t step = (size_t)4 << g.shift;  // granules of 32 dims
      pa_load<STREAM, KS>(reinterpret_cast<const v8*>(p), step, kf[0]);
      pa_load<STREAM, KS>(reinterpret_cast<const v8*>(p) + 4, step, kf[1]);
    };
    const auto load_v = [&](uint32_t pos0, uint32_t page) {
      if (page >= g.n_pages) page = 0;
      const uint16_t* p = a.vc + ((size_t)page * g.n_kv + h) * head_elems +
                          ((size_t)(((pos0 + 8 * grp) & pmask) >> 3) * HD + col) * 8;
      pa_load<STREAM, DS>(reinterpret_cast<const v8*>(p), 16, vf);
    };
    uint32_t pk = 0, pv = 0, pkn = 0, pvn = 0;
    if (ta < t1) {
      pk = pa_page(a, tab, ta * PA_TILE + kpos, len);
      pv = pa_page(a, tab, ta * PA_TILE + 8 * grp, len);
      pkn = pa_page(a, tab, (ta + 4) * PA_TILE + kpos, len);
      pvn = pa_page(a, tab, (ta + 4) * PA_TILE + 8 * grp, len);
    }
    // the query rows as operands in LDS: unit (row, 8 dims) of every thread, a row in HD / 8 lanes
    constexpr int LPR = HD / 8, UNITS = ROWS * LPR, PASSES = (UNITS + PA_NT - 1) / PA_NT;
    typedef typename std::conditional<QT == TY_F32, float, e16>::type QE;
    typedef QE q8v __attribute__((ext_vector_type(8)));
    q8v raw[PASSES];
#pragma unroll
    for (int k = 0; k < PASSES; ++k) {
      const uint32_t u = tid + k * PA_NT, row = rb * ROWS + u / LPR;
      const uint32_t t = pa_token(a, row), qh = h * group + (row - t * group);
      raw[k] = q8v{};
      if (u < UNITS && row < sq.rows)
        raw[k] = *reinterpret_cast<const q8v*>(static_cast<const QE*>(a.q) + ((size_t)s * a.n_new + t) * a.q_stride +
                                               (size_t)qh * HD + 8 * (u % LPR));
    }
    if (ta < t1) {
      load_k(ta * PA_TILE, pk);
      load_v(ta * PA_TILE, pv);
    }
#pragma unroll
    for (int k = 0; k < PASSES; ++k) {
      const uint32_t u = tid + k * PA_NT, row = u / LPR, d8 = u % LPR;
      float factor = a.scale * PA_LOG2E;
      int up = 0;
      if constexpr (QT == TY_F32) {
        // f16 terms: the row's largest element to [2^13, 2^14), whatever it is.  bf16 terms have f32's exponents:
        // rows beyond 2^65 or below 2^-64 to there, so that the first term cannot round to infinity nor the last
        // be subnormal
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, f2u(raw[k][i]) & 0x7fffffffu);
        const int ex = (int)(pa_group_max<LPR>(top) >> 23) - 127;
        if (ex < 128) up = KT == TY_F16 ? 13 - ex : max(-64, min(64, ex)) - ex;
        // a scale so large that log2(e) takes it beyond f32: 4 of it go to the row (whose products with keys of
        // bf16 may be as small as they like)
        if (KT == TY_BF16 && ex < 128 && fabsf(a.scale) > 0x1p126f) up += 2;
        // (other factors beyond f32: the scores' differences are past exp's range with the largest one as well)
        factor = fmaxf(PA_LOWEST, fminf(-PA_LOWEST, ldexpf(a.scale, -up) * PA_LOG2E));
      }
      v8 term[NQ];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (QT != TY_F32) {
          term[0][i] = raw[k][i];
        } else {
          float v = ldexpf(raw[k][i], up);
          const bool fin = fabsf(v) < INFINITY;
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            const e16 b = (e16)v;
            term[n][i] = b;
            v = fin ? v - (float)b : 0.0f;
          }
        }
      }
      if (UNITS >= PA_NT || u < UNITS) {
        // lane 16 (d8 % 4) + row % 16 of 32-dim step d8 / 4
#pragma unroll
        for (int n = 0; n < NQ; ++n)
          *reinterpret_cast<v8*>(&s_q[((((row >> 4) * NQ + n) * KS + (d8 >> 2)) * 64 + (d8 & 3u) * 16 + (row & 15u)) * 4]) = term[n];
        if (d8 == 0) s_c[row] = factor;
      }
    }
    __syncthreads();
    float c[NR];
    uint32_t limit[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const uint32_t row = rb * ROWS + r * 16 + col;
      c[r] = s_c[r * 16 + col];
      limit[r] = first + (row < sq.rows ? pa_token(a, row) : 0u);
    }
    if (ta < t1) {
      for (uint32_t t = ta; t < t1; t += 4) {
        const uint32_t pos0 = t * PA_TILE;
        const bool next = t + 4 < t1;
        f32x4 sc[NR][2];
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            sc[r][b] = f32x4{0, 0, 0, 0};
          }
        asm volatile("" ::: "memory");  // (the query operands stay in LDS: registers)
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int n = NQ - 1; n >= 0; --n)  // the small terms first
#pragma unroll
            for (int j = 0; j < KS; ++j) {
              const v8 qf = *reinterpret_cast<const v8*>(&s_q[(((r * NQ + n) * KS + j) * 64 + lane) * 4]);
              sc[r][0] = Op16<KT>::mfma(kf[0][j], qf, sc[r][0]);
              sc[r][1] = Op16<KT>::mfma(kf[1][j], qf, sc[r][1]);
            }
        uint32_t pv2 = 0;
        const bool page_ok = pv < g.n_pages;
        if (next) {
          const uint32_t pk2 = pa_page(a, tab, (t + 8) * PA_TILE + kpos, len);
          pv2 = pa_page(a, tab, (t + 8) * PA_TILE + 8 * grp, len);
          load_k(pos0 + 4 * PA_TILE, pkn);
          pkn = pk2;
        }
        const uint32_t gpos = pos0 + 8 * grp;  // this lane's 8 positions
        const bool bad = !page_ok;
        if (bad) paged_flag(g, PG_BAD_PAGE);
        const bool edge = pos0 + PA_TILE - 1 > first || __ballot(bad) != 0;
        float top[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          if (edge) {
            top[r] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const bool seen = gpos + i <= limit[r] && page_ok;
              const float v = sc[r][i >> 2][i & 3] * c[r];
              if (seen) top[r] = fmaxf(top[r], fmaxf(v, PA_LOWEST));
            }
          } else {
            top[r] = PA_LOWEST;
#pragma unroll
            for (int i = 0; i < 8; ++i) top[r] = fmaxf(top[r], sc[r][i >> 2][i & 3] * c[r]);
          }
        }
        if (a.scores) {
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            const uint32_t row = rb * ROWS + r * 16 + col;
            if (row < sq.rows && gpos < len) {
              f32x4 u[2];
#pragma unroll
              for (int i = 0; i < 8; ++i)
                u[i >> 2][i & 3] = gpos + i <= limit[r] && page_ok ? sc[r][i >> 2][i & 3] * c[r] : -INFINITY;
              float* p = a.scores + (((size_t)s * g.n_kv + h) * ((size_t)a.n_new * group) + row) * cap + gpos;
              *reinterpret_cast<f32x4*>(p) = u[0];
              *reinterpret_cast<f32x4*>(p + 4) = u[1];
            }
          }
        }
        v8 pf[NR][NP];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          // the reference of the exponents is a whole number: rescaling by powers of two is exact
          const float m_new = fmaxf(m[r], ceilf(pa_max4(top[r])));
          const float ref = m_new == -INFINITY ? 0.0f : m_new;
          if (__ballot(m_new > m[r])) {
            const float alpha = __builtin_amdgcn_exp2f(m[r] - ref);
            l[r] *= alpha;
#pragma unroll
            for (int d = 0; d < DS; ++d) o[r][d] *= alpha;
            m[r] = m_new;
          }
          float cr = c[r], base = a.p_bits - ref;
          if (__ballot(fabsf(ref) >= 1024.0f)) {
            // far from zero the product before its rounding may lie well above the reference, which comes from
            // the rounded ones, and the factor may be lost in the reference
#pragma unroll
            for (int i = 0; i < 8; ++i) sc[r][i >> 2][i & 3] = (sc[r][i >> 2][i & 3] * cr - ref) + a.p_bits;
            cr = 1.0f;
            base = 0.0f;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r][i >> 2][i & 3], cr, base));
            if (edge && !(gpos + i <= limit[r] && page_ok)) p = 0.0f;
            l[r] += p;
#pragma unroll
            for (int n = 0; n < NP; ++n) {
              const e16 b = (e16)p;
              pf[r][n][i] = b;
              p -= (float)b;
            }
          }
        }
        if (edge) {
          // V of masked positions to zero: a zero weight times their bits may be NaN.  Where some rows
          // see a position that others do not, infinities and NaN go to zero too and are added to the
          // rows that see them below
          uint32_t keep[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool lo = gpos + 2 * i < len && page_ok, hi = gpos + 2 * i + 1 < len && page_ok;
            keep[i] = (lo ? 0xffffu : 0u) | (hi ? 0xffff0000u : 0u);
          }
          uint32_t odd = 0;
#pragma unroll
          for (int d = 0; d < DS; ++d) {
            uint4 u = __builtin_bit_cast(uint4, vf[d]);
            uint32_t x4[4] = {u.x & keep[0], u.y & keep[1], u.z & keep[2], u.w & keep[3]};
            if (len - first > 1 && pos0 + PA_TILE - 1 > first) {
              constexpr uint32_t E = KT == TY_F16 ? 0x7c00u : 0x7f80u;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t bits = ((x4[i] & E) == E ? 0xffffu : 0u) | (((x4[i] >> 16) & E) == E ? 0xffff0000u : 0u);
                odd |= bits;
                x4[i] &= ~bits;
              }
            }
            vf[d] = __builtin_bit_cast(v8, make_uint4(x4[0], x4[1], x4[2], x4[3]));
          }
          if (__ballot(odd != 0)) odd_tile = t;
        }
#pragma unroll
        for (int n = NP - 1; n >= 0; --n)
#pragma unroll
          for (int d = 0; d < DS; ++d)
#pragma unroll
            for (int r = 0; r < NR; ++r) o[r][d] = Op16<KT>::mfma(vf[d], pf[r][n], o[r][d]);
        if (next) {
          pv = pvn;
          pvn = pv2;
          load_v(pos0 + 4 * PA_TILE, pv);
        }
      }
      if (odd_tile != ~0u) {
        // this lane's outputs: dims 16 d + 4 grp + i of its rows
#pragma unroll 1
        for (uint32_t pos = odd_tile * PA_TILE; pos < min(len, (odd_tile + 1) * PA_TILE); ++pos) {
          const uint32_t page = tab[pos >> g.shift];
          if (page >= g.n_pages) continue;
          const uint16_t* p = a.vc + ((size_t)page * g.n_kv + h) * head_elems +
                              ((size_t)((pos & pmask) >> 3) * HD + 4 * grp) * 8 + (pos & 7u);
#pragma unroll
          for (int d = 0; d < DS; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float v = from_bits16<KT>(p[(16 * d + i) * 8]);
              const float add = fabsf(v) < INFINITY ? 0.0f : v;
#pragma unroll
              for (int r = 0; r < NR; ++r) o[r][d][i] += pos <= limit[r] ? add : 0.0f;
            }
        }
      }
    }

    // ---- the waves' states joined; rows finished, or a part written
    __syncthreads();  // (the query operands lie where the states go)
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const float sum = pa_sum4(l[r]);
      if (grp == 0) {
        s_ml[(w * ROWS + r * 16 + col) * 2] = m[r];
        s_ml[(w * ROWS + r * 16 + col) * 2 + 1] = sum;
      }
#pragma unroll
      for (int d = 0; d < DS; ++d)
        *reinterpret_cast<f32x4*>(&smem[(w * ROWS + r * 16 + col) * PITCH + 16 * d + 4 * grp]) = o[r][d];
    }
    __syncthreads();
    const bool whole = pc.n == 1;
    if (t0 == 0 && tid == 0) a.cuts[((size_t)s * g.n_kv + h) * a.blocks + rb] = make_uint2(pc.slot, pc.n);
    const uint32_t here = min((uint32_t)ROWS, sq.rows - rb * ROWS);
    for (uint32_t i = tid; i < here * (HD / 4); i += PA_NT) {
      const uint32_t row = i / (HD / 4), d = (i % (HD / 4)) * 4;
      float M = -INFINITY, L = 0.0f;
#pragma unroll
      for (int v = 0; v < 4; ++v) M = fmaxf(M, s_ml[(v * ROWS + row) * 2]);
      const float ref = M == -INFINITY ? 0.0f : M;
      f32x4 y = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float f = __builtin_amdgcn_exp2f(s_ml[(v * ROWS + row) * 2] - ref);
        L += f * s_ml[(v * ROWS + row) * 2 + 1];
        y += f * *reinterpret_cast<const f32x4*>(&smem[(v * ROWS + row) * PITCH + d]);
      }
      const uint32_t full = rb * ROWS + row;
      if (whole) {
        // no position left (bad pages): zeros
        const f32x4 z = M == -INFINITY ? f32x4{0, 0, 0, 0} : y / L;
        const uint32_t t = pa_token(a, full);
        const size_t dst = ((size_t)s * a.n_new + t) * a.out_stride + (size_t)(h * group + (full - t * group)) * HD + d;
        pa_store4<QT>(a.out, dst, z);
        if (a.scores && d == 0) {
          float* st = a.stats + (((size_t)s * g.n_kv + h) * ((size_t)a.n_new * group) + full) * 2;
          st[0] = M;
          st[1] = L;
        }
      } else {
        *reinterpret_cast<f32x4*>(&a.part_o[((size_t)pc.slot * a.part_rows + row) * HD + d]) = y;
        if (d == 0) {
          a.part_ml[((size_t)pc.slot * a.part_rows + row) * 2] = M;
          a.part_ml[((size_t)pc.slot * a.part_rows + row) * 2 + 1] = L;
        }
      }
    }
  }
}

// Joins the cut segments: workgroups of PER rows of a (sequence, KV head), a row's parts dealt out to
// PARTS / PER groups of HD / 4 lanes; then, where weights are kept, workgroups of 256 or 64 positions.  Bound:
// latency (4.4 us for 8 segments of 65 pieces), with weights the scores' bytes too.  A launch of its own:
// joins by the last workgroup of a segment would need device-wide fences, which write back the L2.
// static: several objects of the library instantiate it, and with shared names the linker keeps one object's launch
// stub for both, which another object's kernel may not fit.
constexpr uint32_t PJ_ROWS = 64, PJ_AHEAD = 16;
constexpr uint32_t pj_parts(uint32_t hd) { return PA_NT / (hd / 4); }
template <int HD, int QT, int NR, uint32_t PER>
static __global__ __launch_bounds__(PA_NT) void k_pa_join(PaArgs a, uint32_t n_rows, uint32_t row_groups,
                                                          uint32_t spans, uint32_t span_bits) {
  constexpr uint32_t ROWS = 16 * NR, PARTS = pj_parts(HD), STEP = PARTS / PER;
  __shared__ f32x4 s_o[PARTS][HD / 4];
  __shared__ float s_ml[PARTS][2];
  __shared__ float s_stat[PJ_ROWS][2];
  const Paged& g = a.g;
  const uint32_t tid = threadIdx.x, n_out = g.n_seqs * g.n_kv * row_groups;
  const bool is_out = blockIdx.x < n_out;
  const uint32_t sh = is_out ? blockIdx.x / row_groups : (blockIdx.x - n_out) / spans, s = sh / g.n_kv, h = sh - s * g.n_kv;
  const uint2* cuts = a.cuts + (size_t)sh * a.blocks;
  if (is_out) {
    const uint32_t d = tid % (HD / 4), unit = tid / (HD / 4), part = unit / PER;
    const uint32_t row = (blockIdx.x - sh * row_groups) * PER + unit % PER, rb = row / ROWS, r = row % ROWS;
    const uint2 cut = row < n_rows ? cuts[rb] : make_uint2(0, 1);
    const PaSeq sq = pa_seq<NR>(a, s, false);
    const bool live = row < sq.rows && cut.y > 1;  // (else finished by its one piece)
    float M = -INFINITY, L = 0.0f;
    f32x4 y = f32x4{0, 0, 0, 0};
    const auto add = [&](float m2, float l2, f32x4 y2) {
      const float top = fmaxf(M, m2), ref = top == -INFINITY ? 0.0f : top;
      const float f = __builtin_amdgcn_exp2f(M - ref), f2 = __builtin_amdgcn_exp2f(m2 - ref);
      L = L * f + l2 * f2;
      y = y * f + y2 * f2;
      M = top;
    };
    if (live) {
#pragma unroll 4
      for (uint32_t i = part; i < cut.y; i += STEP) {
        const size_t at = (size_t)(cut.x + i) * a.part_rows + r;
        const float2 ml = *reinterpret_cast<const float2*>(&a.part_ml[at * 2]);
        add(ml.x, ml.y, *reinterpret_cast<const f32x4*>(&a.part_o[at * HD + 4 * d]));
      }
    }
    s_o[unit][d] = y;
    if (d == 0) {
      s_ml[unit][0] = M;
      s_ml[unit][1] = L;
    }
    __syncthreads();
    if (part == 0 && live) {
      for (uint32_t i = unit + PER; i < PARTS; i += PER) add(s_ml[i][0], s_ml[i][1], s_o[i][d]);
      const f32x4 z = M == -INFINITY ? f32x4{0, 0, 0, 0} : y / L;
      const uint32_t t = pa_token(a, row);
      const size_t dst = ((size_t)s * a.n_new + t) * a.out_stride + (size_t)(h * a.group + (row - t * a.group)) * HD + 4 * d;
      pa_store4<QT>(a.out, dst, z);
    }
    return;
  }
  // weights of 1 << span_bits positions, the rows dealt out to the 256 >> span_bits groups of threads that are
  // left: the scores, PJ_AHEAD rows' on their way at a time, against each row's maximum and sum
  const uint32_t span = 1u << span_bits, teams = PA_NT >> span_bits, team = __builtin_amdgcn_readfirstlane(tid >> span_bits);
  const uint32_t pos0 = (blockIdx.x - n_out - sh * spans) << span_bits, pos = pos0 + (tid & (span - 1));
  const PaSeq sq = pa_seq<NR>(a, s, false);
  if (!sq.rows || pos0 >= sq.len) return;
  const uint32_t cap = g.stride << g.shift;
  const size_t all = (size_t)a.n_new * a.group, base = (size_t)sh * all;
  const uint32_t at_pos = min(pos, sq.len - 1);
  float* wp = a.weights + (size_t)sh * cap;
  float acc = team == 0 && at_pos < sq.first ? wp[at_pos] : 0.0f;
  for (uint32_t r0 = 0; r0 < sq.rows; r0 += PJ_ROWS) {
    const uint32_t n = min(PJ_ROWS, sq.rows - r0);
    float sc[PJ_AHEAD];
    const auto fetch = [&](uint32_t k) {
#pragma unroll
      for (uint32_t i = 0; i < PJ_AHEAD; ++i)
        if (k + i * teams < n) sc[i] = a.scores[(base + r0 + k + i * teams) * cap + at_pos];
    };
    fetch(team);
    __syncthreads();
    // a quarter wave per row: 16 lanes over its parts
    for (uint32_t k = tid >> 4; k < n; k += PA_NT / 16) {
      const uint32_t full = r0 + k, rb = full / ROWS, r = full % ROWS, lane = tid & 15u;
      const uint2 cut = cuts[rb];
      float M = -INFINITY, L = 0.0f;
      if (cut.y == 1) {
        M = a.stats[(base + full) * 2];
        L = a.stats[(base + full) * 2 + 1];
      } else {
        for (uint32_t i = lane; i < cut.y; i += 16) {
          const float2 ml = *reinterpret_cast<const float2*>(&a.part_ml[((size_t)(cut.x + i) * a.part_rows + r) * 2]);
          const float top = fmaxf(M, ml.x), ref = top == -INFINITY ? 0.0f : top;
          L = L * __builtin_amdgcn_exp2f(M - ref) + ml.y * __builtin_amdgcn_exp2f(ml.x - ref);
          M = top;
        }
        for (int o = 8; o; o >>= 1) {
          const float m2 = __shfl_xor(M, o), l2 = __shfl_xor(L, o);
          const float top = fmaxf(M, m2), ref = top == -INFINITY ? 0.0f : top;
          // (both orders give the same bits: the two lanes agree)
          const float p = L * __builtin_amdgcn_exp2f(M - ref), q = l2 * __builtin_amdgcn_exp2f(m2 - ref);
          L = p + q;
          M = top;
        }
      }
      if (lane == 0) {
        s_stat[k][0] = M == -INFINITY ? 0.0f : M;
        s_stat[k][1] = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(a.p_bits) / L;
      }
    }
    __syncthreads();
    for (uint32_t k = team; k < n; k += PJ_AHEAD * teams) {
      if (k != team) fetch(k);
#pragma unroll
      for (uint32_t i = 0; i < PJ_AHEAD; ++i) {
        const uint32_t r = k + i * teams;
        if (r < n) acc += __builtin_amdgcn_exp2f(sc[i] - s_stat[r][0]) * s_stat[r][1];
      }
    }
  }
  if (teams > 1) {
    float* s_acc = reinterpret_cast<float*>(s_o);
    s_acc[tid] = acc;
    __syncthreads();
    for (uint32_t t = 1; t < teams; ++t) acc += s_acc[t * span + (tid & (span - 1))];
  }
  if (team == 0 && pos < sq.len) wp[pos] = acc;
}

}  // namespace cm
