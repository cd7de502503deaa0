// kernels_paged_attn.h -- attention of a sequence's newest tokens over a cache in pages.
//
//   s_p = scale (q . k_p) for p <= the row's position;  w = softmax(s);  o = sum_p w_p v_p
//
// Bound: the cache's bytes (4 hd per position and KV head, against 4 hd flop per position and row),
// so the kernel's work is to keep HBM busy whatever the batch looks like.
//
// Split.  A segment is (sequence, KV head, block of 16 NR query rows); its tiles are 32 positions.
// All segments' tiles form one list, dealt out in equal runs to the workgroups (planned on the
// device from lens, so a captured graph follows growing caches): a workgroup's run may cover part of
// a long segment or several short ones.  The query rows of a segment are the new tokens times the KV
// head's query heads, so K and V are read once for all of them.  A segment that lies inside one run is
// finished there; of the others each run writes its part (running maximum, sum, unnormalised rows)
// to one of its two slots, since only its first and its last segment can be cut, and k_pa_join joins
// them.
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
// Numbers.  f32 queries are the sum of two f16 (scaled by a power of two into f16's range; 22 bits) or
// of three bf16, 16-bit queries are used as they are; the weights exp2(s - max) are the sum of
// two 16-bit numbers (three bf16 for f32 outputs), so they keep 16 bits at least where the output
// has 8 or 11.  f16 weights carry a factor 2^14: small ones next to the row's maximum stay normal.
#pragma once
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
  float* stats;    // [seq][kv head][row][2]: maximum and sum of segments finished in one run
  float* part_ml;  // [slot][16 NR][2]
  float* part_o;   // [slot][16 NR][hd]
  float* weights;
  float scale;
  float p_bits;    // weights are held times 2^p_bits
  uint32_t q_stride, out_stride, n_new, n_heads, n_wg;
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

// ---- the plan: tiles of all segments as one list
struct PaSeq {
  uint32_t len, first, rows, tiles, blocks;  // blocks: row blocks of the sequence
};
template <int NR>
__device__ __forceinline__ PaSeq pa_seq(const PaArgs& a, uint32_t s, bool flag) {
  PaSeq q;
  const uint32_t L = a.g.lens[s], m = a.new_lens ? a.new_lens[s] : a.n_new;
  const bool ok = (uint64_t)L <= ((uint64_t)a.g.stride << a.g.shift) && m <= a.n_new && m <= L;
  if (!ok && flag) paged_flag(a.g, PG_BAD_LENGTH);
  q.len = L;
  q.first = L - m;
  q.rows = ok ? m * (a.n_heads / a.g.n_kv) : 0u;
  q.tiles = q.rows ? (L + PA_TILE - 1) / PA_TILE : 0u;
  q.blocks = (q.rows + 16 * NR - 1) / (16 * NR);
  return q;
}
__device__ __forceinline__ uint64_t pa_count(const PaArgs& a, const PaSeq& q) {
  return (uint64_t)q.tiles * q.blocks * a.g.n_kv;
}

struct PaPlan {
  uint64_t total;     // tiles
  uint64_t segments;
  uint64_t before;    // tiles before sequence `at`
  uint32_t at;
};

// Workgroups that get a run: one tile for each wave at least, or one segment.
__device__ __forceinline__ uint32_t pa_runs(const PaArgs& a, uint64_t total, uint64_t segments) {
  uint64_t n = (total + 3) / 4;
  if (segments > n) n = segments;
  return (uint32_t)(n < a.n_wg ? n : a.n_wg);
}
__device__ __forceinline__ uint64_t pa_begin(uint64_t total, uint32_t runs, uint32_t i) {
  return total * i / runs;  // (below 2^40 tiles and 2^12 runs)
}
// The run that holds tile x.
__device__ __forceinline__ uint32_t pa_run_of(uint64_t total, uint32_t runs, uint64_t x) {
  return (uint32_t)(((x + 1) * runs - 1) / total);
}

// Totals, and for want < total the sequence that holds tile `want` (i < n_seqs: tiles before
// sequence i as `want`).  Every thread of the workgroup calls it; sh: 3 x 4 + 3 words.
template <int NR, typename F>
__device__ __forceinline__ PaPlan pa_plan(const PaArgs& a, uint64_t* sh, bool flag, F want_of) {
  const uint32_t tid = threadIdx.x, n = a.g.n_seqs, per = (n + PA_NT - 1) / PA_NT;
  const uint32_t s0 = min(n, tid * per), s1 = min(n, s0 + per);
  uint64_t tiles = 0, segs = 0;
  for (uint32_t s = s0; s < s1; ++s) {
    const PaSeq q = pa_seq<NR>(a, s, flag);
    tiles += pa_count(a, q);
    segs += (uint64_t)q.blocks * a.g.n_kv;
  }
  uint64_t x = tiles, y = segs;
  const uint32_t lane = tid & 63u, w = tid >> 6;
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t u = __shfl_up(x, o), v = __shfl_up(y, o);
    if (lane >= (uint32_t)o) {
      x += u;
      y += v;
    }
  }
  if (lane == 63) {
    sh[w] = x;
    sh[4 + w] = y;
  }
  __syncthreads();
  PaPlan p;
  p.total = sh[0] + sh[1] + sh[2] + sh[3];
  p.segments = sh[4] + sh[5] + sh[6] + sh[7];
  for (uint32_t i = 0; i < w; ++i) x += sh[i];
  const uint64_t want = want_of(p.total, p.segments);
  uint64_t c = x - tiles;
  if (want >= c && want < x) {
    for (uint32_t s = s0; s < s1; ++s) {
      const uint64_t k = pa_count(a, pa_seq<NR>(a, s, false));
      if (want < c + k) {
        sh[8] = c;
        sh[9] = s;
        break;
      }
      c += k;
    }
  }
  __syncthreads();
  p.before = sh[8];
  p.at = (uint32_t)sh[9];
  __syncthreads();
  return p;
}

// A granule's page of the tile at pos0: the table entry of position pos0 + 8 gran.
__device__ __forceinline__ uint32_t pa_page(const PaArgs& a, const uint32_t* tab, uint32_t pos, uint32_t len) {
  return pos < len ? tab[pos >> a.g.shift] : 0u;
}

// One run of tiles per workgroup.
template <int HD, int KT, int QT, int NR>
__global__ __launch_bounds__(PA_NT, HD == 64 ? 3 : (HD == 128 && !(NR == 2 && KT == TY_BF16 && QT == TY_F32)) ? 2 : 1)
void k_pa_split(PaArgs a) {
  typedef typename Op16<KT>::v8 v8;
  typedef typename Op16<KT>::e e16;
  constexpr int NQ = QT != TY_F32 ? 1 : KT == TY_F16 ? 2 : 3;  // 16-bit terms of a query
  constexpr int NP = QT == TY_F32 && KT == TY_BF16 ? 3 : 2;    // ... of a weight
  constexpr int KS = HD / 32, DS = HD / 16;
  constexpr int ROWS = 16 * NR, PITCH = HD + 4;
  extern __shared__ float smem[];  // [4][ROWS][PITCH] rows, [4][ROWS][2] states
  float* s_ml = smem + 4 * ROWS * PITCH;
  uint64_t* s_plan = reinterpret_cast<uint64_t*>(smem);
  const uint32_t tid = threadIdx.x, lane = tid & 63u, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t col = lane & 15u, grp = lane >> 4;
  const Paged& g = a.g;
  const uint32_t group = a.n_heads / g.n_kv, cap = g.stride << g.shift;

  const PaPlan plan = pa_plan<NR>(a, s_plan, blockIdx.x == 0, [&](uint64_t total, uint64_t segs) {
    const uint32_t runs = pa_runs(a, total, segs);
    return blockIdx.x < runs ? pa_begin(total, runs, blockIdx.x) : total;
  });
  if (!plan.total) return;
  const uint32_t runs = pa_runs(a, plan.total, plan.segments);
  if (blockIdx.x >= runs) return;
  const uint64_t x0 = pa_begin(plan.total, runs, blockIdx.x), x1 = pa_begin(plan.total, runs, blockIdx.x + 1);
  uint64_t x = x0, rem = x0 - plan.before;
  uint32_t s = plan.at;
  PaSeq sq = pa_seq<NR>(a, s, false);
  uint64_t in_seq = pa_count(a, sq);

  while (x < x1) {
    while (rem >= in_seq) {  // (sequences without tiles are passed over)
      rem -= in_seq;
      sq = pa_seq<NR>(a, ++s, false);
      in_seq = pa_count(a, sq);
    }
    const uint32_t seg = (uint32_t)(rem / sq.tiles), t0 = (uint32_t)(rem - (uint64_t)seg * sq.tiles);
    const uint32_t t1 = (uint32_t)min((uint64_t)sq.tiles, t0 + (x1 - x));
    const uint32_t h = seg / sq.blocks, rb = seg - h * sq.blocks;
    const uint32_t* tab = g.table + (size_t)s * g.stride;
    const uint32_t len = sq.len, first = sq.first;

    // ---- this lane's query rows (one per 16-row block) as operands
    v8 qf[NR][NQ][KS];
    float c[NR];
    uint32_t limit[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const uint32_t row = rb * ROWS + r * 16 + col;
      const bool real = row < sq.rows;
      const uint32_t t = real ? row / group : 0u, qh = h * group + (real ? row - t * group : 0u);
      limit[r] = first + t;
      const size_t src = ((size_t)s * a.n_new + t) * a.q_stride + (size_t)qh * HD + 8 * grp;
      c[r] = a.scale * PA_LOG2E;
      if constexpr (QT != TY_F32) {
        const e16* p = static_cast<const e16*>(a.q) + src;
#pragma unroll
        for (int j = 0; j < KS; ++j) qf[r][0][j] = *reinterpret_cast<const v8*>(p + 32 * j);
      } else {
        const float* p = static_cast<const float*>(a.q) + src;
        float f[KS][8], top = 0.0f;
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          const f32x4 u = *reinterpret_cast<const f32x4*>(p + 32 * j), v = *reinterpret_cast<const f32x4*>(p + 32 * j + 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f[j][i] = u[i];
            f[j][4 + i] = v[i];
            top = fmaxf(top, fmaxf(fabsf(u[i]), fabsf(v[i])));
          }
        }
        int up = 0;
        if (KT == TY_F16) {  // the row's largest element to [2^13, 2^14)
          top = pa_max4(top);
          const int ex = (int)((f2u(top) >> 23) & 255u) - 127;
          up = ex == 128 ? 0 : max(-100, min(100, 13 - ex));
          c[r] = ldexpf(c[r], -up);
        }
#pragma unroll
        for (int j = 0; j < KS; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float v = KT == TY_F16 ? ldexpf(f[j][i], up) : f[j][i];
            const bool fin = fabsf(v) < INFINITY;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
              const e16 b = (e16)v;
              qf[r][n][j][i] = b;
              v = fin ? v - (float)b : 0.0f;
            }
          }
      }
    }

    f32x4 o[NR][DS];
    float m[NR], l[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.0f;
#pragma unroll
      for (int d = 0; d < DS; ++d) o[r][d] = f32x4{0, 0, 0, 0};
    }

    // ---- tiles t0 + w', t0 + w' + 4, ...: consecutive tiles of the run go to consecutive waves
    const uint32_t ta = t0 + ((w - (uint32_t)(x - x0)) & 3u);
    const uint32_t kpos = 8 * (col >> 2), ko = kpos + (col & 3u);  // this lane's K row in a tile
    const size_t head_elems = (size_t)HD << g.shift;
    const uint32_t pmask = (1u << g.shift) - 1u;
    v8 kf[2][KS], vf[DS];
    uint32_t odd_tile = ~0u;  // the tile whose infinities and NaN were set aside (a wave has one at most)
    const auto load_k = [&](uint32_t pos0, uint32_t page) {
      if (page >= g.n_pages) page = 0;
      const uint16_t* p = a.kc + ((size_t)page * g.n_kv + h) * head_elems +
                          (((size_t)grp << g.shift) + ((pos0 + ko) & pmask)) * 8;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const uint16_t* pj = p + ((size_t)(4 * j) << (g.shift + 3));
        kf[0][j] = *reinterpret_cast<const v8*>(pj);
        kf[1][j] = *reinterpret_cast<const v8*>(pj + 32);
      }
    };
    const auto load_v = [&](uint32_t pos0, uint32_t page) {
      if (page >= g.n_pages) page = 0;
      const uint16_t* p = a.vc + ((size_t)page * g.n_kv + h) * head_elems +
                          ((size_t)(((pos0 + 8 * grp) & pmask) >> 3) * HD + col) * 8;
#pragma unroll
      for (int d = 0; d < DS; ++d) vf[d] = *reinterpret_cast<const v8*>(p + d * 128);
    };
    if (ta < t1) {
      uint32_t pk = pa_page(a, tab, ta * PA_TILE + kpos, len), pv = pa_page(a, tab, ta * PA_TILE + 8 * grp, len);
      uint32_t pkn = pa_page(a, tab, (ta + 4) * PA_TILE + kpos, len),
               pvn = pa_page(a, tab, (ta + 4) * PA_TILE + 8 * grp, len);
      load_k(ta * PA_TILE, pk);
      load_v(ta * PA_TILE, pv);
      for (uint32_t t = ta; t < t1; t += 4) {
        const uint32_t pos0 = t * PA_TILE;
        const bool next = t + 4 < t1;
        f32x4 sc[NR][2];
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            sc[r][b] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int n = NQ - 1; n >= 0; --n)  // the small terms first
#pragma unroll
              for (int j = 0; j < KS; ++j) sc[r][b] = Op16<KT>::mfma(kf[b][j], qf[r][n][j], sc[r][b]);
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
          const float base = a.p_bits - ref;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r][i >> 2][i & 3], c[r], base));
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
    __syncthreads();
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
    const bool whole = t0 == 0 && t1 == sq.tiles;
    const uint32_t slot = 2 * blockIdx.x + (x == x0 ? 0u : 1u);
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
        const size_t dst = ((size_t)s * a.n_new + full / group) * a.out_stride + (size_t)(h * group + full % group) * HD + d;
        if constexpr (QT == TY_F32) {
          *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + dst) = z;
        } else {
          ushort4 b;
          b.x = to_bits16<QT>(z[0]);
          b.y = to_bits16<QT>(z[1]);
          b.z = to_bits16<QT>(z[2]);
          b.w = to_bits16<QT>(z[3]);
          *reinterpret_cast<ushort4*>(static_cast<uint16_t*>(a.out) + dst) = b;
        }
        if (a.scores && d == 0) {
          float* st = a.stats + (((size_t)s * g.n_kv + h) * ((size_t)a.n_new * group) + full) * 2;
          st[0] = M;
          st[1] = L;
        }
      } else {
        *reinterpret_cast<f32x4*>(&a.part_o[((size_t)slot * ROWS + row) * HD + d]) = y;
        if (d == 0) {
          a.part_ml[((size_t)slot * ROWS + row) * 2] = M;
          a.part_ml[((size_t)slot * ROWS + row) * 2 + 1] = L;
        }
      }
    }
    __syncthreads();
    x += t1 - t0;
    rem += t1 - t0;
  }
}

// The slots of a segment that starts at tile x (of `tiles`): runs i0 .. i1, run i0's first or second
// slot, the later runs' first.
struct PaCut {
  uint32_t i0, i1, slot0;
};
__device__ __forceinline__ PaCut pa_cut(const PaPlan& p, uint32_t runs, uint64_t x, uint32_t tiles) {
  PaCut c;
  c.i0 = pa_run_of(p.total, runs, x);
  c.i1 = pa_run_of(p.total, runs, x + tiles - 1);
  c.slot0 = 2 * c.i0 + (pa_begin(p.total, runs, c.i0) == x ? 0u : 1u);
  return c;
}
__device__ __forceinline__ uint32_t pa_slot(const PaCut& c, uint32_t i) { return i == c.i0 ? c.slot0 : 2 * i; }

// Joins the cut segments: workgroup (sequence, KV head, row) for rows below `n_rows`; then, where
// weights are kept, workgroup (sequence, KV head, 1024 positions).
constexpr uint32_t PJ_SPAN = 1024, PJ_ROWS = 64;
template <int HD, int QT, int NR>
__global__ __launch_bounds__(PA_NT) void k_pa_join(PaArgs a, uint32_t n_rows, uint32_t spans) {
  constexpr int ROWS = 16 * NR, PARTS = PA_NT / (HD / 4);
  __shared__ uint64_t s_plan[16];
  __shared__ f32x4 s_o[PARTS][HD / 4];
  __shared__ float s_l[PARTS];
  __shared__ float s_stat[PJ_ROWS][2];
  const Paged& g = a.g;
  const uint32_t tid = threadIdx.x, group = a.n_heads / g.n_kv, n_out = g.n_seqs * g.n_kv * n_rows;
  const bool is_out = blockIdx.x < n_out;
  const uint32_t sh = is_out ? blockIdx.x / n_rows : (blockIdx.x - n_out) / spans, s = sh / g.n_kv, h = sh % g.n_kv;
  const uint32_t row = blockIdx.x % n_rows, span = (blockIdx.x - n_out) % spans;  // (one of the two has a meaning)
  const PaSeq sq = pa_seq<NR>(a, s, false);
  if (is_out ? row >= sq.rows : !sq.rows || span * PJ_SPAN >= sq.len) return;
  // tiles before this sequence: every sequence's own count, as the runs were dealt out
  uint64_t before = 0;
  const PaPlan p = [&] {
    const uint32_t n = g.n_seqs;
    uint64_t tiles = 0, segs = 0, pre = 0;
    for (uint32_t i = tid; i < n; i += PA_NT) {
      const PaSeq q = pa_seq<NR>(a, i, false);
      const uint64_t k = pa_count(a, q);
      tiles += k;
      segs += (uint64_t)q.blocks * g.n_kv;
      if (i < s) pre += k;
    }
    for (int o = 32; o; o >>= 1) {
      tiles += __shfl_xor(tiles, o);
      segs += __shfl_xor(segs, o);
      pre += __shfl_xor(pre, o);
    }
    if ((tid & 63u) == 0) {
      s_plan[tid >> 6] = tiles;
      s_plan[4 + (tid >> 6)] = segs;
      s_plan[8 + (tid >> 6)] = pre;
    }
    __syncthreads();
    PaPlan q;
    q.total = s_plan[0] + s_plan[1] + s_plan[2] + s_plan[3];
    q.segments = s_plan[4] + s_plan[5] + s_plan[6] + s_plan[7];
    before = s_plan[8] + s_plan[9] + s_plan[10] + s_plan[11];
    q.before = before;
    q.at = s;
    return q;
  }();
  const uint32_t runs = pa_runs(a, p.total, p.segments);
  if (is_out) {
    const uint32_t rb = row / ROWS, r = row % ROWS;
    const PaCut c = pa_cut(p, runs, before + ((uint64_t)h * sq.blocks + rb) * sq.tiles, sq.tiles);
    if (c.i0 == c.i1) return;  // finished in its run
    const uint32_t d = tid % (HD / 4), part = tid / (HD / 4);
    float M = -INFINITY;
    for (uint32_t i = c.i0 + (tid & 63u); i <= c.i1; i += 64)
      M = fmaxf(M, a.part_ml[((size_t)pa_slot(c, i) * ROWS + r) * 2]);
    for (int o = 32; o; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
    const float ref = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    f32x4 y = f32x4{0, 0, 0, 0};
    for (uint32_t i = c.i0 + part; i <= c.i1; i += PARTS) {
      const size_t at = (size_t)pa_slot(c, i) * ROWS + r;
      const float f = __builtin_amdgcn_exp2f(a.part_ml[at * 2] - ref);
      L += f * a.part_ml[at * 2 + 1];
      y += f * *reinterpret_cast<const f32x4*>(&a.part_o[at * HD + 4 * d]);
    }
    s_o[part][d] = y;
    if (d == 0) s_l[part] = L;
    __syncthreads();
    if (part == 0) {
      for (int i = 1; i < PARTS; ++i) {
        L += s_l[i];
        y += s_o[i][d];
      }
      const f32x4 z = M == -INFINITY ? f32x4{0, 0, 0, 0} : y / L;
      const size_t dst = ((size_t)s * a.n_new + row / group) * a.out_stride + (size_t)(h * group + row % group) * HD + 4 * d;
      if constexpr (QT == TY_F32) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + dst) = z;
      } else {
        ushort4 b;
        b.x = to_bits16<QT>(z[0]);
        b.y = to_bits16<QT>(z[1]);
        b.z = to_bits16<QT>(z[2]);
        b.w = to_bits16<QT>(z[3]);
        *reinterpret_cast<ushort4*>(static_cast<uint16_t*>(a.out) + dst) = b;
      }
    }
    return;
  }
  // weights of positions [span * 1024, ...): the scores against each row's maximum and sum
  const uint32_t cap = g.stride << g.shift;
  const size_t all = (size_t)a.n_new * group, base = (size_t)sh * all;
  float* wp = a.weights + (size_t)sh * cap;
  float acc[PJ_SPAN / PA_NT];
#pragma unroll
  for (uint32_t k = 0; k < PJ_SPAN / PA_NT; ++k) {
    const uint32_t pos = span * PJ_SPAN + k * PA_NT + tid;
    acc[k] = pos < sq.first ? wp[pos] : 0.0f;
  }
  for (uint32_t r0 = 0; r0 < sq.rows; r0 += PJ_ROWS) {
    __syncthreads();
    if (tid < PJ_ROWS && r0 + tid < sq.rows) {
      const uint32_t full = r0 + tid, rb = full / ROWS, r = full % ROWS;
      const PaCut c = pa_cut(p, runs, before + ((uint64_t)h * sq.blocks + rb) * sq.tiles, sq.tiles);
      float M = -INFINITY, L = 0.0f;
      if (c.i0 == c.i1) {
        M = a.stats[(base + full) * 2];
        L = a.stats[(base + full) * 2 + 1];
      } else {
        for (uint32_t i = c.i0; i <= c.i1; ++i) M = fmaxf(M, a.part_ml[((size_t)pa_slot(c, i) * ROWS + r) * 2]);
        const float ref = M == -INFINITY ? 0.0f : M;
        for (uint32_t i = c.i0; i <= c.i1; ++i) {
          const size_t at = (size_t)pa_slot(c, i) * ROWS + r;
          L += __builtin_amdgcn_exp2f(a.part_ml[at * 2] - ref) * a.part_ml[at * 2 + 1];
        }
      }
      s_stat[tid][0] = M == -INFINITY ? 0.0f : M - a.p_bits;
      s_stat[tid][1] = M == -INFINITY ? 0.0f : 1.0f / L;
    }
    __syncthreads();
    const uint32_t n = min(PJ_ROWS, sq.rows - r0);
#pragma unroll
    for (uint32_t k = 0; k < PJ_SPAN / PA_NT; ++k) {
      const uint32_t pos = span * PJ_SPAN + k * PA_NT + tid;
      if (pos < sq.len)
        for (uint32_t r = 0; r < n; ++r)
          acc[k] += __builtin_amdgcn_exp2f(a.scores[(base + r0 + r) * cap + pos] - s_stat[r][0]) * s_stat[r][1];
    }
  }
#pragma unroll
  for (uint32_t k = 0; k < PJ_SPAN / PA_NT; ++k) {
    const uint32_t pos = span * PJ_SPAN + k * PA_NT + tid;
    if (pos < sq.len) wp[pos] = acc[k];
  }
}

}  // namespace cm
