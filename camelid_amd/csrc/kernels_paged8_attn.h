// kernels_paged8_attn.h -- attention of a sequence's newest tokens over an 8-bit cache in pages.
//
//   s_p = scale 2^ke(p) (q . k_p) for p <= the row's position;  w = softmax(s);  o = sum_p w_p 2^ve(p) v_p
//
// The plan (segments of a sequence, KV head and block of query rows, cut into pieces of tiles), the parts and
// their join are those of kernels_paged_attn.h; tiles are 64 positions here.  k_p8_split: a few rows a sequence,
// k_p8_prompt: many.
//
// Bound, split: the cache's bytes (2 hd per position and KV head, 4 hd flop per position and row).  Heads of 128:
//   64 sequences of up to 4001, 24 + 8 heads: 57 + 4.7 us (split + join) for 270 MB, 4.7 TB/s in the split; calls: all
//     of them 4001 long 96 us for 525 MB, 5.5 TB/s; 4 of 65536 94 us, 5.7 TB/s
//   1 of 32775, 32 + 8 heads: 17 + 4.0 us for 67 MB, 16 of up to 1100 with up to 5 new tokens: 13.4 + 4.0 us for
//     20 MB: chains of latencies (launch, plan, pages, K and V, products, states joined)
// The conversion costs about 320 vector instructions a wave and tile of 16 KB, under the time that its bytes take.
// Bound, prompts: vector instructions, then matrix ones.  A wave's 16 rows of a tile take about 240 (operands 40,
// addresses 40, softmax 140 of which 16 exponentials at a quarter of the rate) and 48 matrix instructions (64 for
// f32 rows).  4096 tokens at 12288, 32 + 8 heads of 128, calls among others: bf16 rows 1.36 to 1.40 ms, 690 to 705
// TFLOP/s, vector units busy 74 % of the cycles with the exponentials' extra, matrix units 49 %; f32 rows 1.58 to 1.63 ms.
//   3 prompts of up to 1023, f32: 44 us: a workgroup's tiles follow each other, 2 us each.
//
// Operands.  Granules of 16 bytes become two operands of v_mfma_f32_16x16x32_f16 each: int8 as the low byte of the
// f16 1024 + u, minus 1152, e4m3 by the conversion instruction, both exact.
//   S^T = K Q^T: the dims of a step are 8 of a K granule for each lane group, the same ones of q.  The rows r of
//   the four products of a tile are the positions 16 (r / 4) + 4 b + r % 4, so that lane group l / 16
//   ends up with the 16 consecutive positions of one block: one exponent of K and V a lane.
//   O^T = V^T P^T: those 16 positions are one V granule, two operands; P never leaves the lane.
//
// Numbers.  q: f32 and bf16 rows are scaled by a power of two into f16's range, f32 as the sum of two f16 (22
// bits), bf16 and f16 as they are.  K's exponent goes to the scores in f32.  V's goes to the weights before
// they become f16: the matrix cores see w 2^ve / 2^D, D the running maximum of (exponent of the block's largest
// weight + ve) over the row, so that what is lost is measured against the largest contribution and not against the
// largest weight.  D is kept relative to the softmax's reference; both are whole numbers and rescaling is exact.  A weight
// is the sum of two f16: 22 bits.
#pragma once
#include <type_traits>
#include "kernels_paged8.h"
#include "kernels_paged_attn.h"
#include "paged8_plan.h"

namespace cm {

constexpr int P8_TERMS = 2;  // f16 that a softmax weight is the sum of

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct P8Args {
  PaArgs a;  // kc and vc: bytes
  const uint8_t* ke;
  const uint8_t* ve;
};

// 16 bytes of a granule -> 16 f16, in order: two operands.
template <int KT>
__device__ __forceinline__ void p8_operands(u32x4 u, f16x8 (&to)[2]) {
  union {
    f16x2 h[8];
    f16x8 v[2];
  } r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (KT == TY_I8) {
      const uint32_t b = u[i] ^ 0x80808080u;
      r.h[2 * i] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) - (_Float16)1152.0f;
      r.h[2 * i + 1] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) - (_Float16)1152.0f;
    } else {
      r.h[2 * i] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)u[i], 1.0f, false));
      r.h[2 * i + 1] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)u[i], 1.0f, true));
    }
  }
  to[0] = r.v[0];
  to[1] = r.v[1];
}

// Terms of 8 elements of a query row.  top: bits of the largest |element| of the row.  Returns the power of two
// that the row was scaled by.
template <int QT, int NQ, typename R>
__device__ __forceinline__ int p8_query(const R& raw, uint32_t top, bool negate, f16x8 (&term)[NQ]) {
  int up = 0;
  if constexpr (QT != TY_F16) {
    const int ex = (int)(top >> 23) - 127;
    if (ex < 128) up = 13 - ex;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float v = (float)raw[i];
    if constexpr (QT != TY_F16) v = ldexpf(v, up);
    if (negate) v = -v;
    const bool fin = fabsf(v) < INFINITY;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const _Float16 b = (_Float16)v;
      term[n][i] = b;
      v = fin ? v - (float)b : 0.0f;
    }
  }
  return up;
}

// |scale| log2(e) 2^-up as a mantissa and an exponent, so that K's exponents can neither overflow nor lose it.
struct P8Factor {
  float m;
  int e;
};
__device__ __forceinline__ P8Factor p8_factor(float scale, int up) {
  int e;
  const float m = frexpf(fabsf(scale), &e);
  return P8Factor{m * PA_LOG2E, e - up};
}
__device__ __forceinline__ float p8_times(const P8Factor& f, uint32_t exp_byte) {
  const float x = fminf(ldexpf(f.m, f.e + (int)exp_byte - 127), -PA_LOWEST);
  return exp_byte == P8_NAN ? u2f(0x7fc00000u) : x;
}

// The page of position min(pos, len - 1).
__device__ __forceinline__ uint32_t p8_page(const PaArgs& a, const uint32_t* tab, uint32_t pos, uint32_t len) {
  return tab[min(pos, len - 1) >> a.g.shift];
}
// page * unit + more, one multiply-add (unit: bytes of a page, at most 2^30).
__device__ __forceinline__ uint64_t p8_at(uint32_t page, uint32_t unit, uint32_t more) { return (uint64_t)page * unit + more; }

constexpr float P8_NONE = -1e30f;  // no reference of o yet

// What a wave keeps of its 16 NR rows (lane: row 16 r + l % 16, outputs of dims 16 d + 4 (l / 16) + i).
template <int HD, int NR>
struct P8Rows {
  f32x4 o[NR][HD / 16];  // in units of 2^(D - 14)
  float m[NR], D[NR];    // softmax reference, and the reference of o relative to it; whole numbers (none: the lowest)
  float l[NR];           // this lane's share of the sum
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      m[r] = PA_LOWEST;
      D[r] = P8_NONE;
      l[r] = 0.0f;
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) o[r][d] = f32x4{0, 0, 0, 0};
    }
  }
};

// One tile's scores sc (positions gpos + 4 b + i of this lane's block) to weights pf (operands of positions gpos
// + 8 half ...), and the rows' states.  edge: some row may not see some position.
template <int HD, int NR>
__device__ __forceinline__ void p8_softmax(P8Rows<HD, NR>& st, f32x4 (&sc)[NR][4], const P8Factor (&factor)[NR], uint32_t ke,
                                           uint32_t ve, uint32_t gpos, const uint32_t (&limit)[NR], bool page_ok, bool edge,
                                           f16x8 (&pf)[NR][P8_TERMS][2]) {
  const float vexp = (float)((int)ve - 127);
  // (each step for all rows: their chains run side by side)
  float fk[NR], m_new[NR], d_tile[NR], base[NR], shift[NR], inside[NR], p[NR][16];
#pragma unroll
  for (int r = 0; r < NR; ++r) fk[r] = p8_times(factor[r], ke);
  if (edge) {  // positions that the row does not see: -infinity (their factor a positive number)
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const uint32_t n = !page_ok || limit[r] < gpos ? 0u : limit[r] - gpos + 1;
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[r][i >> 2][i & 3] = (uint32_t)i < n ? sc[r][i >> 2][i & 3] : -INFINITY;
      fk[r] = n ? fmaxf(fk[r], 0x1p-126f) : 1.0f;
      if (n && ke == P8_NAN) fk[r] = u2f(0x7fc00000u);
    }
  }
  bool rises = false, far = false, fine = false;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    float top = sc[r][0][0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, sc[r][i >> 2][i & 3]);
    const float ctop = ceilf(top * fk[r]);  // (the factor is not negative)
    // the reference of the exponents is a whole number: rescaling by powers of two is exact
    m_new[r] = fmaxf(st.m[r], pa_max4(ctop));
    d_tile[r] = pa_max4(ctop - m_new[r] + vexp);
    rises |= m_new[r] > st.m[r] || d_tile[r] > st.D[r];
    far |= fabsf(m_new[r]) >= 1024.0f;
  }
  if (__ballot(rises)) {
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const float down = st.m[r] - m_new[r], d_old = st.D[r] + down;
      st.l[r] *= __builtin_amdgcn_exp2f(down);
      st.m[r] = m_new[r];
      st.D[r] = fmaxf(fmaxf(d_old, d_tile[r]), P8_NONE);
      const float alpha = __builtin_amdgcn_exp2f(d_old - st.D[r]);
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) st.o[r][d] *= alpha;
    }
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) base[r] = -m_new[r];
  if (__ballot(far)) {
    // far from zero the product before its rounding may lie well above the reference, which comes from the
    // rounded ones, and the shift below may be lost in the reference
#pragma unroll
    for (int r = 0; r < NR; ++r) {
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[r][i >> 2][i & 3] = sc[r][i >> 2][i & 3] * fk[r] - m_new[r];
      fk[r] = 1.0f;
      base[r] = 0.0f;
    }
  }
  // weights times 2^shift are what the matrix cores get: 2^14 at most.  Inside the exponent the shift costs
  // nothing, and up to 16 of it no bits that matter (half a step of an argument of 16 is 2^-21)
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    shift[r] = vexp - st.D[r] + 14.0f;
    inside[r] = fmaxf(shift[r], -16.0f);
    base[r] += inside[r];
    fine |= shift[r] < -16.0f || ve == P8_NAN;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      p[r][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r][i >> 2][i & 3], fk[r], base[r]));
      sum += p[r][i];
    }
    sum = ldexpf(sum, (int)-inside[r]);
    asm volatile("" : "+v"(sum));  // (summed here: later it would keep copies of the weights)
    st.l[r] += sum;
  }
  if (__ballot(fine)) {
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int more = (int)(shift[r] - inside[r]);
      const uint32_t n = !edge ? 16u : !page_ok || limit[r] < gpos ? 0u : limit[r] - gpos + 1;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        p[r][i] = ldexpf(p[r][i], more);
        if (ve == P8_NAN && (uint32_t)i < n) p[r][i] = u2f(0x7fc00000u);
      }
    }
  }
  // two weights' terms in one instruction, what is left of each in one (exact; a known factor would be a conversion and
  // a subtraction)
  float minus = -1.0f;
  asm("" : "+s"(minus));
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      float a = p[r][i], b = p[r][i + 1];
#pragma unroll
      for (int k = 0; k < P8_TERMS; ++k) {
        const f16x2 h = __builtin_convertvector((f32x2{a, b}), f16x2);
        pf[r][k][i >> 3][i & 7] = h[0];
        pf[r][k][i >> 3][(i & 7) + 1] = h[1];
        if (k + 1 == P8_TERMS) break;
        a = __builtin_fmaf((float)h[0], minus, a);
        b = __builtin_fmaf((float)h[1], minus, b);
      }
    }
}

// NaN bytes (e4m3) of an operand's granule to zero: a zero weight times them would be NaN.  Whether there were any.
__device__ __forceinline__ uint32_t p8_clear_nan(u32x4& u) {
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t nan = p8_nan_bytes(u[i]);
    any |= nan;
    u[i] &= ~nan;
  }
  return any;
}

// NaN of tile t's V to the rows that see it (outputs of dims 16 d + 4 (l / 16) + i of this lane).
template <int HD, int NR>
__device__ __forceinline__ void p8_add_nan(P8Rows<HD, NR>& st, const uint8_t* vc, uint32_t page_bytes,
                                           const Paged& g, const uint32_t* tab, uint32_t t, uint32_t len,
                                           const uint32_t (&limit)[NR]) {
  const uint32_t grp = (threadIdx.x & 63u) >> 4;
#pragma unroll 1
  for (uint32_t pos = t * P8_TILE; pos < min(len, (t + 1) * P8_TILE); ++pos) {
    const uint32_t page = tab[pos >> g.shift];
    if (page >= g.n_pages) continue;
    const uint8_t* p = vc + p8_at(page, page_bytes, p8_v(g, pos & ((1u << g.shift) - 1u), 4 * grp));
#pragma unroll
    for (int d = 0; d < HD / 16; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float add = (p[(16 * d + i) * 16] & 0x7fu) == 0x7fu ? u2f(0x7fc00000u) : 0.0f;
#pragma unroll
        for (int r = 0; r < NR; ++r) st.o[r][d][i] += pos <= limit[r] ? add : 0.0f;
      }
  }
}

// One piece per workgroup; its 4 waves take the tiles in turn and join their states through LDS at the end.
template <int HD, int KT, int QT, int NR, bool STREAM>
__global__ __launch_bounds__(PA_NT, p8_per_cu(HD, NR)) void k_p8_split(P8Args p8) {
  typedef typename std::conditional<QT == TY_F32, float, typename std::conditional<QT == TY_F16, _Float16, __bf16>::type>::type QE;
  typedef QE q8v __attribute__((ext_vector_type(8)));
  constexpr int NQ = QT == TY_F32 ? 2 : 1, KS = HD / 32, DS = HD / 16, KG = HD / 64;
  constexpr int ROWS = 16 * NR, PITCH = HD + 4;
  const PaArgs& a = p8.a;
  extern __shared__ float smem[];  // [4][ROWS][PITCH] rows, [4][ROWS][2] states, [ROWS][2] factors
  float* s_ml = smem + 4 * ROWS * PITCH;
  float* s_f = s_ml + 4 * ROWS * 2;
  float* s_q = smem;  // [NR][NQ][KS][64] operands of 16 bytes
  const uint32_t tid = threadIdx.x, lane = tid & 63u, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t col = lane & 15u, grp = lane >> 4;
  const Paged& g = a.g;

  const PaPiece pc = pa_piece<NR, P8_TILE>(a, blockIdx.x, blockIdx.x == 0);
  if (!pc.any) return;
  const PaSeq& sq = pc.q;
  const uint32_t s = pc.s, h = pc.h, rb = pc.rb, t0 = pc.t0, t1 = pc.t1, group = a.group;
  const uint32_t* tab = g.table + (size_t)s * g.stride;
  const uint32_t len = sq.len, first = sq.first;
  const uint8_t *kc = reinterpret_cast<const uint8_t*>(a.kc), *vc = reinterpret_cast<const uint8_t*>(a.vc);

  // ---- tiles t0 + w, t0 + w + 4, ...: the first one's pages, then its K and V, are on their way before
  // the query rows are made ready
  const uint32_t ta = t0 + w;
  const uint32_t kpos = 16 * (col >> 2), ko = kpos + (col & 3u);  // this lane's K rows in a tile: ko + 4 b
  const size_t head_bytes = (size_t)HD << g.shift;
  const uint32_t pmask = (1u << g.shift) - 1u;
  u32x4 kf[4][KG], vf[DS];
  uint32_t ke = 0, ve = 0, odd_tile = ~0u;
  const uint32_t page_bytes = g.n_kv * HD << g.shift, page_exps = g.n_kv << (g.shift - 4);
  const uint32_t head_exps = h << (g.shift - 4);
  kc += h * head_bytes;
  vc += h * head_bytes;
  const auto load_k = [&](uint32_t pos0, uint32_t page) {
    if (page >= g.n_pages) page = 0;
    const uint8_t* p = kc + p8_at(page, page_bytes, ((grp << g.shift) + ((pos0 + ko) & pmask)) * 16);
#pragma unroll
    for (int b = 0; b < 4; ++b)  // granules of 64 dims apart
      pa_load<STREAM, KG>(reinterpret_cast<const u32x4*>(p) + 4 * b, (size_t)4 << g.shift, kf[b]);
  };
  const auto load_v = [&](uint32_t pos0, uint32_t page) {
    if (page >= g.n_pages) page = 0;
    const uint32_t o = (pos0 + 16 * grp) & pmask;
    const uint8_t* p = vc + p8_at(page, page_bytes, ((o >> 4) * HD + col) * 16);
    pa_load<STREAM, DS>(reinterpret_cast<const u32x4*>(p), 16, vf);
  };
  const auto load_e = [&](uint32_t pos0, uint32_t page) {
    if (page >= g.n_pages) page = 0;
    const uint64_t at = p8_at(page, page_exps, head_exps + (((pos0 + 16 * grp) & pmask) >> 4));
    ke = p8.ke[at];
    ve = p8.ve[at];
  };
  uint32_t pk = 0, pv = 0, pkn = 0, pvn = 0;
  if (ta < t1) {
    pk = p8_page(a, tab, ta * P8_TILE + kpos, len);
    pv = p8_page(a, tab, ta * P8_TILE + 16 * grp, len);
    pkn = p8_page(a, tab, (ta + 4) * P8_TILE + kpos, len);
    pvn = p8_page(a, tab, (ta + 4) * P8_TILE + 16 * grp, len);
  }
  // the query rows as operands in LDS: unit (row, 8 dims) of every thread, a row in HD / 8 lanes
  constexpr int LPR = HD / 8, UNITS = ROWS * LPR, PASSES = (UNITS + PA_NT - 1) / PA_NT;
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
    load_k(ta * P8_TILE, pk);
    load_e(ta * P8_TILE, pv);
    load_v(ta * P8_TILE, pv);
  }
#pragma unroll
  for (int k = 0; k < PASSES; ++k) {
    const uint32_t u = tid + k * PA_NT, row = u / LPR, d8 = u % LPR;
    uint32_t top = 0;
    if constexpr (QT != TY_F16) {
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, f2u((float)raw[k][i]) & 0x7fffffffu);
      top = pa_group_max<LPR>(top);
    }
    f16x8 term[NQ];
    const int up = p8_query<QT, NQ>(raw[k], top, a.scale < 0.0f, term);
    if (UNITS >= PA_NT || u < UNITS) {
      // dims 8 d8 are operand (d8 / 8) * 2 + d8 % 2 of lane group (d8 / 2) % 4
      const uint32_t j = (d8 >> 3) * 2 + (d8 & 1u), to = ((d8 >> 1) & 3u) * 16 + (row & 15u);
#pragma unroll
      for (int n = 0; n < NQ; ++n)
        *reinterpret_cast<f16x8*>(&s_q[((((row >> 4) * NQ + n) * KS + j) * 64 + to) * 4]) = term[n];
      if (d8 == 0) {
        const P8Factor f = p8_factor(a.scale, up);
        s_f[2 * row] = f.m;
        s_f[2 * row + 1] = u2f((uint32_t)f.e);
      }
    }
  }
  __syncthreads();
  P8Factor factor[NR];
  uint32_t limit[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const uint32_t row = rb * ROWS + r * 16 + col;
    factor[r] = P8Factor{s_f[2 * (r * 16 + col)], (int)f2u(s_f[2 * (r * 16 + col) + 1])};
    limit[r] = first + (row < sq.rows ? pa_token(a, row) : 0u);
  }
  P8Rows<HD, NR> st;
  st.clear();
  for (uint32_t t = ta; t < t1; t += 4) {
    const uint32_t pos0 = t * P8_TILE;
    const bool next = t + 4 < t1;
    f32x4 sc[NR][4];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int b = 0; b < 4; ++b) sc[r][b] = f32x4{0, 0, 0, 0};
    asm volatile("" ::: "memory");  // (the query operands stay in LDS: registers)
#pragma unroll
    for (int gi = 0; gi < KG; ++gi)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        f16x8 kk[2];
        p8_operands<KT>(kf[b][gi], kk);
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int n = NQ - 1; n >= 0; --n) {
              const f16x8 qf = *reinterpret_cast<const f16x8*>(&s_q[(((r * NQ + n) * KS + 2 * gi + j) * 64 + lane) * 4]);
              sc[r][b] = Op16<TY_F16>::mfma(kk[j], qf, sc[r][b]);
            }
      }
    const bool page_ok = pv < g.n_pages;
    const uint32_t ke_now = ke, ve_now = ve;
    uint32_t pv2 = 0;
    if (next) {
      const uint32_t pk2 = p8_page(a, tab, (t + 8) * P8_TILE + kpos, len);
      pv2 = p8_page(a, tab, (t + 8) * P8_TILE + 16 * grp, len);
      load_k(pos0 + 4 * P8_TILE, pkn);
      load_e(pos0 + 4 * P8_TILE, pvn);
      pkn = pk2;
    }
    const uint32_t gpos = pos0 + 16 * grp;  // this lane's 16 positions
    if (!page_ok) paged_flag(g, PG_BAD_PAGE);
    const bool edge = pos0 + P8_TILE - 1 > first || __ballot(!page_ok) != 0;
    f16x8 pf[NR][P8_TERMS][2];
    p8_softmax<HD, NR>(st, sc, factor, ke_now, ve_now, gpos, limit, page_ok, edge, pf);
    if (KT == TY_E4M3 && edge) {
      uint32_t odd = 0;
#pragma unroll
      for (int d = 0; d < DS; ++d) odd |= p8_clear_nan(vf[d]);
      if (__ballot(odd != 0)) odd_tile = t;
    }
#pragma unroll
    for (int d = 0; d < DS; ++d) {
      f16x8 vv[2];
      p8_operands<KT>(vf[d], vv);
#pragma unroll
      for (int n = P8_TERMS - 1; n >= 0; --n)  // the small terms first
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int k = 0; k < 2; ++k) st.o[r][d] = Op16<TY_F16>::mfma(vv[k], pf[r][n][k], st.o[r][d]);
    }
    if (odd_tile == t) p8_add_nan<HD, NR>(st, vc, page_bytes, g, tab, t, len, limit);
    if (next) {
      pv = pvn;
      pvn = pv2;
      load_v(pos0 + 4 * P8_TILE, pv);
    }
  }

  // ---- the waves' states joined; rows finished, or a part written.  Sums and rows in units of 2^24: over 2^24
  // positions of values near the largest f32 they stay below it
  __syncthreads();  // (the query operands lie where the states go)
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const float sum = pa_sum4(st.l[r]);
    if (grp == 0) {
      s_ml[(w * ROWS + r * 16 + col) * 2] = sum == 0.0f ? -INFINITY : st.m[r];  // (no position: no weight)
      s_ml[(w * ROWS + r * 16 + col) * 2 + 1] = ldexpf(sum, -24);
    }
    const int unit = (int)fmaxf(-512.0f, fminf(512.0f, st.D[r])) - 14 - 24;
#pragma unroll
    for (int d = 0; d < DS; ++d) {
      f32x4 y;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = ldexpf(st.o[r][d][i], unit);
      *reinterpret_cast<f32x4*>(&smem[(w * ROWS + r * 16 + col) * PITCH + 16 * d + 4 * grp]) = y;
    }
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
      const f32x4 z = M == -INFINITY ? f32x4{0, 0, 0, 0} : y / L;  // (no position left: zeros)
      const uint32_t t = pa_token(a, full);
      const size_t dst = ((size_t)s * a.n_new + t) * a.out_stride + (size_t)(h * group + (full - t * group)) * HD + d;
      pa_store4<QT>(a.out, dst, z);
    } else {
      *reinterpret_cast<f32x4*>(&a.part_o[((size_t)pc.slot * a.part_rows + row) * HD + d]) = y;
      if (d == 0) {
        a.part_ml[((size_t)pc.slot * a.part_rows + row) * 2] = M;
        a.part_ml[((size_t)pc.slot * a.part_rows + row) * 2 + 1] = L;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Prompts: blocks of 128 query rows (64 for heads of 256), so that a tile's K and V are turned into operands once for
// all of them, in LDS, while the tile before is worked on.  The plan is the split's; tiles behind a block's last row
// are left out.  8 waves of 16 rows within 128 registers, two workgroups a CU (with 130: 4096 tokens at 12288
// 1716 us and not 1380, 8 sequences of 43 at 4000 87 and not 74; 2048 at 0 74 and not 82); the host's rule says where 4 waves of 32 rows do better.  Weights are two f16 for
// all rows, as for up to 8 new tokens: one takes 11 to 18 % less for 16-bit rows (4096 tokens at 12288, bf16, 1114 us
// against 1363), but with its 11 bits sums whose values cancel are 2^-12 of the values' size off.
constexpr int p8p_lds(int hd) { return 2 * (2 * 64 * hd * 2 + 192) + 16; }
// Tiles of a piece at most: `at_once` (4 where the batch is small, else 16: a piece's part is written and read again,
// 64 KB), and more once that makes over 512 pieces, two for each CU.  Segments cut evenly may make some more than 512 all
// the same, which wait for all the others: an eighth more tiles then, if that brings them to 512 (512 tokens at 32256,
// 24 + 8 heads, bf16: 576 pieces 438 us, 480 324; an eighth more always: 43 at 39957 78 and 82 us).
// Where more than half of the tiles lie behind the first new position, pieces would end at the diagonal, many of them
// empty, so segments stay whole up to P8P_WHOLE tiles if there is one for each CU (2048 tokens at 0, 24 + 8 heads,
// f32: 127 us cut at 16, 77 whole; bf16 97 and 78).
struct P8PromptTarget {
  template <typename F>
  __device__ __forceinline__ uint32_t operator()(const PaArgs& a, uint32_t total, F all) const {
    const auto pieces = [&](uint32_t most) { return all([=](const PaSeq& q) { return (q.tiles + most - 1) / most; }); };
    uint32_t least = a.at_once;
    if (least > 4 && all([](const PaSeq& q) { return q.first / P8_TILE; }) < total / 2)
      least = max(least, all([](const PaSeq&) { return 1u; }) >= 256 ? P8P_WHOLE : 16u);
    const uint32_t even = (total + 511) / 512, fewer = (total + 447) / 448;
    if (even <= least) return least;
    return pieces(even) > 512 && pieces(fewer) <= 512 ? max(fewer, least) : even;
  }
};

template <int HD, int KT, int QT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, HD == 256 ? 1 : WAVES == 8 && QT != TY_F32 ? 4 : 2) void k_p8_prompt(P8Args p8) {
  typedef typename std::conditional<QT == TY_F32, float, typename std::conditional<QT == TY_F16, _Float16, __bf16>::type>::type QE;
  typedef QE q8v __attribute__((ext_vector_type(8)));
  constexpr int NQ = QT == TY_F32 ? 2 : 1, KS = HD / 32, DS = HD / 16;
  constexpr int ROWS = p8p_rows(HD), NR = ROWS / 16 / WAVES, NT = 64 * WAVES;
  constexpr int KG = (HD / 16 + WAVES - 1) / WAVES;  // granules of K (and of V) of a thread
  constexpr bool ALL = HD / 16 >= WAVES;             // else of the first HD / 16 waves
  constexpr uint32_t K_BYTES = 64 * HD * 2 + 192, BUF = K_BYTES + 64 * HD * 2;  // (64 bytes between the products' rows of K)
  const PaArgs& a = p8.a;
  extern __shared__ char lds[];  // [2] K operands [4][KS][64], V operands [DS][2][64]; [2] tiles with NaN, + 1
  uint32_t* s_odd = reinterpret_cast<uint32_t*>(lds + 2 * BUF);
  const uint32_t tid = threadIdx.x, lane = tid & 63u, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t col = lane & 15u, grp = lane >> 4;
  const Paged& g = a.g;
  PaPiece pc = pa_piece<ROWS / 16, P8_TILE, P8PromptTarget>(a, blockIdx.x, blockIdx.x == 0);
  if (!pc.any) return;
  const PaSeq& sq = pc.q;
  // KV heads next to each other, so that with 8 of them each XCD's cache sees one; the rows with the most
  // positions first
  {
    const uint32_t rest = pc.at / g.n_kv, block = rest / pc.n;
    pc.h = pc.at - rest * g.n_kv;
    pc.rb = sq.blocks - 1 - block;
    pc.place(rest - block * pc.n);
  }
  const uint32_t s = pc.s, h = pc.h, rb = pc.rb, group = a.group;
  const uint32_t* tab = g.table + (size_t)s * g.stride;
  const uint32_t len = sq.len, first = sq.first;
  const uint32_t last = first + pa_token(a, min(sq.rows, (rb + 1) * ROWS) - 1);  // position of the block's last row
  const uint32_t t0 = pc.t0, t1 = min(pc.t1, last / P8_TILE + 1);
  const uint8_t *kc = reinterpret_cast<const uint8_t*>(a.kc), *vc = reinterpret_cast<const uint8_t*>(a.vc);
  const size_t head_bytes = (size_t)HD << g.shift;
  const uint32_t pmask = (1u << g.shift) - 1u;
  const uint32_t page_bytes = g.n_kv * HD << g.shift, page_exps = g.n_kv << (g.shift - 4);
  const uint32_t head_exps = h << (g.shift - 4);
  kc += h * head_bytes;
  vc += h * head_bytes;

  // ---- query rows of this wave: operands in registers
  f16x8 qf[NR][NQ][KS];
  P8Factor factor[NR];
  uint32_t limit[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const uint32_t row = rb * ROWS + (w * NR + r) * 16 + col, t = pa_token(a, row), qh = h * group + (row - t * group);
    q8v qr[KS];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      qr[j] = q8v{};
      // dims of operand j: 8 of granule grp + 4 (j / 2)
      if (row < sq.rows)
        qr[j] = *reinterpret_cast<const q8v*>(static_cast<const QE*>(a.q) + ((size_t)s * a.n_new + t) * a.q_stride +
                                               (size_t)qh * HD + 16 * (grp + 4 * (j >> 1)) + 8 * (j & 1));
    }
    if constexpr (QT != TY_F16) {
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, f2u((float)qr[j][i]) & 0x7fffffffu);
      // (over the 4 lanes of a row)
      auto x = __builtin_amdgcn_permlane32_swap(top, top, false, false);
      top = max((uint32_t)x[0], (uint32_t)x[1]);
      auto y = __builtin_amdgcn_permlane16_swap(top, top, false, false);
      top = max((uint32_t)y[0], (uint32_t)y[1]);
    }
    int up = 0;
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      f16x8 term[NQ];
      up = p8_query<QT, NQ>(qr[j], top, a.scale < 0.0f, term);
#pragma unroll
      for (int n = 0; n < NQ; ++n) qf[r][n][j] = term[n];
    }
    factor[r] = p8_factor(a.scale, up);
    limit[r] = first + (row < sq.rows ? t : 0u);
  }

  // ---- this thread's granules of a tile: K of position tid % 64, V of dims (tid + NT i) % HD.  The next
  // tile's are on their way while one is multiplied (two tiles ahead: no gain)
  struct Raw {
    u32x4 k[KG], v[KG];
    uint32_t ke, ve;
    bool ok, v_bad[KG];
  };
  Raw raw;
  uint32_t k_page = 0, v_page[KG], e_page = 0;
  const auto v_grp = [&](int i) { return min(3u, (tid + NT * i) / HD); };
  const auto pages = [&](uint32_t t) {
    const uint32_t pos0 = t * P8_TILE;
    k_page = p8_page(a, tab, pos0 + lane, len);
    e_page = p8_page(a, tab, pos0 + 16 * grp, len);
#pragma unroll
    for (int i = 0; i < KG; ++i) v_page[i] = p8_page(a, tab, pos0 + 16 * v_grp(i), len);
  };
  // tile t's granules, then the pages of the tile behind it (those first in the queue: loads come back in order)
  const auto fetch = [&](uint32_t t, Raw& to) {
    const uint32_t pos0 = t * P8_TILE;
    const uint8_t* kp = kc + p8_at(k_page < g.n_pages ? k_page : 0u, page_bytes, ((w << g.shift) + ((pos0 + lane) & pmask)) * 16);
    const uint8_t* vp[KG];
#pragma unroll
    for (int i = 0; i < KG; ++i) {
      to.v_bad[i] = v_page[i] >= g.n_pages;
      const uint32_t block = ((pos0 + 16 * v_grp(i)) & pmask) >> 4;
      vp[i] = vc + p8_at(to.v_bad[i] ? 0u : v_page[i], page_bytes, (block * HD + (tid + NT * i) % HD) * 16);
    }
    to.ok = e_page < g.n_pages;
    const uint64_t at = p8_at(to.ok ? e_page : 0u, page_exps, head_exps + (((pos0 + 16 * grp) & pmask) >> 4));
    pages(t + 1);
    to.ke = p8.ke[at];
    to.ve = p8.ve[at];
#pragma unroll
    for (int i = 0; i < KG; ++i)
      if (ALL || w < HD / 16) to.k[i] = *reinterpret_cast<const u32x4*>(kp + (((size_t)WAVES * i) << g.shift) * 16);
#pragma unroll
    for (int i = 0; i < KG; ++i)
      if (ALL || w < HD / 16) to.v[i] = *reinterpret_cast<const u32x4*>(vp[i]);
  };
  // the granules as operands into buffer b
  const auto stage = [&](uint32_t t, uint32_t b, Raw& from) {
    if (!ALL && w >= HD / 16) return;
    char* kd = lds + b * BUF;
    char* vd = kd + K_BYTES;
    // position p: row 4 (p / 16) + p % 4 of product (p / 4) % 4
    const uint32_t prod = (lane >> 2) & 3u, pr = 4 * (lane >> 4) + (lane & 3u);
#pragma unroll
    for (int i = 0; i < KG; ++i) {
      f16x8 x[2];
      p8_operands<KT>(from.k[i], x);
      const uint32_t gi = w + WAVES * i;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        *reinterpret_cast<f16x8*>(kd + ((prod * KS + 2 * (gi >> 2) + j) * 64 + 16 * (gi & 3u) + pr) * 16 + 64 * prod) = x[j];
    }
    const bool edge = t * P8_TILE + P8_TILE - 1 > first;
#pragma unroll
    for (int i = 0; i < KG; ++i) {
      const uint32_t dim = (tid + NT * i) % HD;
      if (KT == TY_E4M3 && (edge || from.v_bad[i])) {
        const uint32_t odd = p8_clear_nan(from.v[i]);
        if (odd && !from.v_bad[i]) s_odd[b] = t + 1;
      }
      f16x8 x[2];
      p8_operands<KT>(from.v[i], x);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        *reinterpret_cast<f16x8*>(vd + (((dim >> 4) * 2 + j) * 64 + 16 * v_grp(i) + (dim & 15u)) * 16) = x[j];
    }
  };

  P8Rows<HD, NR> st;
  st.clear();
  uint32_t ke = 0, ve = 0;
  bool ok = true;
  // tile t, in buffer B
  const auto tile = [&](uint32_t t, auto which) {
    constexpr uint32_t B = which.value;
    const char* kd = lds + B * BUF;
    const char* vd = kd + K_BYTES;
    f32x4 sc[NR][4];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int k = 0; k < 4; ++k) sc[r][k] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < KS; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const f16x8 kk = *reinterpret_cast<const f16x8*>(kd + ((k * KS + j) * 64 + lane) * 16 + 64 * k);
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int n = NQ - 1; n >= 0; --n) sc[r][k] = Op16<TY_F16>::mfma(kk, qf[r][n][j], sc[r][k]);
      }
    const uint32_t gpos = t * P8_TILE + 16 * grp;  // this lane's 16 positions
    if (!ok) paged_flag(g, PG_BAD_PAGE);
    f16x8 pf[NR][P8_TERMS][2];
    p8_softmax<HD, NR>(st, sc, factor, ke, ve, gpos, limit, ok,
                           t * P8_TILE + P8_TILE - 1 > first || __ballot(!ok) != 0, pf);
    const bool odd = KT == TY_E4M3 && s_odd[B] == t + 1;
    if (t + 1 < t1) {
      stage(t + 1, B ^ 1, raw);
      ke = raw.ke;
      ve = raw.ve;
      ok = raw.ok;
      if (t + 2 < t1) fetch(t + 2, raw);
    }
#pragma unroll
    for (int d0 = 0; d0 < DS; d0 += 2)  // (two dims' chains in turn)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f16x8 vv[2];
#pragma unroll
        for (int d = 0; d < 2; ++d) vv[d] = *reinterpret_cast<const f16x8*>(vd + (((d0 + d) * 2 + k) * 64 + lane) * 16);
#pragma unroll
        for (int n = P8_TERMS - 1; n >= 0; --n)
#pragma unroll
          for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int r = 0; r < NR; ++r) st.o[r][d0 + d] = Op16<TY_F16>::mfma(vv[d], pf[r][n][k], st.o[r][d0 + d]);
      }
    if (odd) p8_add_nan<HD, NR>(st, vc, page_bytes, g, tab, t, len, limit);
    __syncthreads();
  };
  // half of the waves first: they are at their softmax while the others multiply.  Where half of the positions lie before
  // the new ones, or where there are workgroups for two rounds of all CUs; not where few workgroups of unequal lengths
  // leave CUs to one of them.  With and without: 512 tokens at 32256 324 and 344 us, 4096 at 12288 1408 and 1443, 1024
  // at 7168 223 and 224, 8 of up to 1023 at 0 67 and 70, 4 of up to 1000 at 2000 165 and 169, but 6 of those 198 and
  // 184; left out, 2048 at 0 84 and 78, 3 of up to 1023 48 and 45, but 4096 at 0 187 and 195
  if (HD == 128 && QT != TY_F32 && w < WAVES / 2 && ((pc.n > 1 && first >= len - first) || gridDim.x >= 1024))
    __builtin_amdgcn_s_setprio(1);
  if (t0 < t1) {
    if (tid < 2) s_odd[tid] = 0;
    pages(t0);
    fetch(t0, raw);
    __syncthreads();
    stage(t0, 0, raw);
    ke = raw.ke;
    ve = raw.ve;
    ok = raw.ok;
    if (t0 + 1 < t1) fetch(t0 + 1, raw);
    __syncthreads();
    for (uint32_t t = t0;;) {
      tile(t, std::integral_constant<uint32_t, 0>{});
      if (++t >= t1) break;
      tile(t, std::integral_constant<uint32_t, 1>{});
      if (++t >= t1) break;
    }
  }

  // ---- rows finished, or a part written
  if (pc.t0 == 0 && tid == 0) a.cuts[((size_t)s * g.n_kv + h) * a.blocks + rb] = make_uint2(pc.slot, pc.n);
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const uint32_t in = (w * NR + r) * 16 + col, full = rb * ROWS + in;
    const float L = ldexpf(pa_sum4(st.l[r]), -24);
    const int unit = (int)fmaxf(-512.0f, fminf(512.0f, st.D[r])) - 14 - 24;
    if (full >= sq.rows) continue;
    const uint32_t t = pa_token(a, full);
    const size_t dst = ((size_t)s * a.n_new + t) * a.out_stride + (size_t)(h * group + (full - t * group)) * HD + 4 * grp;
#pragma unroll
    for (int d = 0; d < DS; ++d) {
      f32x4 y;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = ldexpf(st.o[r][d][i], unit);
      if (pc.n == 1)
        pa_store4<QT>(a.out, dst + 16 * d, L == 0.0f ? f32x4{0, 0, 0, 0} : y / L);  // (no position left: zeros)
      else
        *reinterpret_cast<f32x4*>(&a.part_o[((size_t)pc.slot * a.part_rows + in) * HD + 16 * d + 4 * grp]) = y;
    }
    if (pc.n > 1 && grp == 0) {
      a.part_ml[((size_t)pc.slot * a.part_rows + in) * 2] = L == 0.0f ? -INFINITY : st.m[r];
      a.part_ml[((size_t)pc.slot * a.part_rows + in) * 2 + 1] = L;
    }
  }
}

}  // namespace cm
