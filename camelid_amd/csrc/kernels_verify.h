// kernels_verify.h -- speculative sampling: drafted tokens accepted or replaced so that what comes
// out is distributed as the target model's samples are.
//
// Sequence s has drafts x_0 .. x_{n-1}, target logits rows 0 .. n (row t: the distribution of the
// token at draft t's place) and a draft distribution per draft (its logits, or certainty of x_t).
// With p_t = softmax(target_t / T), q_t = softmax(draft_t / T) and uniform numbers u_0 .. in [0, 1):
//   draft t is accepted while u_t q_t(x_t) < p_t(x_t)
//   at the first one that is not, the token comes from max(p_t - q_t, 0) / sum; behind the last
//   draft from p_n: the smallest i with C_i > u S, C the inclusive prefix sums, S the whole sum
// T = 0 (or below, or NaN): the argmax, first of equals, accepts and replaces.
// Exponentials and sums are f64: the token depends on which side of one of ~1e5 prefix sums u S
// lies, and f32 sums would move the borders by more than their distances.
//
// Bound: every row's logits read once (k_vd_stats: a wave per 2048 of them, its maximum and its sum of
// exponentials; no barriers behind the loads).  139 MB of f32 logits (32 sequences with up to 5 drafts of a
// draft model, 151936 tokens) take 31.6 us, 4.4 TB/s; 20 VALU instructions a logit, 9 of them f64, are
// active in 78 % of the CUs' busy cycles, and 44 M logits take 35 us in bf16 as in f32 (83 %).  Only
// sequences that rejected a draft of a draft model read two rows again for max(p - q, 0) (k_vd_rest, spread
// over the chip like the first pass: 15 us there); otherwise the shares' sums are known.  k_vd_pick then needs
// one share's logits: latency (7 us there and for one sequence without a draft model).
// Rest and pick as one launch, the draw by the sequence's last workgroup, took 47 us: its fences write back
// and invalidate the L2.
#pragma once
#include <hip/hip_runtime.h>
#include <type_traits>
#include "device_math.h"
#include "kernels_paged.h"

namespace cm {

constexpr int VD_NT = 256;
constexpr uint32_t VD_SHARE = 2048;  // logits of one wave's share of a row
constexpr uint32_t VD_MAX_ROWS = 63;

// One share of one row: the sum of exp((l - m) / T), the largest logit m and its first index.
struct VdPart {
  double z;
  float m;
  uint32_t i;
};

// ---- exp(y / T) for y <= 0, by = 32 log2(e) / T: y by = k + r, |r| <= 1/2; 2^(k / 32) from a table in
// LDS, e^(r ln 2 / 32) as 1 + r times the cubic that meets (e^(r ln 2 / 32) - 1) / r in the four Chebyshev
// points of [-1/2, 1/2]: relative error below 1.6e-13.  32 entries of 8 bytes: every one in banks of its
// own, lanes that read the same one share it.
// (kExp2Tab: the bits of 2^(i / 32) less i << 47, so that adding k << 47 makes 2^(k / 32).)
__device__ __forceinline__ void vd_table(uint64_t* tab) {
  if (threadIdx.x < 32) tab[threadIdx.x] = kExp2Tab[threadIdx.x];
}
__device__ __forceinline__ double vd_series(double r) {
  double p = fma(r, 0x1.3b2b07bdf576cp-27, 0x1.c6b13c3469da5p-20);
  p = fma(r, p, 0x1.ebfbdff82240ap-13);
  p = fma(r, p, 0x1.62e42fef8dc67p-6);
  return fma(r, p, 1.0);
}
// Any y <= 0, -inf included; 0 below the exponent range.
__device__ __forceinline__ double vd_exp(double y, double by, const uint64_t* tab) {
  const double k = fmax(rint(y * by), -65536.0);
  const double r = fmax(fma(y, by, -k), -1.0);
  const int n = (int)k;
  // 2^(n % 32 / 32) from the table, the rest of n by ldexp (which rounds into the subnormals)
  return ldexp(vd_series(r) * u2d(tab[n & 31] + ((uint64_t)(n & 31) << 47)), n >> 5);
}
__device__ __forceinline__ bool vd_greedy(float t) { return !(t > 0.0f); }
// 32 log2(e) / T; a greedy sequence's log-probabilities are those of T = 1
__device__ __forceinline__ double vd_by(float t) {
  return 32.0 * 0x1.71547652b82fep+0 / (vd_greedy(t) ? 1.0 : (double)t);
}

// A row without a distribution: a NaN or +inf logit, or none above -inf.
__device__ __forceinline__ bool vd_bad(float m) { return !(m > -INFINITY && m < INFINITY); }

// Bits that order as the logits do, -0 as +0, NaN above all.
__device__ __forceinline__ uint32_t vd_key(float l) {
  const uint32_t u = f2u(l + 0.0f);
  return l != l ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float vd_unkey(uint32_t k) {
  return k == 0xffffffffu ? NAN : u2f((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// A lane's value moved by data-parallel moves; 0 where there is none to move.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double vd_dpp(double x) {
  const uint64_t u = d2u(x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
  return u2d(((uint64_t)hi << 32) | lo);
}
// Inclusive prefix sum over the wave.
__device__ __forceinline__ double vd_wave_scan(double x) {
  x += vd_dpp<0x111>(x);
  x += vd_dpp<0x112>(x);
  x += vd_dpp<0x114>(x);
  x += vd_dpp<0x118>(x);
  x += vd_dpp<0x142, 0xa>(x);
  x += vd_dpp<0x143, 0xc>(x);
  return x;
}
// The wave's maximum, NaN passed over, in every lane.
__device__ __forceinline__ float vd_wave_max(float x) {
  x = fmaxf(x, u2f((uint32_t)__builtin_amdgcn_update_dpp((int)f2u(x), (int)f2u(x), 0xb1, 0xf, 0xf, false)));
  x = fmaxf(x, u2f((uint32_t)__builtin_amdgcn_update_dpp((int)f2u(x), (int)f2u(x), 0x4e, 0xf, 0xf, false)));
  x = fmaxf(x, u2f((uint32_t)__builtin_amdgcn_update_dpp((int)f2u(x), (int)f2u(x), 0x141, 0xf, 0xf, false)));
  x = fmaxf(x, u2f((uint32_t)__builtin_amdgcn_update_dpp((int)f2u(x), (int)f2u(x), 0x140, 0xf, 0xf, false)));
  const auto a = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
  x = fmaxf(u2f(a[0]), u2f(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  return fmaxf(u2f(b[0]), u2f(b[1]));
}
// The wave's sum, in its last lane.
__device__ __forceinline__ double vd_wave_sum(double x) { return vd_wave_scan(x); }

// This lane's logits of the share that begins at v0: vectors of 16 bytes (rows may begin at any element),
// vector j of lane i at v0 + (64 j + i) V; -inf behind the row's end.
template <int LT>
struct VdLogits {
  static constexpr int V = LT == TY_F32 ? 4 : 8, N = 32 / V;
  typedef typename std::conditional<LT == TY_F32, float, uint16_t>::type E;
  typedef E vec __attribute__((ext_vector_type(V), aligned(sizeof(E))));
  vec x[N];
  __device__ __forceinline__ void load(const void* row, uint32_t v0, uint32_t vocab) {
    const E* p = static_cast<const E*>(row);
    const uint32_t lane = threadIdx.x & 63u;
    if (v0 + VD_SHARE <= vocab) {
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = *reinterpret_cast<const vec*>(p + v0 + (64 * j + lane) * V);
      return;
    }
    constexpr E low = LT == TY_F32 ? (E)-INFINITY : LT == TY_F16 ? (E)0xfc00u : (E)0xff80u;
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const uint32_t v = v0 + (64 * j + lane) * V + e;
        x[j][e] = v < vocab ? p[v] : low;
      }
  }
  __device__ __forceinline__ float at(int j, int e) const {
    if constexpr (LT == TY_F32) return x[j][e];
    else return from_bits16<LT>(x[j][e]);
  }
  static __device__ __forceinline__ uint32_t index(uint32_t v0, int j, int e) {
    return v0 + (64 * j + (threadIdx.x & 63u)) * V + e;
  }
};

struct VdArgs {
  const void* target;
  const void* draft;  // null: drafts are certain
  const uint32_t* tokens;
  const uint32_t* draft_lens;
  const float* temperature;
  const float* uniforms;
  VdPart* parts;      // [seq][row][share]: target rows 0 .. n_draft, then draft rows
  double* rest;       // [seq][share]: sums of max(p - q, 0) of a sequence that rejected a draft
  VdPart* judged;     // [seq][64]: what k_vd_rest's vd_accept found, the last entry's i took | state << 8
  uint32_t* accepted;
  uint32_t* out;
  float* logprobs;
  uint32_t n_draft, vocab, shares;
};

__device__ __forceinline__ uint32_t vd_rows(const VdArgs& a) { return a.draft ? 2 * a.n_draft + 1 : a.n_draft + 1; }
__device__ __forceinline__ uint32_t vd_drafts(const VdArgs& a, uint32_t s) {
  return a.draft_lens ? min(a.draft_lens[s], a.n_draft) : a.n_draft;
}
template <int LT>
__device__ __forceinline__ const void* vd_target(const VdArgs& a, uint32_t s, uint32_t t) {
  return static_cast<const char*>(a.target) + ((size_t)s * (a.n_draft + 1) + t) * a.vocab * (LT == TY_F32 ? 4 : 2);
}
template <int LT>
__device__ __forceinline__ const void* vd_draft(const VdArgs& a, uint32_t s, uint32_t t) {
  return static_cast<const char*>(a.draft) + ((size_t)s * a.n_draft + t) * a.vocab * (LT == TY_F32 ? 4 : 2);
}

// What a row's exponentials exp((l - m) / T) are taken against.  near: down to `low` = m - 704 T, an f32 well
// below m (not at tiny temperatures) and above the lowest (not at huge ones), 2^(k / 32) has a normal exponent,
// which is added as bits, and l by needs no subtraction: with m by = K + f, K whole, exp((l - m) / T) is
// 2^(-f / 32) (`factor`, once a sum) times 2^((l by - K) / 32).
struct VdRef {
  double by, md, shift, factor;
  float low;
  bool near;
};
__device__ __forceinline__ VdRef vd_ref(float m, float temp) {
  VdRef f;
  f.by = vd_by(temp);
  f.md = (double)m;
  const float span = 704.0f * (vd_greedy(temp) ? 1.0f : temp);
  f.low = m - span;
  f.near = f.low > -1e38f && span > fabsf(m) * 0x1p-16f;
  const double whole = f.near ? rint(f.md * f.by) : 0.0;
  f.shift = 0x1.8p52 - whole;
  f.factor = f.near ? vd_series(-fma(f.md, f.by, -whole)) : 1.0;
  return f;
}
// l >= low; the exponential is *a * *b * factor.
__device__ __forceinline__ void vd_exp_near(float l, const VdRef& f, const uint64_t* tab, double* a, double* b) {
  const double x = (double)l, kd = fma(x, f.by, f.shift);  // k in the low bits
  const uint32_t n = (uint32_t)d2u(kd);
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  u32x2 t = __builtin_bit_cast(u32x2, tab[n & 31u]);  // + n << 47
  t.y += n << 15;
  *a = vd_series(fma(x, f.by, f.shift - kd));
  *b = __builtin_bit_cast(double, t);
}

// The logits' exponentials of a share, one after the other, as two terms of a product that f.factor belongs
// to: 0 below e^-704 (EXACT; else some e^-704 there: nothing beside the 1 of the maximum) where f.near.
template <int LT, bool EXACT, typename F>
__device__ __forceinline__ void vd_each(const VdLogits<LT>& x, const VdRef& f, const uint64_t* tab, F take) {
  if (f.near) {
#pragma unroll
    for (int j = 0; j < x.N; ++j)
#pragma unroll
      for (int e = 0; e < x.V; ++e) {
        const float l = x.at(j, e);
        double a, b;
        vd_exp_near(fmaxf(l, f.low), f, tab, &a, &b);
        take(j, e, !EXACT || l > f.low ? a : 0.0, b);
      }
  } else {
#pragma unroll
    for (int j = 0; j < x.N; ++j)
#pragma unroll
      for (int e = 0; e < x.V; ++e) take(j, e, vd_exp((double)x.at(j, e) - f.md, f.by, tab), 1.0);
  }
}

// Each wave `per` shares of a row.
template <int LT>
__global__ __launch_bounds__(VD_NT) void k_vd_stats(VdArgs a, uint32_t per) {
  __shared__ uint64_t tab[32];
  const uint32_t groups = (a.shares + 4 * per - 1) / (4 * per), row = blockIdx.x / groups;
  const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t first = ((blockIdx.x - row * groups) * 4 + w) * per, end = min(a.shares, first + per);
  const uint32_t rows = vd_rows(a), s = row / rows, r = row - s * rows;
  const uint32_t n = vd_drafts(a, s);
  const bool is_target = r <= a.n_draft;
  const uint32_t t = is_target ? r : r - a.n_draft - 1;
  if (is_target ? t > n : t >= n) return;
  const void* src = is_target ? vd_target<LT>(a, s, t) : vd_draft<LT>(a, s, t);
  const float temp = a.temperature[s];
  const bool greedy = vd_greedy(temp);
  VdLogits<LT> x;
  if (first < end) x.load(src, first * VD_SHARE, a.vocab);
  vd_table(tab);
  __syncthreads();
  for (uint32_t share = first; share < end; ++share) {
    float m = -INFINITY;  // or NaN, where there is one
#pragma unroll
    for (int j = 0; j < x.N; ++j)
#pragma unroll
      for (int e = 0; e < x.V; ++e) m = __builtin_elementwise_maximum(m, x.at(j, e));
    m = __ballot(m != m) ? NAN : vd_wave_max(m);
    uint32_t at = 0xffffffffu;
    double z = 0.0;
    if (greedy) {  // nobody else asks for the index
#pragma unroll
      for (int j = x.N - 1; j >= 0; --j)
#pragma unroll
        for (int e = x.V - 1; e >= 0; --e)
          if (x.at(j, e) == m) at = x.index(share * VD_SHARE, j, e);
      for (int o = 32; o; o >>= 1) at = min(at, (uint32_t)__shfl_xor(at, o));
    }
    if (!vd_bad(m) && (!greedy || a.logprobs)) {
      const VdRef f = vd_ref(m, temp);
      vd_each<LT, false>(x, f, tab, [&](int, int, double p, double q) { z = fma(p, q, z); });
      z = vd_wave_sum(z) * f.factor;
    }
    if ((threadIdx.x & 63u) == 63) a.parts[(size_t)row * a.shares + share] = VdPart{z, m, at};
    if (share + 1 < end) x.load(src, (share + 1) * VD_SHARE, a.vocab);
  }
}

// Logits v0 .. v0 + 7 of a row (-inf behind its end), every load on its way before the first is used.
template <int LT>
__device__ __forceinline__ void vd_load8(const void* row, uint32_t v0, uint32_t vocab, float (&l)[8]) {
  typedef typename VdLogits<LT>::vec vec;
  constexpr int V = VdLogits<LT>::V;
  if (v0 + 8 <= vocab) {
    vec x[8 / V];
#pragma unroll
    for (int k = 0; k < 8 / V; ++k)
      x[k] = *reinterpret_cast<const vec*>(static_cast<const typename VdLogits<LT>::E*>(row) + v0 + k * V);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (LT == TY_F32) l[i] = x[i / V][i % V];
      else l[i] = from_bits16<LT>(x[i / V][i % V]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) l[i] = v0 + i < vocab ? load_as_f32<LT>(row, v0 + i) : -INFINITY;
  }
}
// exp((l - m) / T) of 8 logits, as vd_each's.
__device__ __forceinline__ void vd_exp8(const float (&l)[8], float m, float temp, const uint64_t* tab, double (&y)[8]) {
  const VdRef f = vd_ref(m, temp);
  if (f.near) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      double a, b;
      vd_exp_near(fmaxf(l[i], f.low), f, tab, &a, &b);
      y[i] = l[i] > f.low ? a * b * f.factor : 0.0;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = vd_exp((double)l[i] - f.md, f.by, tab);
  }
}

// ---- acceptance: every workgroup of k_vd_rest, else of k_vd_pick, works out its sequence's
enum { VD_DRAW = 0, VD_GREEDY = 1, VD_NONE = 2 };
struct VdShared {
  uint64_t tab[32];
  VdPart row[VD_MAX_ROWS + 1];  // a row's largest logit, its index, the sum over the row
  uint32_t took, state;
};

template <int LT>
__device__ __forceinline__ void vd_accept(const VdArgs& a, uint32_t s, VdShared& sh) {
  const uint32_t tid = threadIdx.x, rows = vd_rows(a), n = vd_drafts(a, s);
  const float temp = a.temperature[s];
  const bool greedy = vd_greedy(temp);
  const double by = vd_by(temp);
  // what draft t is judged by: lane t of the last wave fetches it while the others sum up the rows
  const uint32_t t = tid - (VD_NT - 64);
  uint32_t x_t = 0xffffffffu;
  float u_t = 0.0f, lp_t = 0.0f, lq_t = 0.0f;
  if (tid >= VD_NT - 64 && t < n) {
    x_t = a.tokens[(size_t)s * a.n_draft + t];
    u_t = a.uniforms[(size_t)s * (a.n_draft + 1) + t];
    if (x_t < a.vocab) {
      lp_t = load_as_f32<LT>(vd_target<LT>(a, s, t), x_t);
      if (a.draft) lq_t = load_as_f32<LT>(vd_draft<LT>(a, s, t), x_t);
    }
  }
  vd_table(sh.tab);
  __syncthreads();
  for (uint32_t r = tid >> 4; r < rows; r += VD_NT / 16) {  // 16 lanes a row, 8 shares a lane at a time
    const uint32_t t = r <= a.n_draft ? r : r - a.n_draft - 1, lane = tid & 15u;
    if (r <= a.n_draft ? t > n : t >= n) continue;
    const VdPart* p = a.parts + ((size_t)s * rows + r) * a.shares;
    uint32_t top = 0, at = 0xffffffffu;
    double z = 0.0;
    for (uint32_t b = lane; b < a.shares; b += 128) {
      VdPart q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = b + 16 * i < a.shares ? p[b + 16 * i] : VdPart{0.0, -INFINITY, 0xffffffffu};
      const uint32_t was = top;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t k = vd_key(q[i].m);
        at = k > top ? q[i].i : at;
        top = max(top, k);
      }
      const float m = vd_unkey(top);
      if (!vd_bad(m)) {
        if (was) z *= vd_exp((double)vd_unkey(was) - (double)m, by, sh.tab);
        float l[8];
        double e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) l[i] = q[i].m;
        vd_exp8(l, m, temp, sh.tab, e);
#pragma unroll
        for (int i = 0; i < 8; ++i) z += q[i].z * e[i];
      }
    }
    // the 16 lanes' sums against the row's maximum (a lane without a finite one holds z = 0)
    const uint32_t mine = top;
    for (int o = 8; o; o >>= 1) {
      const uint32_t k2 = __shfl_xor(top, o), i2 = __shfl_xor(at, o);
      at = k2 > top || (k2 == top && i2 < at) ? i2 : at;
      top = max(top, k2);
    }
    const float m = vd_unkey(top);
    if (!vd_bad(m)) z *= vd_exp((double)vd_unkey(mine) - (double)m, by, sh.tab);
    for (int o = 8; o; o >>= 1) z += __shfl_xor(z, o);
    if (lane == 0) sh.row[r] = VdPart{z, m, at};
  }
  __syncthreads();
  if (tid >= VD_NT - 64) {  // a lane per draft
    bool go = false, none = false;
    if (t <= n) {
      const VdPart P = sh.row[t];
      none = vd_bad(P.m) || (t < n && a.draft && !greedy && vd_bad(sh.row[a.n_draft + 1 + t].m));
      if (t < n && !none) {
        if (greedy) {
          go = x_t == P.i;
        } else if (x_t < a.vocab) {
          const double px = vd_exp((double)lp_t - (double)P.m, by, sh.tab) / P.z;
          double qx = 1.0;
          if (a.draft) {
            const VdPart Q = sh.row[a.n_draft + 1 + t];
            qx = vd_exp((double)lq_t - (double)Q.m, by, sh.tab) / Q.z;
          }
          go = (double)u_t * qx < px;
        }
      }
    }
    const uint32_t took = __builtin_ctzll(~__ballot(go));  // (lane n does not go on)
    if (t == took) {
      sh.took = took;
      sh.state = none ? VD_NONE : greedy ? VD_GREEDY : VD_DRAW;
    }
  }
  __syncthreads();
}

// Draft distributions only: the sums of max(p - q, 0) over the shares, a wave each.
template <int LT>
__global__ __launch_bounds__(VD_NT) void k_vd_rest(VdArgs a) {
  __shared__ VdShared sh;
  const uint32_t groups = (a.shares + 3) / 4, s = blockIdx.x / groups;
  const uint32_t share = (blockIdx.x - s * groups) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  vd_accept<LT>(a, s, sh);
  const uint32_t took = sh.took;
  if (share < 4 && threadIdx.x <= VD_MAX_ROWS)  // the sequence's first workgroup
    a.judged[(size_t)s * (VD_MAX_ROWS + 1) + threadIdx.x] =
        threadIdx.x < VD_MAX_ROWS ? sh.row[threadIdx.x] : VdPart{0.0, 0.0f, took | sh.state << 8};
  if (sh.state != VD_DRAW || took >= vd_drafts(a, s) || share >= a.shares) return;
  VdLogits<LT> x, y;
  x.load(vd_target<LT>(a, s, took), share * VD_SHARE, a.vocab);
  y.load(vd_draft<LT>(a, s, took), share * VD_SHARE, a.vocab);
  const VdPart P = sh.row[took], Q = sh.row[a.n_draft + 1 + took];
  const float temp = a.temperature[s];
  const VdRef fp = vd_ref(P.m, temp), fq = vd_ref(Q.m, temp);
  const double ip = fp.factor / P.z, iq = fq.factor / Q.z;
  double p[32], sum = 0.0;
  vd_each<LT, true>(x, fp, sh.tab, [&](int j, int e, double u, double v) { p[j * x.V + e] = u * v * ip; });
  vd_each<LT, true>(y, fq, sh.tab, [&](int j, int e, double u, double v) { sum += fmax(p[j * x.V + e] - u * v * iq, 0.0); });
  sum = vd_wave_sum(sum);
  if ((threadIdx.x & 63u) == 63) a.rest[(size_t)s * a.shares + share] = sum;
}

// Inclusive prefix sum over the workgroup; *total the whole.
__device__ __forceinline__ double vd_scan(double v, double* wave_sums, double* total) {
  const uint32_t lane = threadIdx.x & 63u, w = threadIdx.x >> 6;
  v = vd_wave_scan(v);
  if (lane == 63) wave_sums[w] = v;
  __syncthreads();
  double all = 0.0;
  for (uint32_t i = 0; i < VD_NT / 64; ++i) {
    if (i == w) v += all;
    all += wave_sums[i];
  }
  __syncthreads();
  *total = all;
  return v;
}

// The first thread's `found`, or the last thread's `last` where nobody found anything (threads hold
// ascending indexes; ~0: none; 0 where there is neither).
__device__ __forceinline__ uint32_t vd_first_or_last(uint32_t found, uint32_t last, uint2* waves) {
  const uint64_t f = __ballot(found != 0xffffffffu), l = __ballot(last != 0xffffffffu);
  const uint32_t a = f ? __builtin_amdgcn_readlane(found, __builtin_ctzll(f)) : 0xffffffffu;
  const uint32_t b = l ? __builtin_amdgcn_readlane(last, 63 - __builtin_clzll(l)) : 0xffffffffu;
  if ((threadIdx.x & 63u) == 0) waves[threadIdx.x >> 6] = make_uint2(a, b);
  __syncthreads();
  uint32_t first = 0xffffffffu, end = 0;
  for (uint32_t i = 0; i < VD_NT / 64; ++i) {
    const uint2 x = waves[i];
    first = min(first, x.x);
    end = x.y != 0xffffffffu ? x.y : end;
  }
  __syncthreads();
  return first != 0xffffffffu ? first : end;
}

// One workgroup per sequence: acceptance, the share that the number falls into, the token in it.
template <int LT>
__global__ __launch_bounds__(VD_NT) void k_vd_pick(VdArgs a) {
  __shared__ VdShared sh;
  __shared__ double wave_sums[VD_NT / 64];
  __shared__ double s_x;
  __shared__ uint2 waves[VD_NT / 64];
  __shared__ double s_before;
  const uint32_t s = blockIdx.x, tid = threadIdx.x, n = vd_drafts(a, s);
  if (a.draft) {  // k_vd_rest has worked it out (32 sequences: 6.9 us, 9.4 with working it out again)
    vd_table(sh.tab);
    if (tid <= VD_MAX_ROWS) {
      const VdPart x = a.judged[(size_t)s * (VD_MAX_ROWS + 1) + tid];
      sh.row[tid] = x;
      if (tid == VD_MAX_ROWS) {
        sh.took = x.i & 0xffu;
        sh.state = x.i >> 8;
      }
    }
    __syncthreads();
  } else {
    vd_accept<LT>(a, s, sh);
  }
  const uint32_t took = sh.took, state = sh.state;
  const float temp = a.temperature[s];
  const double by = vd_by(temp);
  const uint32_t* tok = a.tokens + (size_t)s * a.n_draft;
  uint32_t pick = 0xffffffffu;
  if (state == VD_GREEDY) {
    pick = sh.row[took].i;
  } else if (state == VD_DRAW) {
    const VdPart P = sh.row[took];
    const bool rejected = took < n, apart = rejected && a.draft;  // apart: max(p - q, 0), in units of p
    const VdPart Q = apart ? sh.row[a.n_draft + 1 + took] : P;
    const uint32_t x_tok = rejected && !a.draft ? tok[took] : 0xffffffffu;  // its whole mass is taken away
    const void* prow = vd_target<LT>(a, s, took);
    const void* qrow = apart ? vd_draft<LT>(a, s, took) : prow;
    const VdPart* parts = a.parts + ((size_t)s * vd_rows(a) + took) * a.shares;
    // this thread's 8 logits of a share: their masses (without a draft distribution in units of
    // exp((l - max) / T))
    const double ip = 1.0 / P.z, iq = 1.0 / Q.z;
    const auto masses = [&](uint32_t share, bool whole, double (&m)[8]) {
      const uint32_t v0 = share * VD_SHARE + tid * 8;
      float lp[8], lq[8];
      vd_load8<LT>(prow, v0, a.vocab, lp);
      if (apart && !whole) vd_load8<LT>(qrow, v0, a.vocab, lq);
      vd_exp8(lp, P.m, temp, sh.tab, m);
      if (apart && !whole) {
        double q[8];
        vd_exp8(lq, Q.m, temp, sh.tab, q);
#pragma unroll
        for (int i = 0; i < 8; ++i) m[i] = fmax(m[i] * ip - q[i] * iq, 0.0);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) m[i] = v0 + i < a.vocab && (whole || v0 + i != x_tok) ? m[i] : 0.0;
    };
    double m[8];
    if (x_tok < a.vocab) {  // the share of a certain draft, without it
      masses(x_tok / VD_SHARE, false, m);
      double sum = 0.0, total;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += m[i];
      vd_scan(sum, wave_sums, &total);
      if (tid == 0) s_x = total;
      __syncthreads();
    }
    const uint32_t per = (a.shares + VD_NT - 1) / VD_NT, i0 = min(a.shares, tid * per), i1 = min(a.shares, i0 + per);
    bool whole = false;
    double total = 0.0, before = 0.0, first_sum = 0.0;
    const auto share_sum = [&](uint32_t i) {
      if (apart && !whole) return a.rest[(size_t)s * a.shares + i];
      if (!whole && i == x_tok / VD_SHARE && x_tok < a.vocab) return s_x;
      return parts[i].z * vd_exp((double)parts[i].m - (double)P.m, by, sh.tab);
    };
    for (int again = 0; again < 2; ++again) {  // (nothing left: p itself)
      double sum = 0.0;
      first_sum = i0 < i1 ? share_sum(i0) : 0.0;
      for (uint32_t i = i0; i < i1; ++i) sum += i == i0 ? first_sum : share_sum(i);
      const double incl = vd_scan(sum, wave_sums, &total);
      before = incl - sum;
      if (total > 0.0) break;
      whole = true;
    }
    const double want = (double)a.uniforms[(size_t)s * (a.n_draft + 1) + a.n_draft] * total;
    uint32_t share;  // (u S rounded up to S: the last with any mass)
    {
      double c = before;
      uint32_t last = 0xffffffffu, found = 0xffffffffu;
      for (uint32_t i = i0; i < i1; ++i) {
        const double y = i == i0 ? first_sum : share_sum(i);
        c += y;
        if (y > 0.0) last = i;
        if (c > want && y > 0.0) {
          found = i;
          break;
        }
      }
      share = vd_first_or_last(found, last, waves);
    }
    if (share >= i0 && share < i1) {
      double c = before;
      for (uint32_t i = i0; i < share; ++i) c += i == i0 ? first_sum : share_sum(i);
      s_before = c;
    }
    __syncthreads();
    masses(share, whole, m);
    double sum = 0.0, unused;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += m[i];
    const double incl = vd_scan(sum, wave_sums, &unused);
    {
      double c = s_before + (incl - sum);
      uint32_t last = 0xffffffffu, found = 0xffffffffu;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t v = share * VD_SHARE + tid * 8 + i;
        c += m[i];
        if (m[i] > 0.0) {
          last = v;
          if (c > want && found == 0xffffffffu) found = v;
        }
      }
      pick = vd_first_or_last(found, last, waves);
    }
  }
  if (tid == 0) a.accepted[s] = took;
  if (tid <= a.n_draft) {
    const uint32_t x = tid < took ? tok[tid] : tid == took ? pick : 0xffffffffu;
    a.out[(size_t)s * (a.n_draft + 1) + tid] = x;
    if (a.logprobs) {
      float lp = 0.0f;
      if (tid <= took) {
        lp = NAN;
        if (x < a.vocab) {
          const VdPart R = sh.row[tid];
          const double y = (double)load_as_f32<LT>(vd_target<LT>(a, s, tid), x) - (double)R.m;
          lp = (float)(y / (vd_greedy(temp) ? 1.0 : (double)temp) - log(R.z));
        }
      }
      a.logprobs[(size_t)s * (a.n_draft + 1) + tid] = lp;
    }
  }
}

}  // namespace cm
