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
// exponentials; no barriers behind the loads), where 12 f64 operations a logit take about 0.6 of the
// time that f32 logits take to arrive from HBM.  Only sequences that rejected a draft of a draft
// model read two rows again for max(p - q, 0) (k_vd_rest, spread over the chip like the first pass);
// otherwise the shares' sums are known.  k_vd_pick then needs one share's logits.
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

// ---- 2^(x / 64) for whole x: a table of 64 powers in LDS
__device__ __forceinline__ void vd_table(double* tab) {
  if (threadIdx.x < 64) tab[threadIdx.x] = exp2((double)threadIdx.x / 64.0);
}
// exp(y / T) for y <= 0, by = 64 log2(e) / T: y by = k + r, |r| <= 1/2; 2^(k / 64) from the table, e^(r ln 2 / 64)
// by its series to the fifth power (the next term is below 4e-17).
__device__ __forceinline__ double vd_exp(double y, double by, const double* tab) {
  constexpr double A = 0x1.62e42fefa39efp-1 / 64.0;  // ln 2 / 64
  const double k = fmax(rint(y * by), -131072.0);  // (2^-2048 and below, y = -inf: 0)
  const double r = fmax(fma(y, by, -k), -1.0);
  const int n = (int)k;
  double p = fma(r, A * A * A * A * A / 120.0, A * A * A * A / 24.0);
  p = fma(r, p, A * A * A / 6.0);
  p = fma(r, p, A * A / 2.0);
  p = fma(r, p, A);
  p = fma(r, p, 1.0);
  return ldexp(p * tab[n & 63], n >> 6);
}

__device__ __forceinline__ bool vd_greedy(float t) { return !(t > 0.0f); }
// 64 log2(e) / T; a greedy sequence's log-probabilities are those of T = 1
__device__ __forceinline__ double vd_by(float t) {
  return 64.0 * 0x1.71547652b82fep+0 / (vd_greedy(t) ? 1.0 : (double)t);
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

__device__ __forceinline__ double vd_wave_sum(double v) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

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

// Each wave a share of a row: grid (4 shares, row) flattened.
template <int LT>
__global__ __launch_bounds__(VD_NT) void k_vd_stats(VdArgs a) {
  __shared__ double tab[64];
  const uint32_t groups = (a.shares + 3) / 4, row = blockIdx.x / groups;
  const uint32_t share = (blockIdx.x - row * groups) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t rows = vd_rows(a), s = row / rows, r = row - s * rows;
  const uint32_t n = vd_drafts(a, s);
  const bool is_target = r <= a.n_draft;
  const uint32_t t = is_target ? r : r - a.n_draft - 1;
  if (is_target ? t > n : t >= n) return;
  const bool live = share < a.shares;
  VdLogits<LT> x;
  const uint32_t v0 = share * VD_SHARE;
  const float temp = a.temperature[s];
  if (live) x.load(is_target ? vd_target<LT>(a, s, t) : vd_draft<LT>(a, s, t), v0, a.vocab);
  vd_table(tab);
  __syncthreads();
  if (!live) return;
  uint32_t top = 0, at = 0xffffffffu;
#pragma unroll
  for (int j = 0; j < x.N; ++j)
#pragma unroll
    for (int e = 0; e < x.V; ++e) top = max(top, vd_key(x.at(j, e)));
  for (int o = 32; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor(top, o));
#pragma unroll
  for (int j = x.N - 1; j >= 0; --j)
#pragma unroll
    for (int e = x.V - 1; e >= 0; --e)
      if (vd_key(x.at(j, e)) == top) at = x.index(v0, j, e);
  for (int o = 32; o; o >>= 1) at = min(at, (uint32_t)__shfl_xor(at, o));
  const float m = vd_unkey(top);
  double z = 0.0;
  if (!vd_bad(m)) {
    const double by = vd_by(temp), md = (double)m;
#pragma unroll
    for (int j = 0; j < x.N; ++j)
#pragma unroll
      for (int e = 0; e < x.V; ++e) z += vd_exp((double)x.at(j, e) - md, by, tab);
    z = vd_wave_sum(z);
  }
  if ((threadIdx.x & 63u) == 0) a.parts[(size_t)row * a.shares + share] = VdPart{z, m, at};
}

// ---- acceptance: every workgroup of k_vd_rest and k_vd_pick works out its sequence's
enum { VD_DRAW = 0, VD_GREEDY = 1, VD_NONE = 2 };
struct VdShared {
  double tab[64];
  VdPart row[VD_MAX_ROWS + 1];  // a row's largest logit, its index, the sum over the row
  uint32_t took, state;
};

template <int LT>
__device__ __forceinline__ void vd_accept(const VdArgs& a, uint32_t s, VdShared& sh) {
  const uint32_t tid = threadIdx.x, rows = vd_rows(a), n = vd_drafts(a, s);
  const float temp = a.temperature[s];
  const bool greedy = vd_greedy(temp);
  const double by = vd_by(temp);
  vd_table(sh.tab);
  __syncthreads();
  for (uint32_t r = tid >> 4; r < rows; r += VD_NT / 16) {  // 16 lanes a row
    const uint32_t t = r <= a.n_draft ? r : r - a.n_draft - 1, lane = tid & 15u;
    if (r <= a.n_draft ? t > n : t >= n) continue;
    const VdPart* p = a.parts + ((size_t)s * rows + r) * a.shares;
    uint32_t top = 0, at = 0xffffffffu;
    for (uint32_t i = lane; i < a.shares; i += 16) {
      const uint32_t k = vd_key(p[i].m);
      if (k > top) {
        top = k;
        at = p[i].i;
      }
    }
    for (int o = 8; o; o >>= 1) {
      const uint32_t k2 = __shfl_xor(top, o), i2 = __shfl_xor(at, o);
      if (k2 > top || (k2 == top && i2 < at)) {
        top = k2;
        at = i2;
      }
    }
    const float m = vd_unkey(top);
    double z = 0.0;
    if (!vd_bad(m))
      for (uint32_t i = lane; i < a.shares; i += 16) z += p[i].z * vd_exp((double)p[i].m - (double)m, by, sh.tab);
    for (int o = 8; o; o >>= 1) z += __shfl_xor(z, o);
    if (lane == 0) sh.row[r] = VdPart{z, m, at};
  }
  __syncthreads();
  if (tid < 64) {  // a lane per draft
    const uint32_t t = tid;
    bool go = false, none = false;
    if (t <= n) {
      const VdPart P = sh.row[t];
      none = vd_bad(P.m) || (t < n && a.draft && !greedy && vd_bad(sh.row[a.n_draft + 1 + t].m));
      if (t < n && !none) {
        const uint32_t x = a.tokens[(size_t)s * a.n_draft + t];
        if (greedy) {
          go = x == P.i;
        } else if (x < a.vocab) {
          const double px = vd_exp((double)load_as_f32<LT>(vd_target<LT>(a, s, t), x) - (double)P.m, by, sh.tab) / P.z;
          double qx = 1.0;
          if (a.draft) {
            const VdPart Q = sh.row[a.n_draft + 1 + t];
            qx = vd_exp((double)load_as_f32<LT>(vd_draft<LT>(a, s, t), x) - (double)Q.m, by, sh.tab) / Q.z;
          }
          go = (double)a.uniforms[(size_t)s * (a.n_draft + 1) + t] * qx < px;
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

// max(p - q, 0) of this lane's logits of a share, in its order
template <int LT, typename F>
__device__ __forceinline__ void vd_rest_of(const VdLogits<LT>& x, const VdLogits<LT>& y, VdPart P, VdPart Q, double by,
                                           const double* tab, F take) {
  const double ip = 1.0 / P.z, iq = 1.0 / Q.z, mp = (double)P.m, mq = (double)Q.m;
#pragma unroll
  for (int j = 0; j < x.N; ++j)
#pragma unroll
    for (int e = 0; e < x.V; ++e)
      take(j, e, fmax(vd_exp((double)x.at(j, e) - mp, by, tab) * ip - vd_exp((double)y.at(j, e) - mq, by, tab) * iq, 0.0));
}

// Draft distributions only: the sums of max(p - q, 0) over the shares, a wave each.
template <int LT>
__global__ __launch_bounds__(VD_NT) void k_vd_rest(VdArgs a) {
  __shared__ VdShared sh;
  const uint32_t groups = (a.shares + 3) / 4, s = blockIdx.x / groups;
  const uint32_t share = (blockIdx.x - s * groups) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  vd_accept<LT>(a, s, sh);
  const uint32_t took = sh.took;
  if (sh.state != VD_DRAW || took >= vd_drafts(a, s) || share >= a.shares) return;
  VdLogits<LT> x, y;
  x.load(vd_target<LT>(a, s, took), share * VD_SHARE, a.vocab);
  y.load(vd_draft<LT>(a, s, took), share * VD_SHARE, a.vocab);
  double sum = 0.0;
  vd_rest_of<LT>(x, y, sh.row[took], sh.row[a.n_draft + 1 + took], vd_by(a.temperature[s]), sh.tab,
                 [&](int, int, double v) { sum += v; });
  sum = vd_wave_sum(sum);
  if ((threadIdx.x & 63u) == 0) a.rest[(size_t)s * a.shares + share] = sum;
}

// Inclusive prefix sum over the workgroup; *total the whole.
__device__ __forceinline__ double vd_scan(double v, double* wave_sums, double* total) {
  const uint32_t lane = threadIdx.x & 63u, w = threadIdx.x >> 6;
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(v, o);
    if (lane >= (uint32_t)o) v += y;
  }
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

// One workgroup per sequence: acceptance, the share that the number falls into, the token in it.
template <int LT>
__global__ __launch_bounds__(VD_NT) void k_vd_pick(VdArgs a) {
  __shared__ VdShared sh;
  __shared__ double wave_sums[VD_NT / 64];
  __shared__ double s_x;
  __shared__ uint32_t s_first, s_last, s_share;
  __shared__ double s_before;
  const uint32_t s = blockIdx.x, tid = threadIdx.x, n = vd_drafts(a, s);
  vd_accept<LT>(a, s, sh);
  const uint32_t took = sh.took, state = sh.state;
  const double by = vd_by(a.temperature[s]);
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
    const auto masses = [&](uint32_t share, bool whole, double (&m)[8]) {
      const uint32_t v0 = share * VD_SHARE + tid * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t v = v0 + i;
        double y = 0.0;
        if (v < a.vocab && (whole || v != x_tok)) {
          y = vd_exp((double)load_as_f32<LT>(prow, v) - (double)P.m, by, sh.tab);
          if (apart && !whole)
            y = fmax(y * (1.0 / P.z) - vd_exp((double)load_as_f32<LT>(qrow, v) - (double)Q.m, by, sh.tab) * (1.0 / Q.z), 0.0);
        }
        m[i] = y;
      }
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
    double total = 0.0, before = 0.0;
    const auto share_sum = [&](uint32_t i) {
      if (apart && !whole) return a.rest[(size_t)s * a.shares + i];
      if (!whole && i == x_tok / VD_SHARE && x_tok < a.vocab) return s_x;
      return parts[i].z * vd_exp((double)parts[i].m - (double)P.m, by, sh.tab);
    };
    for (int round = 0; round < 2; ++round) {  // (nothing left: p itself)
      double sum = 0.0;
      for (uint32_t i = i0; i < i1; ++i) sum += share_sum(i);
      const double incl = vd_scan(sum, wave_sums, &total);
      before = incl - sum;
      if (total > 0.0) break;
      whole = true;
    }
    const double want = (double)a.uniforms[(size_t)s * (a.n_draft + 1) + a.n_draft] * total;
    if (tid == 0) {
      s_first = s_share = 0xffffffffu;
      s_last = 0;
    }
    __syncthreads();
    {
      double c = before;
      uint32_t last = 0xffffffffu, found = 0xffffffffu;
      for (uint32_t i = i0; i < i1; ++i) {
        const double y = share_sum(i);
        c += y;
        if (y > 0.0) last = i;
        if (c > want && y > 0.0) {
          found = i;
          break;
        }
      }
      if (found != 0xffffffffu) atomicMin(&s_share, found);
      if (last != 0xffffffffu) atomicMax(&s_last, last);
    }
    __syncthreads();
    const uint32_t share = s_share != 0xffffffffu ? s_share : s_last;  // (u S rounded up to S: the last with any mass)
    if (share >= i0 && share < i1) {
      double c = before;
      for (uint32_t i = i0; i < share; ++i) c += share_sum(i);
      s_before = c;
    }
    __syncthreads();
    masses(share, whole, m);
    double sum = 0.0, unused;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += m[i];
    const double incl = vd_scan(sum, wave_sums, &unused);
    if (tid == 0) s_last = 0;
    __syncthreads();
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
      if (found != 0xffffffffu) atomicMin(&s_first, found);
      if (last != 0xffffffffu) atomicMax(&s_last, last);
    }
    __syncthreads();
    pick = s_first != 0xffffffffu ? s_first : s_last;
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
          const float temp = a.temperature[s];
          const double y = (double)load_as_f32<LT>(vd_target<LT>(a, s, tid), x) - (double)R.m;
          lp = (float)(y / (vd_greedy(temp) ? 1.0 : (double)temp) - log(R.z));
        }
      }
      a.logprobs[(size_t)s * (a.n_draft + 1) + tid] = lp;
    }
  }
}

}  // namespace cm
