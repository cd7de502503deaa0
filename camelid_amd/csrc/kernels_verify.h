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
#pragma once
#include <hip/hip_runtime.h>
#include "device_math.h"
#include "kernels_paged.h"

namespace cm {

constexpr int VD_NT = 256;
constexpr uint32_t VD_CHUNK = 4096;  // logits of one workgroup's share of a row

// One share of one row: the largest logit, its first index, and the sum of exp((l - max) / T).
struct VdPart {
  double z;
  float m;
  uint32_t i;
};

// exp((l - m) / T) for l <= m, m finite
__device__ __forceinline__ double vd_exp(float l, float m, double inv_t) {
  return l == -INFINITY ? 0.0 : exp(((double)l - (double)m) * inv_t);
}

__device__ __forceinline__ bool vd_greedy(float t) { return !(t > 0.0f); }
// 1 / T; a greedy sequence's log-probabilities are those of T = 1
__device__ __forceinline__ double vd_inv(float t) { return vd_greedy(t) ? 1.0 : 1.0 / (double)t; }

// A row without a distribution: a NaN or +inf logit, or none above -inf.
__device__ __forceinline__ bool vd_bad(float m) { return !(m > -INFINITY && m < INFINITY); }

// (m, i) of the larger logit; a NaN is larger than all; the lower index of equals.
__device__ __forceinline__ void vd_max(float& m, uint32_t& i, float m2, uint32_t i2) {
  const bool take = (m2 != m2) ? (m == m || i2 < i) : (m == m && (m2 > m || (m2 == m && i2 < i)));
  if (take) {
    m = m2;
    i = i2;
  }
}

__device__ __forceinline__ double vd_wave_sum(double v) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// Row r of a sequence: rows [0, n_draft] target, [n_draft + 1, 2 n_draft] draft t = r - n_draft - 1.
template <int LT>
__global__ __launch_bounds__(VD_NT) void k_vd_stats(const void* __restrict__ target, const void* __restrict__ draft,
                                                    const uint32_t* __restrict__ draft_lens, uint32_t n_draft,
                                                    uint32_t vocab, const float* __restrict__ temperature,
                                                    VdPart* __restrict__ parts) {
  __shared__ float sm[VD_NT / 64];
  __shared__ uint32_t si[VD_NT / 64];
  __shared__ double sz[VD_NT / 64];
  const uint32_t rows = draft ? 2 * n_draft + 1 : n_draft + 1;
  const uint32_t s = blockIdx.y / rows, r = blockIdx.y % rows;
  const uint32_t n = draft_lens ? min(draft_lens[s], n_draft) : n_draft;
  const bool is_target = r <= n_draft;
  const uint32_t t = is_target ? r : r - n_draft - 1;
  if (is_target ? t > n : t >= n) return;
  const void* src = is_target ? target : draft;
  const size_t base = ((size_t)s * (is_target ? n_draft + 1 : n_draft) + t) * vocab;
  const uint32_t v0 = blockIdx.x * VD_CHUNK, v1 = min(vocab, v0 + VD_CHUNK);
  float m = -INFINITY;
  uint32_t at = v0;
  for (uint32_t v = v0 + threadIdx.x; v < v1; v += VD_NT) vd_max(m, at, load_as_f32<LT>(src, base + v), v);
  for (int o = 32; o; o >>= 1) {
    const float m2 = __shfl_xor(m, o);
    const uint32_t i2 = __shfl_xor(at, o);
    vd_max(m, at, m2, i2);
  }
  const uint32_t w = threadIdx.x >> 6;
  if ((threadIdx.x & 63u) == 0) {
    sm[w] = m;
    si[w] = at;
  }
  __syncthreads();
  m = sm[0];
  at = si[0];
  for (int i = 1; i < VD_NT / 64; ++i) vd_max(m, at, sm[i], si[i]);
  double z = 0.0;
  if (!vd_bad(m)) {
    const double inv_t = vd_inv(temperature[s]);
    for (uint32_t v = v0 + threadIdx.x; v < v1; v += VD_NT) z += vd_exp(load_as_f32<LT>(src, base + v), m, inv_t);
  }
  z = vd_wave_sum(z);
  if ((threadIdx.x & 63u) == 0) sz[w] = z;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < VD_NT / 64; ++i) z += sz[i];
    parts[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = VdPart{z, m, at};
  }
}

// A row's statistics from its shares.
__device__ __forceinline__ VdPart vd_row(const VdPart* p, uint32_t n, double inv_t) {
  float m = p[0].m;
  uint32_t at = p[0].i;
  for (uint32_t i = 1; i < n; ++i) vd_max(m, at, p[i].m, p[i].i);
  double z = 0.0;
  if (!vd_bad(m))
    for (uint32_t i = 0; i < n; ++i) z += p[i].z * vd_exp(p[i].m, m, inv_t);
  return VdPart{z, m, at};
}

// One workgroup per sequence: acceptance, then the token drawn at the row where it ends.
constexpr int VP_NT = 1024;
template <int LT>
__global__ __launch_bounds__(VP_NT) void k_vd_pick(const void* __restrict__ target, const void* __restrict__ draft,
                                                   const uint32_t* __restrict__ tokens,
                                                   const uint32_t* __restrict__ draft_lens, uint32_t n_draft,
                                                   uint32_t vocab, const float* __restrict__ temperature,
                                                   const float* __restrict__ uniforms, uint32_t n_parts,
                                                   const VdPart* __restrict__ parts, uint32_t* __restrict__ accepted,
                                                   uint32_t* __restrict__ out, float* __restrict__ logprobs) {
  __shared__ VdPart s_row[64];
  __shared__ uint32_t s_took, s_state;  // state 0: draw, 1: greedy, 2: no distribution
  __shared__ double s_sum[VP_NT];
  __shared__ uint32_t s_pick;
  const uint32_t s = blockIdx.x, tid = threadIdx.x;
  const uint32_t rows = draft ? 2 * n_draft + 1 : n_draft + 1;
  const uint32_t n = draft_lens ? min(draft_lens[s], n_draft) : n_draft;
  const float temp = temperature[s];
  const bool greedy = vd_greedy(temp);
  const double inv_t = vd_inv(temp);
  if (tid < rows) {
    const uint32_t t = tid <= n_draft ? tid : tid - n_draft - 1;
    if (tid <= n_draft ? t <= n : t < n) s_row[tid] = vd_row(parts + ((size_t)s * rows + tid) * n_parts, n_parts, inv_t);
  }
  __syncthreads();
  const uint32_t* tok = tokens + (size_t)s * n_draft;
  const float* u = uniforms + (size_t)s * (n_draft + 1);
  if (tid == 0) {
    uint32_t t = 0, state = greedy ? 1 : 0;
    for (;; ++t) {
      const VdPart& P = s_row[t];
      if (vd_bad(P.m)) state = 2;
      if (t < n && draft && !greedy && vd_bad(s_row[n_draft + 1 + t].m)) state = 2;
      if (t == n || state == 2) break;
      const uint32_t x = tok[t];
      if (greedy) {
        if (x != P.i) break;
        continue;
      }
      if (x >= vocab) break;
      const double px = vd_exp(load_as_f32<LT>(target, ((size_t)s * (n_draft + 1) + t) * vocab + x), P.m, inv_t) / P.z;
      double qx = 1.0;
      if (draft) {
        const VdPart& Q = s_row[n_draft + 1 + t];
        qx = vd_exp(load_as_f32<LT>(draft, ((size_t)s * n_draft + t) * vocab + x), Q.m, inv_t) / Q.z;
      }
      if (!((double)u[t] * qx < px)) break;
    }
    s_took = t;
    s_state = state;
  }
  __syncthreads();
  const uint32_t took = s_took;
  const VdPart P = s_row[took];
  const size_t pb = ((size_t)s * (n_draft + 1) + took) * vocab;
  uint32_t pick = 0xffffffffu;
  if (s_state == 1) {
    pick = P.i;
  } else if (s_state == 0) {
    const bool rejected = took < n;
    const VdPart Q = rejected && draft ? s_row[n_draft + 1 + took] : VdPart{1.0, 0.0f, 0};
    const size_t qb = ((size_t)s * n_draft + took) * vocab;
    const uint32_t x = rejected ? tok[took] : 0xffffffffu;
    auto mass = [&](uint32_t v, bool whole) {
      const double p = vd_exp(load_as_f32<LT>(target, pb + v), P.m, inv_t) / P.z;
      if (!rejected || whole) return p;
      const double q = draft ? vd_exp(load_as_f32<LT>(draft, qb + v), Q.m, inv_t) / Q.z : (v == x ? 1.0 : 0.0);
      return fmax(p - q, 0.0);
    };
    const uint32_t per = (vocab + VP_NT - 1) / VP_NT, a = tid * per, b = min(vocab, a + per);
    bool whole = false;
    double total = 0.0;
    for (int round = 0; round < 2; ++round) {  // (nothing left of p - q: p itself)
      double z = 0.0;
      for (uint32_t v = a; v < b; ++v) z += mass(v, whole);
      s_sum[tid] = z;
      __syncthreads();
      total = 0.0;
      if (tid == 0) {
        for (int i = 0; i < VP_NT; ++i) {
          const double y = s_sum[i];
          s_sum[i] = total;
          total += y;
        }
        s_sum[0] = total;  // (the first share begins at 0)
        s_pick = 0xffffffffu;
      }
      __syncthreads();
      total = s_sum[0];
      if (total > 0.0) break;
      __syncthreads();
      whole = true;
    }
    const double want = (double)u[n_draft] * total;
    double c = tid == 0 ? 0.0 : s_sum[tid];
    uint32_t last = 0xffffffffu;
    for (uint32_t v = a; v < b; ++v) {
      const double y = mass(v, whole);
      c += y;
      if (y > 0.0) last = v;
      if (c > want) {
        atomicMin(&s_pick, v);
        break;
      }
    }
    __syncthreads();
    pick = s_pick;
    __syncthreads();
    if (pick == 0xffffffffu) {  // u S rounded up to S: the last token with any mass
      if (tid == 0) s_pick = 0;
      __syncthreads();
      if (last != 0xffffffffu) atomicMax(&s_pick, last);
      __syncthreads();
      pick = s_pick;
    }
  }
  if (tid == 0) accepted[s] = took;
  if (tid <= n_draft) {
    const uint32_t x = tid < took ? tok[tid] : tid == took ? pick : 0xffffffffu;
    out[(size_t)s * (n_draft + 1) + tid] = x;
    if (logprobs) {
      float lp = 0.0f;
      if (tid <= took) {
        const VdPart& R = s_row[tid];
        lp = x < vocab ? (float)(((double)load_as_f32<LT>(target, ((size_t)s * (n_draft + 1) + tid) * vocab + x) -
                                  (double)R.m) * inv_t - log(R.z))
                       : NAN;
      }
      logprobs[(size_t)s * (n_draft + 1) + tid] = lp;
    }
  }
}

}  // namespace cm
