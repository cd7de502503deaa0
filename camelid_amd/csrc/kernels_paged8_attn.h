// kernels_paged8_attn.h -- attention of a sequence's newest tokens over an 8-bit cache in pages.
//
//   s_p = scale 2^ke(p) (q . k_p) for p <= the row's position;  w = softmax(s);  o = sum_p w_p 2^ve(p) v_p
#pragma once
#include "kernels_paged8.h"

namespace cm {

struct P8Args {
  Paged8 c;
  const void* q;
  const uint32_t* new_lens;
  void* out;
  float scale;
  uint32_t q_stride, out_stride, n_new, n_heads, group;
};

// One wave per (row, head): a lane per position for the scores of 64 positions, a lane per dim for the sum.
template <int HD, int KT, int QT>
__global__ __launch_bounds__(64) void k_p8_rows(P8Args a) {
  __shared__ float s_q[HD], s_w[64];
  const Paged& g = a.c.g;
  const uint32_t lane = threadIdx.x, head = blockIdx.x % a.n_heads, row = blockIdx.x / a.n_heads;
  const uint32_t s = row / a.n_new, t = row - s * a.n_new, h = head / a.group;
  uint32_t first, len;
  if (!paged_rows(g, a.new_lens, a.n_new, s, &first, &len)) return;
  if (first + t >= len) return;
  const uint32_t seen = first + t + 1, mask = (1u << g.shift) - 1u;
  for (uint32_t d = lane; d < HD; d += 64) s_q[d] = load_as_f32<QT>(a.q, (size_t)row * a.q_stride + (size_t)head * HD + d);
  __syncthreads();
  const uint32_t* tab = g.table + (size_t)s * g.stride;
  float m = -INFINITY, l = 0.0f, o[HD / 64] = {};
  for (uint32_t p0 = 0; p0 < seen; p0 += 64) {
    const uint32_t p = p0 + lane, pg = p < seen ? tab[p >> g.shift] : 0u;
    const bool here = p < seen && pg < g.n_pages;
    if (p < seen && !here) paged_flag(g, PG_BAD_PAGE);
    float x = -INFINITY;
    if (here) {
      const uint8_t* k = a.c.kc + p8_base(g, pg, h);
      float dot = 0.0f;
      for (uint32_t d = 0; d < HD; d += 4) {
        float y[4];
        p8_unpack4<KT>(*reinterpret_cast<const uint32_t*>(k + p8_k(g, p & mask, d)), y);
        for (int i = 0; i < 4; ++i) dot += y[i] * s_q[d + i];
      }
      x = dot * p8_scale(a.c.ke[p8_exp(g, pg, h, p & mask)]) * a.scale;
    }
    float top = x;
    for (int i = 32; i; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));
    const float now = fmaxf(m, top), ref = now == -INFINITY ? 0.0f : now;
    const float keep = expf(m - ref), w = here ? expf(x - ref) : 0.0f;
    m = now;
    float sum = w;
    for (int i = 32; i; i >>= 1) sum += __shfl_xor(sum, i);
    l = l * keep + sum;
    __syncthreads();
    s_w[lane] = w;
    __syncthreads();
    for (int i = 0; i < HD / 64; ++i) o[i] *= keep;
    for (uint32_t j = 0; j < 64 && p0 + j < seen; ++j) {
      const uint32_t at = p0 + j, page = tab[at >> g.shift];
      if (page >= g.n_pages) continue;
      const float e = p8_scale(a.c.ve[p8_exp(g, page, h, at & mask)]);
      const uint8_t* v = a.c.vc + p8_base(g, page, h);
      for (int i = 0; i < HD / 64; ++i) {
        float y[4];
        p8_unpack4<KT>(v[p8_v(g, at & mask, lane + 64 * i)], y);
        o[i] += s_w[j] * (y[0] * e);
      }
    }
  }
  for (int i = 0; i < HD / 64; ++i)
    store_from_f32<QT>(a.out, (size_t)row * a.out_stride + (size_t)head * HD + lane + 64 * i,
                       m == -INFINITY ? 0.0f : o[i] / l);
}

}  // namespace cm
