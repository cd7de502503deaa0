// kernels_paged.h -- a key/value cache in pages, shared by many sequences: RoPE + store of new
// tokens, their attention, and eviction by accumulated attention weight.
//
// Pages: n_pages of page_size positions (a power of two >= 8), 16-bit elements.  K of one page is
// [n_kv][hd / 8][page_size][8], V is [n_kv][page_size / 8][hd][8]: the granules of 16 bytes of the
// engine's own cache (8 dims of one position for K, 8 positions of one dim for V), a page in the
// place of the whole position range.  Position p of sequence s lies at offset p % page_size of
// page table[s][p / page_size].
//
// Sequence s holds lens[s] positions; the last new_lens[s] of them are this call's new tokens, rows
// s * n_new + t of the activations (t < new_lens[s]), at positions lens[s] - new_lens[s] + t.
#pragma once
#include <hip/hip_runtime.h>
#include "device_math.h"

namespace cm {

enum { TY_F32 = 0, TY_F16 = 1, TY_BF16 = 2 };  // CAMELID_F32, CAMELID_F16, CAMELID_BF16

// Bits of the caller's status word (CAMELID_PAGED_BAD_PAGE, CAMELID_PAGED_BAD_LENGTH).
enum { PG_BAD_PAGE = 1, PG_BAD_LENGTH = 2 };

struct Paged {
  const uint32_t* table;  // [n_seqs][stride]
  const uint32_t* lens;   // [n_seqs]
  uint32_t* status;       // may be null
  uint32_t stride;        // pages of one sequence's table row
  uint32_t n_pages;
  uint32_t shift;         // log2(page_size)
  uint32_t n_kv, hd, n_seqs;
};

__device__ __forceinline__ void paged_flag(const Paged& g, uint32_t bit) {
  if (g.status) atomicOr(g.status, bit);
}

// The new tokens of sequence s: positions [first, len).  False (and the status word) where the
// lengths do not fit the table or each other.
__device__ __forceinline__ bool paged_rows(const Paged& g, const uint32_t* new_lens, uint32_t n_new, uint32_t s,
                                           uint32_t* first, uint32_t* len) {
  const uint32_t L = g.lens[s], m = new_lens ? new_lens[s] : n_new;
  *len = L;
  *first = L - m;
  if ((uint64_t)L <= ((uint64_t)g.stride << g.shift) && m <= n_new && m <= L) return true;
  paged_flag(g, PG_BAD_LENGTH);
  return false;
}

// Element offset of (page, kv head) in the K or V buffer.
__device__ __forceinline__ size_t paged_base(const Paged& g, uint32_t page, uint32_t h) {
  return ((size_t)page * g.n_kv + h) * ((size_t)g.hd << g.shift);
}
// Offset inside it of dim d of the page's position o.
__device__ __forceinline__ uint32_t paged_k(const Paged& g, uint32_t o, uint32_t d) {
  return ((((d >> 3) << g.shift) + o) << 3) + (d & 7u);
}
__device__ __forceinline__ uint32_t paged_v(const Paged& g, uint32_t o, uint32_t d) {
  return (((o >> 3) * g.hd + d) << 3) + (o & 7u);
}

// f32 -> 16 bits, round to nearest even; NaN becomes the canonical quiet NaN.
template <int T>
__device__ __forceinline__ uint16_t to_bits16(float v) {
  if (T == TY_F16) {
    const _Float16 h = (_Float16)v;
    return v != v ? (uint16_t)0x7e00u : __builtin_bit_cast(uint16_t, h);
  }
  const __bf16 b = (__bf16)v;
  return v != v ? (uint16_t)0x7fc0u : __builtin_bit_cast(uint16_t, b);
}
template <int T>
__device__ __forceinline__ float from_bits16(uint16_t b) {
  if (T == TY_F16) return (float)__builtin_bit_cast(_Float16, b);
  return u2f((uint32_t)b << 16);
}
template <int T>
__device__ __forceinline__ float load_as_f32(const void* p, size_t i) {
  if (T == TY_F32) return static_cast<const float*>(p)[i];
  return from_bits16<T>(static_cast<const uint16_t*>(p)[i]);
}
template <int T>
__device__ __forceinline__ void store_from_f32(void* p, size_t i, float v) {
  if (T == TY_F32)
    static_cast<float*>(p)[i] = v;
  else
    static_cast<uint16_t*>(p)[i] = to_bits16<T>(v);
}

// ---------------------------------------------------------------------------
// Per-head RMSNorm (optional) + RoPE of the new tokens' q and k rows, K and V into the pages.
//   norm: x_d = (x_d * (1 / sqrt(sum x^2 / hd + eps))) * w_d, the sum over d in order
//   pair: (a, b) -> (a c - b s, a s + b c), each product and sum rounded in f32
// the arithmetic of k_rope_kv, so an f16 cache holds the same bits.  One wave per (row, head), for
// rope_dim < head_dim: pairs fall anywhere in the head.
template <int QT, int KT>
__global__ __launch_bounds__(64) void k_paged_rope_kv(Paged g, const float* __restrict__ qkv, uint32_t n_new,
                                                      const uint32_t* __restrict__ new_lens, uint32_t n_heads,
                                                      uint32_t rope_dim, uint32_t split_half,
                                                      const float* __restrict__ cosv, const float* __restrict__ sinv,
                                                      const float* __restrict__ q_norm,
                                                      const float* __restrict__ k_norm, float eps,
                                                      void* __restrict__ q_out, uint16_t* __restrict__ kc,
                                                      uint16_t* __restrict__ vc) {
  __shared__ float buf[256];
  __shared__ float s_scale;
  const uint32_t per = n_heads + g.n_kv;
  const size_t row = blockIdx.x / per;
  const uint32_t h = blockIdx.x % per;
  const uint32_t s = (uint32_t)(row / n_new), t = (uint32_t)(row % n_new);
  uint32_t first, len;
  if (!paged_rows(g, new_lens, n_new, s, &first, &len)) return;
  const uint32_t pos = first + t;
  if (pos >= len) return;
  const bool isq = h < n_heads;
  const size_t width = (size_t)(n_heads + 2 * g.n_kv) * g.hd;
  const float* src = qkv + row * width + (size_t)h * g.hd;
  for (uint32_t d = threadIdx.x; d < g.hd; d += 64) buf[d] = src[d];
  const float* nw = isq ? q_norm : k_norm;
  __syncthreads();
  if (nw) {
    if (threadIdx.x == 0) {
      float acc = 0.0f;
      for (uint32_t d = 0; d < g.hd; ++d) acc = acc + buf[d] * buf[d];
      s_scale = 1.0f / sqrtf(acc / (float)g.hd + eps);
    }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < g.hd; d += 64) buf[d] = (buf[d] * s_scale) * nw[d];
    __syncthreads();
  }
  const uint32_t half = rope_dim >> 1;
  for (uint32_t p = threadIdx.x; p < half; p += 64) {
    const uint32_t d0 = split_half ? p : 2 * p, d1 = split_half ? p + half : 2 * p + 1;
    const float c = cosv[row * half + p], sn = sinv[row * half + p];
    const float x0 = buf[d0], x1 = buf[d1];
    buf[d0] = (x0 * c) - (x1 * sn);
    buf[d1] = (x0 * sn) + (x1 * c);
  }
  __syncthreads();
  if (isq) {
    for (uint32_t d = threadIdx.x; d < g.hd; d += 64)
      store_from_f32<QT>(q_out, (row * n_heads + h) * g.hd + d, buf[d]);
    return;
  }
  const uint32_t page = g.table[(size_t)s * g.stride + (pos >> g.shift)];
  if (page >= g.n_pages) {
    if (threadIdx.x == 0) paged_flag(g, PG_BAD_PAGE);
    return;
  }
  const size_t base = paged_base(g, page, h - n_heads);
  const uint32_t o = pos & ((1u << g.shift) - 1u);
  const float* vsrc = src + (size_t)g.n_kv * g.hd;
  for (uint32_t d = threadIdx.x; d < g.hd; d += 64) {
    kc[base + paged_k(g, o, d)] = to_bits16<KT>(buf[d]);
    vc[base + paged_v(g, o, d)] = to_bits16<KT>(vsrc[d]);
  }
}

// The same for rope_dim = head_dim, one workgroup per (granule of 8 positions, role): q heads, K
// heads or V heads, so that the up to 8 new tokens of a granule are stored together: V as whole granules
// (a granule holds 8 positions of a dim), K as 8 granules side by side.
//   q, K: HD / 16 lanes per (token, head), each 8 dims of either half, which hold the pairs of both
//         pairings; the norm's sum in order by one lane per (token, head) from LDS.
//   V:    a lane per dim.
// Bound: HBM.  207 MB (4 prompts of up to 2047 tokens, 24 + 8 + 8 heads of 128): 37 us, 5.6 TB/s (84 us
// with one wave per (token, head) and 2-byte stores); launch and latency for decode steps: 3 us for one
// token of 32 + 4 + 4 heads of 64, 6 us for 24 sequences of up to 5 tokens of 32 + 8 + 8 heads of 128.
constexpr uint32_t RK_NT = 256;
constexpr uint32_t rk_heads(uint32_t hd) { return RK_NT / (hd / 16) / 8; }  // q or K heads of a workgroup
constexpr uint32_t rk_v_heads(uint32_t hd) { return RK_NT / hd; }
__host__ __device__ constexpr uint32_t rk_roles(uint32_t hd, uint32_t n_heads, uint32_t n_kv) {
  return (n_heads + rk_heads(hd) - 1) / rk_heads(hd) + (n_kv + rk_heads(hd) - 1) / rk_heads(hd) +
         (n_kv + rk_v_heads(hd) - 1) / rk_v_heads(hd);
}
// Granules that n_new consecutive positions can reach into.
constexpr uint32_t rk_granules(uint32_t n_new) { return (n_new + 6) / 8 + 1; }

typedef float f32x4v __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ void rk_load8(const float* p, float (&x)[8]) {
  const f32x4v a = *reinterpret_cast<const f32x4v*>(p), b = *reinterpret_cast<const f32x4v*>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = a[i];
    x[4 + i] = b[i];
  }
}
typedef uint32_t rk_u32x4 __attribute__((ext_vector_type(4)));
template <int T>
__device__ __forceinline__ rk_u32x4 rk_pack8(const float (&x)[8]) {
  rk_u32x4 u;
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = to_bits16<T>(x[2 * i]) | (uint32_t)to_bits16<T>(x[2 * i + 1]) << 16;
  return u;
}

template <int HD, int QT, int KT>
__global__ __launch_bounds__(RK_NT) void k_paged_rope_kv8(Paged g, const float* __restrict__ qkv, uint32_t n_new,
                                                          const uint32_t* __restrict__ new_lens, uint32_t n_heads,
                                                          uint32_t split_half, const float* __restrict__ cosv,
                                                          const float* __restrict__ sinv,
                                                          const float* __restrict__ q_norm,
                                                          const float* __restrict__ k_norm, float eps,
                                                          void* __restrict__ q_out, uint16_t* __restrict__ kc,
                                                          uint16_t* __restrict__ vc, uint32_t roles,
                                                          uint32_t granules) {
  constexpr uint32_t LPR = HD / 16, PAIRS = RK_NT / LPR, HEADS = rk_heads(HD), V_HEADS = rk_v_heads(HD), HALF = HD / 2;
  __shared__ float s_x[PAIRS][HD + 4];
  __shared__ float s_scale[PAIRS];
  const uint32_t tid = threadIdx.x, role = blockIdx.x % roles, sg = blockIdx.x / roles;
  const uint32_t s = sg / granules, gi = sg - s * granules;
  uint32_t first, len;
  if (!paged_rows(g, new_lens, n_new, s, &first, &len)) return;
  const uint32_t p0 = (first & ~7u) + 8 * gi;  // the granule's first position
  if (p0 >= len) return;
  const size_t width = (size_t)(n_heads + 2 * g.n_kv) * HD;
  const uint32_t q_roles = (n_heads + HEADS - 1) / HEADS, k_roles = (g.n_kv + HEADS - 1) / HEADS;
  const uint32_t mask = (1u << g.shift) - 1u;
  const bool isq = role < q_roles;
  uint32_t page = 0;
  if (!isq) {
    page = g.table[(size_t)s * g.stride + (p0 >> g.shift)];
    if (page >= g.n_pages) {
      if (tid == 0) paged_flag(g, PG_BAD_PAGE);
      return;
    }
  }
  if (role >= q_roles + k_roles) {
    const uint32_t h = (role - q_roles - k_roles) * V_HEADS + tid / HD, d = tid % HD;
    if (h >= g.n_kv) return;
    const float* src = qkv + ((size_t)s * n_new) * width + (size_t)(n_heads + g.n_kv + h) * HD + d;
    float x[8];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const uint32_t p = p0 + i;
      x[i] = p >= first && p < len ? src[(size_t)(p - first) * width] : 0.0f;
    }
    uint16_t* dst = vc + paged_base(g, page, h) + paged_v(g, p0 & mask, d);
    const rk_u32x4 u = rk_pack8<KT>(x);
    if (p0 >= first && p0 + 8 <= len) {
      *reinterpret_cast<rk_u32x4*>(dst) = u;
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i)
        if (p0 + i >= first && p0 + i < len) dst[i] = (uint16_t)(u[i / 2] >> (16 * (i & 1)));
    }
    return;
  }
  const uint32_t j = tid % LPR, pair = tid / LPR, i8 = pair % 8;
  const uint32_t h = (isq ? role : role - q_roles) * HEADS + pair / 8;
  const uint32_t p = p0 + i8;
  const bool live = p >= first && p < len && h < (isq ? n_heads : g.n_kv);
  const size_t row = (size_t)s * n_new + (p - first);
  float a[8], b[8];  // dims 8 j .. and HALF + 8 j ..
  float ca[8], sa[8];
  if (live) {
    const float* src = qkv + row * width + (size_t)(isq ? h : n_heads + h) * HD;
    rk_load8(src + 8 * j, a);
    rk_load8(src + HALF + 8 * j, b);
    const float *c = cosv + row * HALF, *sn = sinv + row * HALF;
    if (split_half) {  // pairs 8 j .. 8 j + 7: (a, b)
      rk_load8(c + 8 * j, ca);
      rk_load8(sn + 8 * j, sa);
    } else {  // pairs 4 j .. inside a, HALF / 2 + 4 j .. inside b
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const f32x4v x = *reinterpret_cast<const f32x4v*>(c + k * (HALF / 2) + 4 * j);
        const f32x4v y = *reinterpret_cast<const f32x4v*>(sn + k * (HALF / 2) + 4 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ca[4 * k + i] = x[i];
          sa[4 * k + i] = y[i];
        }
      }
    }
  }
  const float* nw = isq ? q_norm : k_norm;
  if (nw) {
    if (live) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s_x[pair][8 * j + i] = a[i];
        s_x[pair][HALF + 8 * j + i] = b[i];
      }
    }
    __syncthreads();
    if (tid < PAIRS) {  // (padding rows sum what lies there)
      float acc = 0.0f;
#pragma unroll 8
      for (uint32_t d = 0; d < HD; ++d) {
        const float x = s_x[tid][d];
        acc = acc + x * x;
      }
      s_scale[tid] = 1.0f / sqrtf(acc / (float)HD + eps);
    }
    __syncthreads();
    if (live) {
      const float sc = s_scale[pair];
      float wa[8], wb[8];
      rk_load8(nw + 8 * j, wa);
      rk_load8(nw + HALF + 8 * j, wb);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a[i] = (a[i] * sc) * wa[i];
        b[i] = (b[i] * sc) * wb[i];
      }
    }
  }
  if (!live) return;
  if (split_half) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x0 = a[i], x1 = b[i];
      a[i] = (x0 * ca[i]) - (x1 * sa[i]);
      b[i] = (x0 * sa[i]) + (x1 * ca[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x0 = a[2 * i], x1 = a[2 * i + 1], y0 = b[2 * i], y1 = b[2 * i + 1];
      a[2 * i] = (x0 * ca[i]) - (x1 * sa[i]);
      a[2 * i + 1] = (x0 * sa[i]) + (x1 * ca[i]);
      b[2 * i] = (y0 * ca[4 + i]) - (y1 * sa[4 + i]);
      b[2 * i + 1] = (y0 * sa[4 + i]) + (y1 * ca[4 + i]);
    }
  }
  if (!isq) {
    uint16_t* dst = kc + paged_base(g, page, h);
    *reinterpret_cast<rk_u32x4*>(dst + paged_k(g, p & mask, 8 * j)) = rk_pack8<KT>(a);
    *reinterpret_cast<rk_u32x4*>(dst + paged_k(g, p & mask, HALF + 8 * j)) = rk_pack8<KT>(b);
    return;
  }
  const size_t at = (row * n_heads + h) * HD + 8 * j;
  if constexpr (QT == TY_F32) {
    f32x4v* dst = reinterpret_cast<f32x4v*>(static_cast<float*>(q_out) + at);
    dst[0] = f32x4v{a[0], a[1], a[2], a[3]};
    dst[1] = f32x4v{a[4], a[5], a[6], a[7]};
    dst[HALF / 4] = f32x4v{b[0], b[1], b[2], b[3]};
    dst[HALF / 4 + 1] = f32x4v{b[4], b[5], b[6], b[7]};
  } else {
    uint16_t* dst = static_cast<uint16_t*>(q_out) + at;
    *reinterpret_cast<rk_u32x4*>(dst) = rk_pack8<QT>(a);
    *reinterpret_cast<rk_u32x4*>(dst + HALF) = rk_pack8<QT>(b);
  }
}

// ---------------------------------------------------------------------------
// Eviction.  A sequence of more than `keep` positions keeps, for each KV head, its last `recent`
// positions and the keep - recent of highest accumulated weight among the others (equal weights:
// the lower position; a NaN counts as the lowest weight), in their order, moved to positions
// [0, keep).  Two launches: the selection, then the move.

// Bits that order as the weights do (-0 as +0, NaN lowest).
__device__ __forceinline__ uint32_t evict_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = f2u(w + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Inclusive prefix sum over the wave by data-parallel moves.
__device__ __forceinline__ uint32_t ev_wave_scan(uint32_t x) {
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false);  // 1, 2, 4, 8 lanes below
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false);  // the row below's end
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false);  // the lower half's end
  return x;
}

// What the selection leaves for the move, for each (sequence, KV head).
struct EvictPlan {
  uint32_t* slot;     // [keep] the slots (page * page_size + offset) of the kept positions, in order
  uint32_t* from;     // [keep] where row j comes from: 8 * (index of its granule of 8 positions) + position % 8
  uint32_t* granule;  // [keep] the distinct granules in order: slot / 8
  uint32_t* old_lens; // [n_seqs] the length before where rows have to move, else 0
  uint32_t* new_lens; // [n_seqs]
};

// One workgroup per (sequence, KV head): the plan, `kept` (the positions themselves), the weights
// compacted.
//
// The smallest kept weight by its digits from the top: for each a histogram in two copies and a suffix sum of
// its counts.  A thread holds K weights in registers, runs of V at a time, so up to K * NT positions are read
// once; longer rows go through the same code in pieces that are read again.  Then prefix sums of two counts
// in a word (weights above the smallest, weights equal to it) give every kept position its place.
// Rows of up to 512 positions: 256 threads, four digits of 8 bits (95 x 8 rows of up to 78 weights 15.3 ->
// 7.8 us against 1024 threads).  Longer ones: 1024 threads, digits of 11, 11 and 10 bits (of 8 bits the first
// takes 5.2 us for 16383 weights, which crowd in few counters).
// Bound: latency (barriers between the digits): 16 x 8 rows of 1088 weights 7.6 us (43 with a histogram
// searched by one thread), 4 x 8 rows of up to 16383 weights 16.6 us.
template <int K, uint32_t NT>
__global__ __launch_bounds__(NT) void k_evict_select(Paged g, float* __restrict__ weights, uint32_t keep,
                                                        uint32_t recent, EvictPlan plan, uint32_t* __restrict__ kept) {
  constexpr uint32_t COPIES = 2, BITS = NT == 1024 ? 11 : 8, BINS = 1u << BITS, PIECE = NT * K;
  constexpr uint32_t PER = BINS / NT;          // digits of a thread
  constexpr int V = K < 4 ? K : 4, N = K / V;  // N runs of V positions, NT * V apart
  typedef float vec __attribute__((ext_vector_type(V), aligned(4)));
  __shared__ uint32_t hist[COPIES][BINS];
  __shared__ uint32_t wave_sums[N][NT / 64], wave_touched[N][NT / 64];
  __shared__ uint32_t s_digit, s_rank, s_bad;
  const uint32_t s = blockIdx.x / g.n_kv, h = blockIdx.x - s * g.n_kv, tid = threadIdx.x, lane = tid & 63u;
  const uint32_t L = g.lens[s], cap = g.stride << g.shift, mask = (1u << g.shift) - 1u;
  const uint32_t* tab = g.table + (size_t)s * g.stride;
  float* w = weights + (size_t)blockIdx.x * cap;
  const bool too_long = (uint64_t)L > ((uint64_t)g.stride << g.shift);
  // the first piece's weights, on their way while the pages are looked through
  float x[N][V];
  const auto at = [&](uint32_t p0, int i, int e) { return p0 + (i * NT + tid) * V + e; };
  const auto read = [&](uint32_t p0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (at(p0, i, V) <= L) {
        const vec y = *reinterpret_cast<const vec*>(w + at(p0, i, 0));
#pragma unroll
        for (int e = 0; e < V; ++e) x[i][e] = y[e];
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) x[i][e] = at(p0, i, e) < L ? w[at(p0, i, e)] : 0.0f;
      }
    }
  };
  if (tid == 0) s_bad = 0;
  __syncthreads();
  if (too_long) {
    if (tid == 0) paged_flag(g, PG_BAD_LENGTH);
  } else {
    if (L > keep) read(0);
    bool bad = false;
    for (uint32_t i = tid; i < (L + mask) >> g.shift; i += NT) bad |= tab[i] >= g.n_pages;
    if (bad) s_bad = 1;
  }
  __syncthreads();
  if (s_bad && tid == 0) paged_flag(g, PG_BAD_PAGE);
  const bool moves = !too_long && !s_bad && L > keep;
  if (h == 0 && tid == 0) {
    plan.old_lens[s] = moves ? L : 0u;
    plan.new_lens[s] = moves ? keep : L;
  }
  uint32_t* kp = kept ? kept + (size_t)blockIdx.x * keep : nullptr;
  if (!moves) {
    if (kp && !too_long)
      for (uint32_t j = tid; j < min(L, keep); j += NT) kp[j] = j;
    return;
  }
  const size_t row0 = (size_t)blockIdx.x * keep;
  const uint32_t cut = L - recent;
  const bool one = L <= PIECE;  // the weights stay in registers
  uint32_t key[N][V];
  const auto make_keys = [&] {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) key[i][e] = evict_key(x[i][e]);
  };
  make_keys();
  uint32_t rank = keep - recent;  // positions still to be found among the keys equal in the digits so far
  const bool any = rank != 0;
  uint32_t prefix = 0;
  for (int top = 32; top > 0 && any;) {  // the digit in bits b .. top - 1, those above are in `prefix`
    const int b = max(0, top - (int)BITS);
    const uint32_t bins = 1u << (top - b);
    for (uint32_t i = tid; i < COPIES * BINS; i += NT) hist[0][i] = 0;
    __syncthreads();
    for (uint32_t p0 = 0; p0 < cut; p0 += PIECE) {
      if (!one) {
        read(p0);
        make_keys();
      }
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const uint32_t k = key[i][e];
          if (at(p0, i, e) < cut && (top == 32 || k >> (top & 31) == prefix >> (top & 31)))
            atomicAdd(&hist[(tid >> 6) % COPIES][(k >> b) & (bins - 1)], 1u);
        }
    }
    __syncthreads();
    // thread t: digit BINS - 1 - PER t and, for PER = 2, the one below it
    const uint32_t hi = BINS - 1 - PER * tid, c0 = hist[0][hi] + hist[1][hi];
    const uint32_t c1 = PER == 2 ? hist[0][hi - 1] + hist[1][hi - 1] : 0u;
    const uint32_t incl = ev_wave_scan(c0 + c1);
    if (lane == 63) wave_sums[0][tid >> 6] = incl;
    __syncthreads();
    uint32_t above = incl - c0 - c1;
    for (uint32_t v = 0; v < NT / 64; ++v) above += v < tid >> 6 ? wave_sums[0][v] : 0u;
    if (above < rank && above + c0 + c1 >= rank) {
      const bool first = above + c0 >= rank;
      s_digit = first ? hi : hi - 1;
      s_rank = rank - above - (first ? 0u : c0);
    }
    __syncthreads();
    prefix |= s_digit << b;
    rank = s_rank;
    top = b;
  }
  // kept: every key above `prefix`, the first `rank` keys equal to it, and the recent positions
  uint32_t eq0 = 0, gt0 = 0, touched0 = 0;  // of the pieces before
  for (uint32_t p0 = 0; p0 < L; p0 += PIECE) {
    if (!one) {
      read(p0);
      make_keys();
    }
    uint32_t gts[N], eqs[N], before[N], page[N];  // before: counts in a word: gt, eq << 16 (at most 4096 each)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      page[i] = at(p0, i, 0) < L ? tab[at(p0, i, 0) >> g.shift] : 0u;  // (a run lies in one page)
      gts[i] = eqs[i] = 0;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const uint32_t p = at(p0, i, e), k = key[i][e];
        gts[i] |= (uint32_t)(p < L && (p >= cut || (any && k > prefix))) << e;
        eqs[i] |= (uint32_t)(p < cut && any && k == prefix) << e;
      }
      const uint32_t count = __popc(gts[i]) + (__popc(eqs[i]) << 16), incl = ev_wave_scan(count);
      before[i] = incl - count;
      if (lane == 63) wave_sums[i][tid >> 6] = incl;
    }
    __syncthreads();  // (every weight of the piece has been read, too)
    uint32_t first[N], takes[N], seen[N];  // first: the run's first output position
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uint32_t all = 0;
      for (uint32_t v = 0; v < NT / 64; ++v) {
        const uint32_t y = wave_sums[i][v];
        if (v < tid >> 6) before[i] += y;
        all += y;
      }
      const uint32_t gt = gt0 + (before[i] & 0xffffu);
      uint32_t eq = eq0 + (before[i] >> 16);
      first[i] = gt + min(eq, rank);
      takes[i] = gts[i];
#pragma unroll
      for (int e = 0; e < V; ++e)
        if ((eqs[i] >> e) & 1u) {
          if (eq < rank) takes[i] |= 1u << e;
          ++eq;
        }
      gt0 += all & 0xffffu;
      eq0 += all >> 16;
      // a granule is 8 / V runs: its first lane counts it where any of them is taken from
      uint32_t some = takes[i];
      some |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)some, 0xb1, 0xf, 0xf, false);
      if (V < 4) some |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)some, 0x4e, 0xf, 0xf, false);
      const uint32_t incl = ev_wave_scan(some && (lane & (8 / V - 1)) == 0 ? 1u : 0u);
      seen[i] = incl;
      if (lane == 63) wave_touched[i][tid >> 6] = incl;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uint32_t t = touched0 + seen[i] - 1;
      for (uint32_t v = 0; v < NT / 64; ++v) {
        const uint32_t y = wave_touched[i][v];
        if (v < tid >> 6) t += y;
        touched0 += y;
      }
      uint32_t j = first[i];
      const uint32_t slot0 = (page[i] << g.shift) + (at(p0, i, 0) & mask);
      if (takes[i]) plan.granule[row0 + t] = slot0 >> 3;  // (the granule's runs write the same)
#pragma unroll
      for (int e = 0; e < V; ++e)
        if ((takes[i] >> e) & 1u) {  // j <= p: no weight still to be read
          plan.slot[row0 + j] = slot0 + e;
          plan.from[row0 + j] = 8 * t + ((slot0 + e) & 7u);
          w[j] = x[i][e];
          if (kp) kp[j] = at(p0, i, e);
          ++j;
        }
    }
    __syncthreads();
  }
}

// The move, in place: output positions in chunks, a chunk's sources read before any of it is
// written.  A source is never below its output position, so no later chunk misses a row.  A workgroup takes
// as many dims as leave all kept rows one chunk (ks, vs; 95 x 8 x 22 of up to 78 rows: 25 -> 8.4 us against 8
// dims of K and 16 of V), and where there are few workgroups larger chunks (F; 8 x 14511 of 20144 rows of
// one of two sequences: 40 -> 36 us).  Bound: HBM: 16 x 8 x 1024 of 1088 rows of 128 dims 26.6 us, 83 MB of
// lines read and 67 written, 5.6 TB/s; 4 x 8 x 2048 of up to 16383 rows 19 us, where rows far apart share their 128-byte lines with rows that
// are left behind (68 MB of lines read for the 34 MB that are written).
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// K: one workgroup per (sequence, KV head, 8 << ks dims), whole granules, chunks of 2048 F >> ks rows in
// registers.
constexpr uint32_t EM_NT = 512, EM_K_LOG2 = 11;
template <uint32_t F>
__device__ __forceinline__ void evict_move_k(const Paged& g, uint16_t* __restrict__ kc, uint32_t keep,
                                             const EvictPlan& plan, uint32_t sh, uint32_t sl, uint32_t ks) {
  constexpr uint32_t R = (F << EM_K_LOG2) / EM_NT;
  const uint32_t tid = threadIdx.x, s = sh / g.n_kv, h = sh - s * g.n_kv;
  const uint32_t* tab = g.table + (size_t)s * g.stride;
  const uint32_t* sp = plan.slot + (size_t)sh * keep;
  const uint32_t mask = (1u << g.shift) - 1u, bits = EM_K_LOG2 + __builtin_ctz(F) - ks, rows = 1u << bits;
  for (uint32_t j0 = 0; j0 < keep; j0 += rows) {
    u32x4 x[R];
    uint32_t to[R], slot[R];
#pragma unroll
    for (uint32_t r = 0; r < R; ++r) {
      const uint32_t j = min(j0 + ((r * EM_NT + tid) & (rows - 1)), keep - 1);
      slot[r] = sp[j];
      to[r] = (tab[j >> g.shift] << g.shift) + (j & mask);
    }
    const auto place = [&](uint32_t at, uint32_t r) {
      return kc + paged_base(g, at >> g.shift, h) + paged_k(g, at & mask, 8 * ((sl << ks) + ((r * EM_NT + tid) >> bits)));
    };
#pragma unroll
    for (uint32_t r = 0; r < R; ++r)
      if (j0 + ((r * EM_NT + tid) & (rows - 1)) < keep) x[r] = *reinterpret_cast<const u32x4*>(place(slot[r], r));
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < R; ++r)
      if (j0 + ((r * EM_NT + tid) & (rows - 1)) < keep && slot[r] != to[r])
        *reinterpret_cast<u32x4*>(place(to[r], r)) = x[r];
  }
}

// V: one workgroup per (sequence, KV head, 8 << vs dims).  A granule holds 8 positions, an output granule
// gathers from up to 8 of them, so a chunk is as many rows as 256 F >> vs distinct granules feed; these go to
// LDS whole (2-byte loads from memory, 16 bytes apart between lanes, took the L1 47 accesses each: 24 us of
// the 37 us that the move of 16x1088 -> 1024 rows took) and the output granules are put together from there.
constexpr uint32_t EM_G = 256;
constexpr uint32_t em_lds(uint32_t f) { return f * EM_G * 8 * 16; }
template <uint32_t F>
__device__ __forceinline__ void evict_move_v(const Paged& g, uint16_t* __restrict__ vc, uint32_t keep,
                                             const EvictPlan& plan, uint32_t sh, uint32_t sl, uint32_t vs, u32x4* s_g,
                                             uint32_t* s_end) {
  const uint32_t tid = threadIdx.x, s = sh / g.n_kv, h = sh - s * g.n_kv;
  const uint32_t* tab = g.table + (size_t)s * g.stride;
  const uint32_t* fp = plan.from + (size_t)sh * keep;
  const uint32_t* gp = plan.granule + (size_t)sh * keep;
  const uint32_t bits = 3 + vs, dim = tid & ((1u << bits) - 1u), granules = F * EM_G >> vs;
  const uint32_t mask = (1u << g.shift) - 1u, d = (sl << bits) + dim;
  const uint16_t* elems = reinterpret_cast<const uint16_t*>(s_g);
  constexpr uint32_t U = F * EM_G * 8 / EM_NT;  // granules of a thread
  for (uint32_t j0 = 0, j1; j0 < keep; j0 = j1) {
    // the chunk's rows [j0, j1): whole output granules (but for the last) whose sources are granules t0 and up;
    // 512 ends of 8 rows are looked at, and granules up to the last that any of them can have; more than
    // the chunk's are not loaded
    const uint32_t t0 = fp[j0] >> 3;
    const uint32_t t_end = fp[min(keep, j0 + 8 * (tid + 1)) - 1] >> 3;
    uint32_t slot[U];
#pragma unroll
    for (uint32_t k = 0; k < U; ++k) slot[k] = gp[min(t0 + ((k * EM_NT + tid) >> bits), keep - 1)] << 3;
    const uint64_t fit = __ballot(j0 + 8 * tid < keep && t_end < t0 + granules);
    if ((tid & 63u) == 0) s_end[tid >> 6] = __popcll(fit);
    __syncthreads();
    uint32_t n8 = 0;
    for (uint32_t i = 0; i < EM_NT / 64; ++i) n8 += s_end[i];
    j1 = min(keep, j0 + 8 * n8);
    const uint32_t n_u = ((fp[j1 - 1] >> 3) - t0 + 1) << bits;
    u32x4 x[U];
#pragma unroll
    for (uint32_t k = 0; k < U; ++k)
      if (k * EM_NT + tid < n_u)
        x[k] = *reinterpret_cast<const u32x4*>(vc + paged_base(g, slot[k] >> g.shift, h) + paged_v(g, slot[k] & mask, d));
#pragma unroll
    for (uint32_t k = 0; k < U; ++k)
      if (k * EM_NT + tid < n_u) s_g[k * EM_NT + tid] = x[k];
    __syncthreads();
    for (uint32_t j = j0 + ((tid >> bits) << 3); j < j1; j += (EM_NT >> bits) << 3) {
      uint32_t v[8];
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t f = fp[min(j + i, keep - 1)];
        v[i] = elems[(((((f >> 3) - t0) << bits) + dim) << 3) + (f & 7u)];
      }
      uint16_t* dst = vc + paged_base(g, tab[j >> g.shift], h) + paged_v(g, j & mask, d);
      if (j + 8 <= keep) {
        *reinterpret_cast<u32x4*>(dst) = u32x4{v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16};
      } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
          if (j + i < keep) dst[i] = (uint16_t)v[i];
      }
    }
    __syncthreads();
  }
}

// V's workgroups first: they take longer.
template <uint32_t F>
__global__ __launch_bounds__(EM_NT, F == 1 ? 8 : F == 2 ? 4 : 2)
void k_evict_move(Paged g, uint16_t* __restrict__ kc, uint16_t* __restrict__ vc, uint32_t keep, EvictPlan plan,
                  uint32_t* __restrict__ lens_out, uint32_t ks, uint32_t vs) {
  extern __shared__ u32x4 s_g[];  // [granule][dim], 8 positions each
  __shared__ uint32_t s_end[EM_NT / 64];
  const uint32_t v_slices = g.hd >> (3 + vs), n_v = g.n_seqs * g.n_kv * v_slices;
  const bool is_v = blockIdx.x < n_v;
  const uint32_t b = is_v ? blockIdx.x : blockIdx.x - n_v, slices = is_v ? v_slices : g.hd >> (3 + ks);
  const uint32_t sh = b / slices, sl = b - sh * slices, s = sh / g.n_kv;
  if (is_v && sl == 0 && sh == s * g.n_kv && threadIdx.x == 0) lens_out[s] = plan.new_lens[s];
  if (!plan.old_lens[s]) return;
  if (is_v) evict_move_v<F>(g, vc, keep, plan, sh, sl, vs, s_g, s_end);
  else evict_move_k<F>(g, kc, keep, plan, sh, sl, ks);
}

}  // namespace cm
