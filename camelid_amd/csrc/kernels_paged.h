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
// the arithmetic of k_rope_kv, so an f16 cache holds the same bits.  One wave per (row, head).
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

constexpr int EV_NT = 1024;

// Exclusive prefix sum of v over the workgroup's threads; *total the whole sum.
__device__ __forceinline__ uint32_t evict_scan(uint32_t v, uint32_t* wave_sums, uint32_t* total) {
  const uint32_t lane = threadIdx.x & 63u, w = threadIdx.x >> 6;
  uint32_t x = v;
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(x, o);
    if (lane >= (uint32_t)o) x += y;
  }
  if (lane == 63) wave_sums[w] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
  for (uint32_t i = 0; i < EV_NT / 64; ++i) {
    const uint32_t y = wave_sums[i];
    if (i < w) before += y;
    all += y;
  }
  __syncthreads();
  *total = all;
  return before + x - v;
}

// One workgroup per (sequence, KV head): src[keep] = the kept positions in order (also to `kept`),
// the weights compacted, old_lens[s] = the length before where rows have to move, else 0.
__global__ __launch_bounds__(EV_NT) void k_evict_select(Paged g, float* __restrict__ weights, uint32_t keep,
                                                        uint32_t recent, uint32_t* __restrict__ src,
                                                        uint32_t* __restrict__ old_lens,
                                                        uint32_t* __restrict__ new_lens,
                                                        uint32_t* __restrict__ kept) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t wave_sums[EV_NT / 64];
  __shared__ uint32_t s_digit, s_rank, s_bad;
  const uint32_t s = blockIdx.x / g.n_kv, h = blockIdx.x % g.n_kv, tid = threadIdx.x;
  const uint32_t L = g.lens[s], cap = g.stride << g.shift;
  if (tid == 0) s_bad = 0;
  __syncthreads();
  const bool too_long = (uint64_t)L > ((uint64_t)g.stride << g.shift);
  if (too_long) {
    if (tid == 0) paged_flag(g, PG_BAD_LENGTH);
  } else {
    for (uint32_t i = tid; i < (L + (1u << g.shift) - 1u) >> g.shift; i += EV_NT)
      if (g.table[(size_t)s * g.stride + i] >= g.n_pages) s_bad = 1;
  }
  __syncthreads();
  if (s_bad && tid == 0) paged_flag(g, PG_BAD_PAGE);
  const bool moves = !too_long && !s_bad && L > keep;
  if (h == 0 && tid == 0) {
    old_lens[s] = moves ? L : 0u;
    new_lens[s] = moves ? keep : L;
  }
  uint32_t* kp = kept ? kept + (size_t)blockIdx.x * keep : nullptr;
  if (!moves) {
    if (kp && !too_long)
      for (uint32_t j = tid; j < min(L, keep); j += EV_NT) kp[j] = j;
    return;
  }
  float* w = weights + (size_t)blockIdx.x * cap;
  uint32_t* sp = src + (size_t)blockIdx.x * keep;
  const uint32_t cut = L - recent;
  uint32_t rank = keep - recent;  // positions still to be found among the keys equal in the digits so far
  uint32_t prefix = 0;
  for (int b = 24; b >= 0 && rank; b -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (uint32_t p = tid; p < cut; p += EV_NT) {
      const uint32_t k = evict_key(w[p]);
      if (b == 24 || (k >> (b + 8)) == (prefix >> (b + 8))) atomicAdd(&hist[(k >> b) & 255u], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t left = rank;
      int d = 255;
      while (hist[d] < left) left -= hist[d--];
      s_digit = (uint32_t)d;
      s_rank = left;
    }
    __syncthreads();
    prefix |= s_digit << b;
    rank = s_rank;
    __syncthreads();
  }
  // kept: every key above `prefix`, the first `rank` keys equal to it, and the recent positions
  const bool any = keep > recent;
  uint32_t eq_before = 0, out = 0;
  for (uint32_t p0 = 0; p0 < L; p0 += EV_NT) {
    const uint32_t p = p0 + tid;
    const float x = p < L ? w[p] : 0.0f;
    const uint32_t k = evict_key(x);
    const bool other = p < cut && any;
    const bool eq = other && k == prefix;
    uint32_t total;
    const uint32_t eq_rank = eq_before + evict_scan(eq ? 1u : 0u, wave_sums, &total);
    eq_before += total;
    const bool take = p < L && (p >= cut || (other && (k > prefix || (eq && eq_rank < rank))));
    const uint32_t j = out + evict_scan(take ? 1u : 0u, wave_sums, &total);
    out += total;
    if (take) {  // j <= p: every later position is still in place
      sp[j] = p;
      w[j] = x;
      if (kp) kp[j] = p;
    }
    __syncthreads();
  }
}

// The move, in place: output positions in chunks, a chunk's sources read before any of it is
// written.  A source is never below its output position, so no later chunk misses a row.  One
// workgroup per (sequence, KV head, 8 dims of K) and per (sequence, KV head, 32 dims of V).
constexpr uint32_t EM_NT = 256;
__global__ __launch_bounds__(EM_NT) void k_evict_move(Paged g, uint16_t* __restrict__ kc, uint16_t* __restrict__ vc,
                                                      uint32_t keep, const uint32_t* __restrict__ src,
                                                      const uint32_t* __restrict__ old_lens,
                                                      const uint32_t* __restrict__ new_lens,
                                                      uint32_t* __restrict__ lens_out) {
  const uint32_t slices = g.hd / 8 + g.hd / 32, tid = threadIdx.x;
  const uint32_t sl = blockIdx.x % slices, sh = blockIdx.x / slices, s = sh / g.n_kv, h = sh % g.n_kv;
  if (sl == 0 && h == 0 && tid == 0) lens_out[s] = new_lens[s];
  if (!old_lens[s]) return;
  const uint32_t* tab = g.table + (size_t)s * g.stride;
  const uint32_t* sp = src + (size_t)sh * keep;
  const uint32_t mask = (1u << g.shift) - 1u;
  if (sl < g.hd / 8) {
    for (uint32_t j0 = 0; j0 < keep; j0 += EM_NT) {
      const uint32_t j = j0 + tid;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (j < keep) {
        const uint32_t p = sp[j];
        x = *reinterpret_cast<const uint4*>(kc + paged_base(g, tab[p >> g.shift], h) + paged_k(g, p & mask, sl * 8));
      }
      __syncthreads();
      if (j < keep)
        *reinterpret_cast<uint4*>(kc + paged_base(g, tab[j >> g.shift], h) + paged_k(g, j & mask, sl * 8)) = x;
      __syncthreads();
    }
    return;
  }
  const uint32_t d = (sl - g.hd / 8) * 32 + (tid & 31u), step = EM_NT / 32 * 8;
  for (uint32_t j0 = 0; j0 < keep; j0 += step) {
    const uint32_t j = j0 + (tid >> 5) * 8;
    union { uint16_t e[8]; uint4 v; } x;
    for (uint32_t i = 0; i < 8; ++i) {
      if (j + i >= keep) continue;
      const uint32_t p = sp[j + i];
      x.e[i] = vc[paged_base(g, tab[p >> g.shift], h) + paged_v(g, p & mask, d)];
    }
    __syncthreads();
    if (j < keep) {
      uint16_t* dst = vc + paged_base(g, tab[j >> g.shift], h) + paged_v(g, j & mask, d);
      if (j + 8 <= keep) {
        *reinterpret_cast<uint4*>(dst) = x.v;
      } else {
        for (uint32_t i = 0; j + i < keep; ++i) dst[i] = x.e[i];
      }
    }
    __syncthreads();
  }
}

}  // namespace cm
