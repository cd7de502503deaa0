// kernels_paged8.h -- a key/value cache in pages, held in 8 bits: RoPE + store of new tokens, and reading back.
//
// Pages of page_size positions (a power of two >= 16).  K of one page is [n_kv][hd / 16][page_size][16]
// bytes, V is [n_kv][page_size / 16][hd][16]: granules of 16 bytes, 16 dims of one position for K, 16
// positions of one dim for V.  A block is 16 positions (one granule row of V) of one KV head; K and V have
// an exponent byte each for it, [page][n_kv][page_size / 16]: b stands for 2^(b - 127), 255 for NaN.  An
// element stands for its byte (int8 or e4m3) times that.
//
// Scales are powers of two, so that a block can grow: when a later token needs a larger one, the block's
// earlier positions are rounded again, by a shift (int8: the two half steps add up to less than one of
// the new steps) or not at all (e4m3, but for subnormals).  A scale amax / 127 would round every earlier
// position again with each new maximum, and a block filled token by token would not have the scale of one filled
// at once.  int8 pays up to one of its bits for it, e4m3 nothing.
#pragma once
#include "kernels_paged.h"

namespace cm {

enum { TY_I8 = 3, TY_E4M3 = 4 };  // CAMELID_I8, CAMELID_E4M3

constexpr uint32_t P8_BLOCK = 16;
constexpr uint32_t P8_NAN = 255;  // exponent byte of a block that holds NaN

struct Paged8 {
  Paged g;
  uint8_t* kc;
  uint8_t* vc;
  uint8_t* ke;
  uint8_t* ve;
};

// Byte offset of (page, kv head) in the K or V buffer, of a block's exponent.
__device__ __forceinline__ size_t p8_base(const Paged& g, uint32_t page, uint32_t h) { return paged_base(g, page, h); }
__device__ __forceinline__ size_t p8_exp(const Paged& g, uint32_t page, uint32_t h, uint32_t o) {
  return (((size_t)page * g.n_kv + h) << (g.shift - 4)) + (o >> 4);
}
// Offset inside it of dim d of the page's position o.
__device__ __forceinline__ uint32_t p8_k(const Paged& g, uint32_t o, uint32_t d) {
  return ((((d >> 4) << g.shift) + o) << 4) + (d & 15u);
}
__device__ __forceinline__ uint32_t p8_v(const Paged& g, uint32_t o, uint32_t d) {
  return (((o >> 4) * g.hd + d) << 4) + (o & 15u);
}

// The exponent byte of a block whose largest |element| has the bits `top`: the smallest 2^e with
// top <= 127 2^e (int8) or 448 2^e (e4m3), from 2^-126 on, and so that the largest element is an f32
// (values of f32's last binade saturate).  Infinity and NaN: P8_NAN.
template <int KT>
__device__ __forceinline__ uint32_t p8_exponent(uint32_t top) {
  if (top >= 0x7f800000u) return P8_NAN;
  const int bits = KT == TY_I8 ? 6 : 8, most = KT == TY_I8 ? 248 : 246;
  const uint32_t edge = KT == TY_I8 ? 0x7e0000u : 0x600000u;  // mantissas of 127 / 64 and 448 / 256
  const int e = (int)(top >> 23) - bits + ((top & 0x7fffffu) > edge ? 1 : 0);
  return (uint32_t)max(1, min(most, e));
}

// f32 values (already divided by the scale) -> bytes, to nearest even.
template <int KT>
__device__ __forceinline__ uint32_t p8_pack4(float a, float b, float c, float d) {
  if constexpr (KT == TY_I8) {
    const auto q = [](float x) { return (uint32_t)(int)fminf(127.0f, fmaxf(-127.0f, rintf(x))) & 0xffu; };
    return q(a) | q(b) << 8 | q(c) << 16 | q(d) << 24;
  } else {
    const auto q = [](float x) { return fminf(448.0f, fmaxf(-448.0f, x)); };
    int u = __builtin_amdgcn_cvt_pk_fp8_f32(q(a), q(b), 0, false);
    u = __builtin_amdgcn_cvt_pk_fp8_f32(q(c), q(d), u, true);
    return (uint32_t)u;
  }
}
// Byte i of a word as the number that it stands for without its block's scale.
template <int KT>
__device__ __forceinline__ void p8_unpack4(uint32_t u, float (&x)[4]) {
  if constexpr (KT == TY_I8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(u >> (8 * i));
  } else {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, true);
    x[0] = lo[0];
    x[1] = lo[1];
    x[2] = hi[0];
    x[3] = hi[1];
  }
}
// 2^(b - 127) of an exponent byte.
__device__ __forceinline__ float p8_scale(uint32_t b) {
  return b == P8_NAN ? u2f(0x7fc00000u) : b ? u2f(b << 23) : 0x1p-127f;
}
// x 2^(from - to) of exponent bytes, rounded once (x of up to 8 bits: exact unless subnormal).
__device__ __forceinline__ float p8_shift(float x, uint32_t from, uint32_t to) { return ldexpf(x, (int)from - (int)to); }

// ---------------------------------------------------------------------------
// Per-head RMSNorm (optional) + RoPE of the new tokens' q and k rows (the arithmetic of k_paged_rope_kv: the
// same q bits), K and V to 8 bits.  One workgroup per (sequence, block of 16 positions, head of q, K or V),
// so that whoever writes into a block sees all of it.
constexpr uint32_t R8_NT = 256;
// Blocks that n_new consecutive positions can reach into.
constexpr uint32_t r8_blocks(uint32_t n_new) { return (uint32_t)(((uint64_t)n_new + 14) / 16 + 1); }

template <int QT, int KT>
__global__ __launch_bounds__(R8_NT) void k_paged8_rope_kv(Paged8 c, const float* __restrict__ qkv, uint32_t n_new,
                                                          const uint32_t* __restrict__ new_lens, uint32_t n_heads,
                                                          uint32_t rope_dim, uint32_t split_half,
                                                          const float* __restrict__ cosv, const float* __restrict__ sinv,
                                                          const float* __restrict__ q_norm,
                                                          const float* __restrict__ k_norm, float eps,
                                                          void* __restrict__ q_out, uint32_t blocks) {
  __shared__ float s_x[P8_BLOCK][256 + 1];
  __shared__ float s_scale[P8_BLOCK];
  __shared__ uint32_t s_top;
  const Paged& g = c.g;
  const uint32_t tid = threadIdx.x, hd = g.hd, roles = n_heads + 2 * g.n_kv;
  const uint32_t role = blockIdx.x % roles, sb = blockIdx.x / roles, s = sb / blocks;
  uint32_t first, len;
  if (!paged_rows(g, new_lens, n_new, s, &first, &len)) return;
  const uint32_t p0 = (first & ~15u) + P8_BLOCK * (sb - s * blocks);
  if (p0 >= len || first == len) return;
  const uint32_t lo = max(p0, first) - p0, hi = min(p0 + P8_BLOCK, len) - p0;  // the block's new positions
  const size_t width = (size_t)roles * hd, row0 = (size_t)s * n_new - first + p0;  // activation row of offset 0
  for (uint32_t i = tid; i < (hi - lo) * hd; i += R8_NT)
    s_x[lo + i / hd][i % hd] = qkv[(row0 + lo + i / hd) * width + (size_t)role * hd + i % hd];
  if (tid == 0) s_top = 0;
  __syncthreads();
  const bool isq = role < n_heads, isk = !isq && role < n_heads + g.n_kv;
  const float* nw = isq ? q_norm : isk ? k_norm : nullptr;
  if (nw) {
    if (tid >= lo && tid < hi) {
      float acc = 0.0f;
      for (uint32_t d = 0; d < hd; ++d) acc = acc + s_x[tid][d] * s_x[tid][d];
      s_scale[tid] = 1.0f / sqrtf(acc / (float)hd + eps);
    }
    __syncthreads();
    for (uint32_t i = tid; i < (hi - lo) * hd; i += R8_NT)
      s_x[lo + i / hd][i % hd] = (s_x[lo + i / hd][i % hd] * s_scale[lo + i / hd]) * nw[i % hd];
    __syncthreads();
  }
  const uint32_t half = rope_dim >> 1;
  if (isq || isk) {
    for (uint32_t i = tid; i < (hi - lo) * half; i += R8_NT) {
      const uint32_t t = lo + i / half, p = i % half;
      const uint32_t d0 = split_half ? p : 2 * p, d1 = split_half ? p + half : 2 * p + 1;
      const float cs = cosv[(row0 + t) * half + p], sn = sinv[(row0 + t) * half + p];
      const float x0 = s_x[t][d0], x1 = s_x[t][d1];
      s_x[t][d0] = (x0 * cs) - (x1 * sn);
      s_x[t][d1] = (x0 * sn) + (x1 * cs);
    }
    __syncthreads();
  }
  if (isq) {
    for (uint32_t i = tid; i < (hi - lo) * hd; i += R8_NT)
      store_from_f32<QT>(q_out, ((row0 + lo + i / hd) * n_heads + role) * hd + i % hd, s_x[lo + i / hd][i % hd]);
    return;
  }
  const uint32_t h = role - n_heads - (isk ? 0u : g.n_kv);
  const uint32_t page = g.table[(size_t)s * g.stride + (p0 >> g.shift)], o0 = p0 & ((1u << g.shift) - 1u);
  if (page >= g.n_pages) {
    if (tid == 0) paged_flag(g, PG_BAD_PAGE);
    return;
  }
  uint32_t top = 0;
  for (uint32_t i = tid; i < (hi - lo) * hd; i += R8_NT) top = max(top, f2u(s_x[lo + i / hd][i % hd]) & 0x7fffffffu);
  atomicMax(&s_top, top);
  __syncthreads();
  uint8_t* e = (isk ? c.ke : c.ve) + p8_exp(g, page, h, o0);
  uint8_t* base = (isk ? c.kc : c.vc) + p8_base(g, page, h);
  const uint32_t need = p8_exponent<KT>(s_top), was = lo ? *e : 0u, now = max(need, was);
  __syncthreads();  // (all have read the old exponent)
  if (tid == 0) *e = (uint8_t)now;
  if (now == P8_NAN) return;  // (its bytes stand for nothing)
  for (uint32_t i = tid; i < hi * hd; i += R8_NT) {
    const uint32_t t = i / hd, d = i % hd;
    uint8_t* p = base + (isk ? p8_k(g, o0 + t, d) : p8_v(g, o0 + t, d));
    float x;
    if (t >= lo) {
      x = ldexpf(s_x[t][d], 127 - (int)now);
    } else {
      if (now == was) continue;
      float old[4];
      p8_unpack4<KT>(*p, old);
      x = p8_shift(old[0], was, now);
    }
    *p = (uint8_t)p8_pack4<KT>(x, 0.0f, 0.0f, 0.0f);
  }
}

// ---------------------------------------------------------------------------
// K and V of each sequence's positions [0, min(lens, n_out)) as rows [n_kv][n_out][hd] of type T.  One
// workgroup per (sequence, KV head, 16 positions, K or V); V's granules are turned in LDS.  Bound: HBM.
constexpr uint32_t RD_NT = 256;
template <int HD, int KT, int T>
__global__ __launch_bounds__(RD_NT) void k_paged8_read(Paged8 c, void* __restrict__ k_out, void* __restrict__ v_out,
                                                       uint32_t n_out, uint32_t blocks) {
  const Paged& g = c.g;
  __shared__ float s_v[P8_BLOCK][HD + 1];
  const uint32_t tid = threadIdx.x, which = blockIdx.x & 1u, rest = blockIdx.x >> 1;
  const uint32_t sh = rest / blocks, p0 = (rest - sh * blocks) * P8_BLOCK, s = sh / g.n_kv, h = sh - s * g.n_kv;
  const uint32_t len = g.lens[s];
  if ((uint64_t)len > ((uint64_t)g.stride << g.shift)) {
    if (tid == 0) paged_flag(g, PG_BAD_LENGTH);
    return;
  }
  const uint32_t end = min(len, n_out);
  if (p0 >= end) return;
  const uint32_t page = g.table[(size_t)s * g.stride + (p0 >> g.shift)], o0 = p0 & ((1u << g.shift) - 1u);
  if (page >= g.n_pages) {
    if (tid == 0) paged_flag(g, PG_BAD_PAGE);
    return;
  }
  const uint8_t* src = (which ? c.vc : c.kc) + p8_base(g, page, h);
  const float scale = p8_scale((which ? c.ve : c.ke)[p8_exp(g, page, h, o0)]);
  const size_t dst = ((size_t)sh * n_out + p0) * HD;
  const uint32_t rows = min(P8_BLOCK, end - p0);
  for (uint32_t i = tid; i < P8_BLOCK * HD / 16; i += RD_NT) {
    const uint32_t t = i % P8_BLOCK, d = which ? i : i / P8_BLOCK;  // K: granule d of position t; V: dim d
    if (!which && t >= rows) continue;
    const uint4 u = *reinterpret_cast<const uint4*>(src + (which ? p8_v(g, o0, d) : p8_k(g, o0 + t, 16 * d)));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x[4];
      p8_unpack4<KT>(w[j], x);
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        if (which) s_v[4 * j + n][d] = x[n] * scale;
        else store_from_f32<T>(k_out, dst + (size_t)t * HD + 16 * d + 4 * j + n, x[n] * scale);
      }
    }
  }
  if (!which) return;
  __syncthreads();
  for (uint32_t i = tid; i < rows * HD; i += RD_NT) store_from_f32<T>(v_out, dst + i, s_v[i / HD][i % HD]);
}

}  // namespace cm
