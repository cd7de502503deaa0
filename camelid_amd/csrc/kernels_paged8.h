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

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

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

// The same for a largest |element| in f64.
template <int KT>
__device__ __forceinline__ uint32_t p8_exponent(uint64_t top) {
  if (top >= 0x7ff0000000000000ull) return P8_NAN;
  const int bits = KT == TY_I8 ? 6 : 8, most = KT == TY_I8 ? 248 : 246;
  const uint64_t edge = KT == TY_I8 ? 0xfc00000000000ull : 0xc000000000000ull;
  const int e = (int)(top >> 52) - 1023 + 127 - bits + ((top & 0xfffffffffffffull) > edge ? 1 : 0);
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
// f64 values -> f32 that p8_pack4 takes to the byte which is nearest to the f64 value (f32 first would round twice).
template <int KT>
__device__ __forceinline__ float p8_round(double x) {
  if constexpr (KT == TY_I8) return (float)rint(x);
  // four bits from the leading one on, 2^-9 at the least: the sum's last bit is that one
  const int e = max((int)(d2u(x) >> 52 & 0x7ffu) - 1023, -6);
  const double c = u2d((uint64_t)(min(e, 64) + 49 + 1023) << 52) * 1.5;
  return (float)((x + c) - c);
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
// The bytes of a word that are NaN in e4m3, as 255.
__device__ __forceinline__ uint32_t p8_nan_bytes(uint32_t u) {
  return ((((u & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 255u;
}
// 2^(b - 127) of an exponent byte.
__device__ __forceinline__ float p8_scale(uint32_t b) {
  return b == P8_NAN ? u2f(0x7fc00000u) : b ? u2f(b << 23) : 0x1p-127f;
}
// x 2^(from - to) of exponent bytes, rounded once (x of up to 8 bits: exact unless subnormal).
__device__ __forceinline__ float p8_shift(float x, uint32_t from, uint32_t to) { return ldexpf(x, (int)from - (int)to); }

// ---------------------------------------------------------------------------
// Per-head RMSNorm (optional) + RoPE of the new tokens' q and k rows, K and V to 8 bits.  q: the arithmetic and
// bits of k_paged_rope_kv.  K is worked out in f64 and rounded once: a byte is on the right side of its
// border then, however sums are ordered (f32 with the norm's sum in order put three times as many on the wrong one as a
// tree sum).  Whoever writes into a block of 16 positions sees all of it: one workgroup does a block of a sequence
// for some heads of q, K or V (a role).
//   q, K: HD / 16 lanes per (token, head), each 8 dims of either half, which hold the pairs of both pairings.
//   V:    a lane per dim, its granule in registers.
// Bound: HBM and, with 3 workgroups a CU (the f64 registers of K), its latency: 55 us for 196 MB (4 prompts of up to 2047
// tokens, 32 + 8 + 8 heads of 128, QK norm; 46 us without the norm), 9.0 us for a token of each of 64 sequences of those
// heads, 3.9 us for one token of 32 + 4 + 4 heads of 64.
constexpr uint32_t R8_NT = 256;
constexpr uint32_t r8_heads(uint32_t hd) { return R8_NT / (hd / 16) / P8_BLOCK; }  // q or K heads of a workgroup
constexpr uint32_t r8_v_heads(uint32_t hd) { return R8_NT / hd; }
__host__ __device__ constexpr uint32_t r8_roles(uint32_t hd, uint32_t n_heads, uint32_t n_kv) {
  return (n_heads + r8_heads(hd) - 1) / r8_heads(hd) + (n_kv + r8_heads(hd) - 1) / r8_heads(hd) +
         (n_kv + r8_v_heads(hd) - 1) / r8_v_heads(hd);
}
// Blocks that n_new consecutive positions can reach into.
constexpr uint32_t r8_blocks(uint32_t n_new) { return (uint32_t)(((uint64_t)n_new + 14) / 16 + 1); }

__device__ __forceinline__ uint64_t r8_max64(uint64_t a, uint64_t b) { return a > b ? a : b; }
// |x| as bits that order as it does, NaN above all.
__device__ __forceinline__ uint64_t r8_size(double x) { return d2u(x) & ~(1ull << 63); }
// Maximum over the wave.
__device__ __forceinline__ uint32_t r8_wave_max(uint32_t x) {
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) x = max(x, (uint32_t)__shfl_xor((int)x, i));
  return x;
}

// 4 bytes from a block's exponent `was` to `now`; NaN stays NaN.
template <int KT>
__device__ __forceinline__ uint32_t p8_requantised(uint32_t u, uint32_t was, uint32_t now) {
  float x[4];
  p8_unpack4<KT>(u, x);
  const uint32_t w = p8_pack4<KT>(p8_shift(x[0], was, now), p8_shift(x[1], was, now), p8_shift(x[2], was, now),
                                  p8_shift(x[3], was, now));
  const uint32_t nan = KT == TY_E4M3 ? p8_nan_bytes(u) : 0u;
  return (w & ~nan) | (u & nan);
}
template <int KT>
__device__ __forceinline__ uint2 p8_requantised(uint2 u, uint32_t was, uint32_t now) {
  return make_uint2(p8_requantised<KT>(u.x, was, now), p8_requantised<KT>(u.y, was, now));
}

// Pairs (a, b) rotated: a and b hold dims 8 j .. and HALF + 8 j .., pairs across them or inside each.
template <typename F>
__device__ __forceinline__ void r8_turn(F (&a)[8], F (&b)[8], const float (&c)[8], const float (&s)[8], bool split_half) {
  if (split_half) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const F x0 = a[i], x1 = b[i];
      a[i] = (x0 * c[i]) - (x1 * s[i]);
      b[i] = (x0 * s[i]) + (x1 * c[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const F x0 = a[2 * i], x1 = a[2 * i + 1], y0 = b[2 * i], y1 = b[2 * i + 1];
      a[2 * i] = (x0 * c[i]) - (x1 * s[i]);
      a[2 * i + 1] = (x0 * s[i]) + (x1 * c[i]);
      b[2 * i] = (y0 * c[4 + i]) - (y1 * s[4 + i]);
      b[2 * i + 1] = (y0 * s[4 + i]) + (y1 * c[4 + i]);
    }
  }
}

template <int HD, int QT, int KT>
__global__ __launch_bounds__(R8_NT, 3) void k_paged8_rope_kv16(Paged8 c, const float* __restrict__ qkv, uint32_t n_new,
                                                            const uint32_t* __restrict__ new_lens, uint32_t n_heads,
                                                            uint32_t split_half, const float* __restrict__ cosv,
                                                            const float* __restrict__ sinv,
                                                            const float* __restrict__ q_norm,
                                                            const float* __restrict__ k_norm, float eps,
                                                            void* __restrict__ q_out, uint32_t roles, uint32_t blocks) {
  constexpr uint32_t LPR = HD / 16, PAIRS = R8_NT / LPR, HEADS = r8_heads(HD), V_HEADS = r8_v_heads(HD), HALF = HD / 2;
  __shared__ float s_x[PAIRS][HD + 4];
  __shared__ float s_scale[PAIRS];
  __shared__ uint64_t s_top[HEADS > V_HEADS ? HEADS : V_HEADS];
  const Paged& g = c.g;
  const uint32_t tid = threadIdx.x, role = blockIdx.x % roles, sb = blockIdx.x / roles, s = sb / blocks;
  uint32_t first, len;
  if (!paged_rows(g, new_lens, n_new, s, &first, &len)) return;
  const uint32_t p0 = (first & ~15u) + P8_BLOCK * (sb - s * blocks);  // the block's first position
  if (p0 >= len || first == len) return;
  const size_t width = (size_t)(n_heads + 2 * g.n_kv) * HD;
  const uint32_t q_roles = (n_heads + HEADS - 1) / HEADS, k_roles = (g.n_kv + HEADS - 1) / HEADS;
  const uint32_t o0 = p0 & ((1u << g.shift) - 1u), lo = max(p0, first) - p0, hi = min(p0 + P8_BLOCK, len) - p0;
  const bool isq = role < q_roles;
  uint32_t page = 0;
  if (!isq) {
    page = g.table[(size_t)s * g.stride + (p0 >> g.shift)];
    if (page >= g.n_pages) {
      if (tid == 0) paged_flag(g, PG_BAD_PAGE);
      return;
    }
    if (tid < (HEADS > V_HEADS ? HEADS : V_HEADS)) s_top[tid] = 0;
    __syncthreads();
  }
  if (role >= q_roles + k_roles) {
    const uint32_t hl = tid / HD, h = (role - q_roles - k_roles) * V_HEADS + hl, d = tid % HD;
    const bool live = h < g.n_kv;
    const float* src = qkv + ((size_t)s * n_new) * width + (size_t)(n_heads + g.n_kv + h) * HD + d;
    uint8_t* e = c.ve + p8_exp(g, page, h, o0);
    u32x4* dst = reinterpret_cast<u32x4*>(c.vc + p8_base(g, page, h) + p8_v(g, o0, d));
    float x[16];
    uint32_t top = 0;
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) x[i] = live && i >= lo && i < hi ? src[(size_t)(p0 + i - first) * width] : 0.0f;
    u32x4 old{};
    uint32_t was = 0;
    if (live && hi - lo < 16) old = *dst;
    if (live && lo) was = *e;
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) top = max(top, f2u(x[i]) & 0x7fffffffu);
    top = r8_wave_max(top);
    if ((tid & 63u) == 0) atomicMax(reinterpret_cast<uint32_t*>(&s_top[hl]), top);
    __syncthreads();
    if (!live) return;
    const uint32_t now = max(p8_exponent<KT>((uint32_t)s_top[hl]), was);
    if (d == 0) *e = (uint8_t)now;
    if (now == P8_NAN) return;  // (its bytes stand for nothing)
    u32x4 u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      u[i] = p8_pack4<KT>(ldexpf(x[4 * i], 127 - (int)now), ldexpf(x[4 * i + 1], 127 - (int)now),
                          ldexpf(x[4 * i + 2], 127 - (int)now), ldexpf(x[4 * i + 3], 127 - (int)now));
    if (hi - lo < 16) {
      u32x4 kept = old;
      if (lo && now != was) {
#pragma unroll
        for (int i = 0; i < 4; ++i) kept[i] = p8_requantised<KT>(old[i], was, now);
      }
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) {
        const uint32_t m = 0xffu << (8 * (i & 3));
        const uint32_t from = i < lo ? kept[i >> 2] : i < hi ? u[i >> 2] : old[i >> 2];
        u[i >> 2] = (u[i >> 2] & ~m) | (from & m);
      }
    }
    *dst = u;
    return;
  }
  const uint32_t j = tid % LPR, pair = tid / LPR, i16 = pair % P8_BLOCK, hl = pair / P8_BLOCK;
  const uint32_t h = (isq ? role : role - q_roles) * HEADS + hl;
  const bool real = h < (isq ? n_heads : g.n_kv), live = real && i16 >= lo && i16 < hi;
  const size_t row = (size_t)s * n_new + (p0 + i16 - first);
  float a[8], b[8];  // dims 8 j .. and HALF + 8 j ..
  float ca[8], sa[8];
  if (live) {
    const float* src = qkv + row * width + (size_t)(isq ? h : n_heads + h) * HD;
    rk_load8(src + 8 * j, a);
    rk_load8(src + HALF + 8 * j, b);
    const float *cr = cosv + row * HALF, *sr = sinv + row * HALF;
    if (split_half) {  // pairs 8 j .. 8 j + 7: (a, b)
      rk_load8(cr + 8 * j, ca);
      rk_load8(sr + 8 * j, sa);
    } else {  // pairs 4 j .. inside a, HALF / 2 + 4 j .. inside b
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const f32x4v x = *reinterpret_cast<const f32x4v*>(cr + k * (HALF / 2) + 4 * j);
        const f32x4v y = *reinterpret_cast<const f32x4v*>(sr + k * (HALF / 2) + 4 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ca[4 * k + i] = x[i];
          sa[4 * k + i] = y[i];
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = b[i] = ca[i] = sa[i] = 0.0f;
  }
  const float* nw = isq ? q_norm : k_norm;
  if (isq) {
    if (nw) {
      if (live) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          s_x[pair][8 * j + i] = a[i] * a[i];  // (the squares, rounded: the sum in order is left to one lane)
          s_x[pair][HALF + 8 * j + i] = b[i] * b[i];
        }
      }
      __syncthreads();
      if (tid < PAIRS) {  // (padding rows sum what lies there)
        float acc = 0.0f;
#pragma unroll 8
        for (uint32_t d = 0; d < HD; d += 4) {
          const f32x4v x = *reinterpret_cast<const f32x4v*>(&s_x[tid][d]);
          acc = (((acc + x[0]) + x[1]) + x[2]) + x[3];
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
    r8_turn(a, b, ca, sa, split_half);
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
    return;
  }
  // K: 8 bytes of either half (dims 8 j are half a granule)
  uint8_t* e = c.ke + p8_exp(g, page, h, o0);
  uint8_t* base = c.kc + p8_base(g, page, h);
  uint2* at0 = reinterpret_cast<uint2*>(base + p8_k(g, o0 + i16, 8 * j));
  uint2* at1 = reinterpret_cast<uint2*>(base + p8_k(g, o0 + i16, HALF + 8 * j));
  const bool earlier = real && i16 < lo;
  uint2 old0{}, old1{};
  if (earlier) {
    old0 = *at0;
    old1 = *at1;
  }
  const uint32_t was = real && lo ? *e : 0u;
  double x[8], y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = a[i];
    y[i] = b[i];
  }
  if (nw) {
    double acc = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc += x[i] * x[i] + y[i] * y[i];
#pragma unroll
    for (uint32_t i = 1; i < LPR; i <<= 1) acc += __shfl_xor(acc, i);
    const double sc = 1.0 / sqrt(acc / (double)HD + (double)eps);
    if (live) {
      float wa[8], wb[8];
      rk_load8(nw + 8 * j, wa);
      rk_load8(nw + HALF + 8 * j, wb);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = (x[i] * sc) * wa[i];
        y[i] = (y[i] * sc) * wb[i];
      }
    }
  }
  r8_turn(x, y, ca, sa, split_half);
  uint64_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = r8_max64(top, r8_max64(r8_size(x[i]), r8_size(y[i])));
  if (!live) top = 0;
#pragma unroll
  for (uint32_t i = 1; i < 64 && i < LPR * P8_BLOCK; i <<= 1) top = r8_max64(top, __shfl_xor((unsigned long long)top, i));
  if ((tid & 63u) == 0) atomicMax(reinterpret_cast<unsigned long long*>(&s_top[hl]), (unsigned long long)top);
  __syncthreads();
  if (!real) return;
  const uint32_t now = max(p8_exponent<KT>(s_top[hl]), was);
  if (i16 == 0 && j == 0) *e = (uint8_t)now;
  if (now == P8_NAN) return;
  if (live) {
    float u[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      u[i] = p8_round<KT>(ldexp(x[i], 127 - (int)now));
      v[i] = p8_round<KT>(ldexp(y[i], 127 - (int)now));
    }
    *at0 = make_uint2(p8_pack4<KT>(u[0], u[1], u[2], u[3]), p8_pack4<KT>(u[4], u[5], u[6], u[7]));
    *at1 = make_uint2(p8_pack4<KT>(v[0], v[1], v[2], v[3]), p8_pack4<KT>(v[4], v[5], v[6], v[7]));
  } else if (earlier && now != was) {
    *at0 = p8_requantised<KT>(old0, was, now);
    *at1 = p8_requantised<KT>(old1, was, now);
  }
}

// The same with part of a head rotated, or none (rope_dim < head_dim): pairs fall anywhere.  One workgroup per
// (sequence, block, head of q, K or V), rows in LDS.  Bound: LDS and bytes stored one by one; right, not made fast:
// the prompts above with half of a head rotated take 247 us, 164 without the norm (sums by one lane a row).
template <int QT, int KT>
__global__ __launch_bounds__(R8_NT) void k_paged8_rope_kv(Paged8 c, const float* __restrict__ qkv, uint32_t n_new,
                                                          const uint32_t* __restrict__ new_lens, uint32_t n_heads,
                                                          uint32_t rope_dim, uint32_t split_half,
                                                          const float* __restrict__ cosv, const float* __restrict__ sinv,
                                                          const float* __restrict__ q_norm,
                                                          const float* __restrict__ k_norm, float eps,
                                                          void* __restrict__ q_out, uint32_t blocks) {
  __shared__ double s_x[P8_BLOCK][256 + 1];
  __shared__ double s_scale[P8_BLOCK];
  __shared__ uint64_t s_top;
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
      if (isq) {
        float acc = 0.0f;
        for (uint32_t d = 0; d < hd; ++d) acc = acc + (float)s_x[tid][d] * (float)s_x[tid][d];
        s_scale[tid] = 1.0f / sqrtf(acc / (float)hd + eps);
      } else {
        double acc = 0.0;
        for (uint32_t d = 0; d < hd; ++d) acc += s_x[tid][d] * s_x[tid][d];
        s_scale[tid] = 1.0 / sqrt(acc / (double)hd + (double)eps);
      }
    }
    __syncthreads();
    for (uint32_t i = tid; i < (hi - lo) * hd; i += R8_NT) {
      double& x = s_x[lo + i / hd][i % hd];
      const double sc = s_scale[lo + i / hd];
      x = isq ? (double)(((float)x * (float)sc) * nw[i % hd]) : (x * sc) * nw[i % hd];
    }
    __syncthreads();
  }
  const uint32_t half = rope_dim >> 1;
  if (isq || isk) {
    for (uint32_t i = tid; i < (hi - lo) * half; i += R8_NT) {
      const uint32_t t = lo + i / half, p = i % half;
      const uint32_t d0 = split_half ? p : 2 * p, d1 = split_half ? p + half : 2 * p + 1;
      const float cs = cosv[(row0 + t) * half + p], sn = sinv[(row0 + t) * half + p];
      const double x0 = s_x[t][d0], x1 = s_x[t][d1];
      s_x[t][d0] = isq ? (double)(((float)x0 * cs) - ((float)x1 * sn)) : (x0 * cs) - (x1 * sn);
      s_x[t][d1] = isq ? (double)(((float)x0 * sn) + ((float)x1 * cs)) : (x0 * sn) + (x1 * cs);
    }
    __syncthreads();
  }
  if (isq) {
    for (uint32_t i = tid; i < (hi - lo) * hd; i += R8_NT)
      store_from_f32<QT>(q_out, ((row0 + lo + i / hd) * n_heads + role) * hd + i % hd, (float)s_x[lo + i / hd][i % hd]);
    return;
  }
  const uint32_t h = role - n_heads - (isk ? 0u : g.n_kv);
  const uint32_t page = g.table[(size_t)s * g.stride + (p0 >> g.shift)], o0 = p0 & ((1u << g.shift) - 1u);
  if (page >= g.n_pages) {
    if (tid == 0) paged_flag(g, PG_BAD_PAGE);
    return;
  }
  uint64_t top = 0;
  for (uint32_t i = tid; i < (hi - lo) * hd; i += R8_NT) top = r8_max64(top, r8_size(s_x[lo + i / hd][i % hd]));
  atomicMax(reinterpret_cast<unsigned long long*>(&s_top), (unsigned long long)top);
  uint8_t* e = (isk ? c.ke : c.ve) + p8_exp(g, page, h, o0);
  uint8_t* base = (isk ? c.kc : c.vc) + p8_base(g, page, h);
  const uint32_t was = lo ? *e : 0u;
  __syncthreads();  // (all have read the old exponent)
  const uint32_t now = max(p8_exponent<KT>(s_top), was);
  if (tid == 0) *e = (uint8_t)now;
  if (now == P8_NAN) return;
  for (uint32_t i = tid; i < hi * hd; i += R8_NT) {
    const uint32_t t = i / hd, d = i % hd;
    uint8_t* p = base + (isk ? p8_k(g, o0 + t, d) : p8_v(g, o0 + t, d));
    if (t >= lo) {
      *p = (uint8_t)p8_pack4<KT>(p8_round<KT>(ldexp(s_x[t][d], 127 - (int)now)), 0.0f, 0.0f, 0.0f);
    } else if (now != was) {
      *p = (uint8_t)p8_requantised<KT>((uint32_t)*p, was, now);
    }
  }
}

// ---------------------------------------------------------------------------
// K and V of each sequence's positions [0, min(lens, n_out)) as rows [n_kv][n_out][hd] of type T.  One workgroup per
// (sequence, KV head, 4096 bytes of K or V: a granule a thread), which go through LDS so that rows are written
// whole.  Bound: HBM: 13 us for 39 MB (4 sequences of up to 2247 positions, 8 heads of 128, to f16), 3 TB/s; with
// K's 16 values stored by the lane that has them and V's one by one 35 us.
constexpr uint32_t RD_NT = 256;
constexpr uint32_t rd_span(uint32_t hd) { return RD_NT * 16 / hd; }  // positions of a workgroup
template <int HD, int KT, int T>
__global__ __launch_bounds__(RD_NT) void k_paged8_read(Paged8 c, void* __restrict__ k_out, void* __restrict__ v_out,
                                                       uint32_t n_out, uint32_t spans) {
  constexpr uint32_t SPAN = rd_span(HD), PITCH = HD + 4;
  const Paged& g = c.g;
  __shared__ float s_x[SPAN * PITCH];
  const uint32_t tid = threadIdx.x, which = blockIdx.x & 1u, rest = blockIdx.x >> 1;
  const uint32_t sh = rest / spans, p0 = (rest - sh * spans) * SPAN, s = sh / g.n_kv, h = sh - s * g.n_kv;
  const uint32_t len = g.lens[s];
  if ((uint64_t)len > ((uint64_t)g.stride << g.shift)) {
    if (tid == 0) paged_flag(g, PG_BAD_LENGTH);
    return;
  }
  const uint32_t end = min(len, n_out);
  if (p0 >= end) return;
  // K: granule tid / SPAN of position tid % SPAN; V: dim tid % HD of block tid / HD
  const uint32_t t = which ? 16 * (tid / HD) : tid % SPAN, d = which ? tid % HD : tid / SPAN;
  const uint32_t pos = min(p0 + t, end - 1), page = g.table[(size_t)s * g.stride + (pos >> g.shift)];
  const uint32_t o = pos & ((1u << g.shift) - 1u);
  const bool good = page < g.n_pages;
  if (!good) paged_flag(g, PG_BAD_PAGE);
  if (good) {
    const uint8_t* src = (which ? c.vc : c.kc) + p8_base(g, page, h) + (which ? p8_v(g, o & ~15u, d) : p8_k(g, o, 16 * d));
    const float scale = p8_scale((which ? c.ve : c.ke)[p8_exp(g, page, h, o)]);
    const u32x4 u = *reinterpret_cast<const u32x4*>(src);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x[4];
      p8_unpack4<KT>(u[j], x);
#pragma unroll
      for (int n = 0; n < 4; ++n)
        s_x[which ? (t + 4 * j + n) * PITCH + d : t * PITCH + 16 * d + 4 * j + n] = x[n] * scale;
    }
  }
  __syncthreads();
  constexpr uint32_t V = T == TY_F32 ? 4 : 8;  // elements of a store
  const uint32_t rows = min(SPAN, end - p0);
  char* out = static_cast<char*>(which ? v_out : k_out) + ((size_t)sh * n_out + p0) * HD * (T == TY_F32 ? 4 : 2);
  for (uint32_t i = tid; i < rows * (HD / V); i += RD_NT) {
    const uint32_t row = i / (HD / V), at = (i % (HD / V)) * V;
    if (g.table[(size_t)s * g.stride + ((p0 + row) >> g.shift)] >= g.n_pages) continue;
    const f32x4v a = *reinterpret_cast<const f32x4v*>(&s_x[row * PITCH + at]);
    if constexpr (T == TY_F32) {
      reinterpret_cast<f32x4v*>(out)[i] = a;
    } else {
      const f32x4v b = *reinterpret_cast<const f32x4v*>(&s_x[row * PITCH + at + 4]);
      const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      reinterpret_cast<rk_u32x4*>(out)[i] = rk_pack8<T>(x);
    }
  }
}

}  // namespace cm
