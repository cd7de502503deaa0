// kernels_logits.h -- logits before a token is drawn from them: penalties for repeated tokens, biases, masks.
//
//   x' = x / r where x > 0, else x r, for tokens that the row's text has (history and drafts before the row)
//   x' -= f count, x' -= p where count > 0, of the text's tokens behind the prompt
//   x' += bias of the token (the last one listed);  -infinity where the mask's bit is 0
// each step rounded in f32, the result once to the logits' type.
#pragma once
#include "kernels_paged.h"

namespace cm {

constexpr uint32_t LG_NT = 512;
constexpr uint32_t LG_SLICE = 4096;  // tokens of a workgroup
constexpr uint32_t LG_SEEN = 1u << 31, LG_DRAFT = 1u << 30, LG_BIAS = 1u << 29, LG_COUNT = LG_BIAS - 1;

struct LogitsArgs {
  const void* in;
  void* out;
  const uint32_t* history;
  const uint32_t* history_lens;
  const uint32_t* prompt_lens;
  const uint32_t* drafts;
  const uint32_t* draft_lens;
  const float* repetition;
  const float* frequency;
  const float* presence;
  const uint32_t* bias_tokens;
  const float* bias_values;
  const uint32_t* bias_lens;
  const uint32_t* mask;
  uint64_t in_stride, out_stride, history_stride, mask_stride;
  uint32_t n_rows, vocab, slices, bias_stride;
};

// What the lists say of a token (its word w, not 0) applied to its logit.
struct LogitsRow {
  float r, f, p;
  const uint32_t* drafts;
  uint32_t n_drafts;  // before the row
  const float* biases;
};
__device__ __forceinline__ float lg_adjusted(float x, uint32_t w, uint32_t token, uint32_t bias, const LogitsRow& a) {
  uint32_t count = w & LG_COUNT;
  bool seen = w & LG_SEEN;
  if (w & LG_DRAFT) {
    for (uint32_t j = 0; j < a.n_drafts; ++j) {
      const bool same = a.drafts[j] == token;
      count += same;
      seen |= same;
    }
  }
  if (seen) x = x > 0.0f ? x / a.r : x * a.r;
  if (count) x = (x - a.f * (float)count) - a.p;
  if (w & LG_BIAS) x = x + a.biases[bias - 1];
  return x;
}

// One workgroup per (sequence, slice of the vocabulary): what the lists say of the slice's tokens goes to LDS
// once, then the sequence's rows, 8 logits a thread.  In place without a mask only the tokens that the lists name
// are read and written.  Bound: HBM where every logit is written; the history, which every slice
// reads, costs 4 bytes a token from the L2.
template <int T, bool SPARSE>
__global__ __launch_bounds__(LG_NT) void k_adjust_logits(LogitsArgs a) {
  __shared__ uint32_t s_word[LG_SLICE];  // LG_COUNT: occurrences behind the prompt
  __shared__ uint32_t s_bias[LG_SLICE];  // index of the last bias + 1 (where LG_BIAS is set)
  const uint32_t tid = threadIdx.x, s = blockIdx.x / a.slices, v0 = (blockIdx.x - s * a.slices) * LG_SLICE;
  const uint32_t n = min(LG_SLICE, a.vocab - v0);
  const uint32_t known = a.history ? (uint32_t)min((uint64_t)(a.history_lens ? a.history_lens[s] : ~0u), a.history_stride) : 0u;
  const uint32_t prompt = a.prompt_lens ? a.prompt_lens[s] : 0u;
  const uint32_t last = a.draft_lens ? min(a.draft_lens[s], a.n_rows - 1) : a.n_rows - 1;
  const uint32_t n_drafts = a.drafts ? last : 0u, rows = last + 1;
  const uint32_t biases = a.bias_tokens ? (a.bias_lens ? min(a.bias_lens[s], a.bias_stride) : a.bias_stride) : 0u;
  LogitsRow row{a.repetition ? a.repetition[s] : 1.0f, a.frequency ? a.frequency[s] : 0.0f,
                a.presence ? a.presence[s] : 0.0f, a.drafts + (size_t)s * (a.n_rows - 1), 0,
                a.bias_values + (size_t)s * a.bias_stride};
  // this thread's 8 logits of a row, as they lie, and their mask bits; a row's are on their way while the lists are
  // read or the two rows before are worked on
  constexpr uint32_t E = T == TY_F32 ? 4 : 2, W = 2 * E;
  static_assert(LG_SLICE == 8 * LG_NT, "8 logits a thread");
  const uint32_t i0 = 8 * tid, mine = i0 < n ? min(8u, n - i0) : 0u;
  struct Raw {
    uint32_t x[W], bits;
  };
  Raw sets[2];
  const auto load = [&](uint32_t t, Raw& to) {
    uint32_t(&raw)[W] = to.x;
    const uint64_t at = (uint64_t)s * a.n_rows + t;
    const char* src = static_cast<const char*>(a.in) + (at * a.in_stride + v0 + i0) * E;
    if (mine == 8 && (reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
#pragma unroll
      for (uint32_t i = 0; i < W / 4; ++i) {
        const rk_u32x4 u = reinterpret_cast<const rk_u32x4*>(src)[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) raw[4 * i + j] = u[j];
      }
    } else {
#pragma unroll
      for (uint32_t i = 0; i < W; ++i) raw[i] = 0;
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {
        if (i >= mine) continue;
        if constexpr (T == TY_F32) raw[i] = reinterpret_cast<const uint32_t*>(src)[i];
        else raw[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(src)[i] << (16 * (i & 1));
      }
    }
    // (8 bits are a byte of the row)
    to.bits = !a.mask ? 0xffu : mine ? reinterpret_cast<const uint8_t*>(a.mask + at * a.mask_stride)[(v0 + i0) >> 3] : 0u;
  };
  if (!SPARSE) {
    load(0, sets[0]);
    if (rows > 1) load(1, sets[1]);
  }
  for (uint32_t i = tid; i < LG_SLICE; i += LG_NT) {
    s_word[i] = 0;
    if (biases) s_bias[i] = 0;
  }
  __syncthreads();
  const uint32_t* history = a.history + s * a.history_stride;
  for (uint32_t i0 = tid; i0 < known; i0 += 4 * LG_NT) {
    uint32_t v[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) v[j] = i0 + j * LG_NT < known ? history[i0 + j * LG_NT] - v0 : ~0u;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      if (v[j] >= n) continue;
      atomicOr(&s_word[v[j]], LG_SEEN);
      if (i0 + j * LG_NT >= prompt) atomicAdd(&s_word[v[j]], 1u);
    }
  }
  if (tid < n_drafts) {
    const uint32_t v = row.drafts[tid] - v0;
    if (v < n) atomicOr(&s_word[v], LG_DRAFT);
  }
  for (uint32_t i = tid; i < biases; i += LG_NT) {
    const uint32_t v = a.bias_tokens[(size_t)s * a.bias_stride + i] - v0;
    if (v < n) {
      atomicOr(&s_word[v], LG_BIAS);
      atomicMax(&s_bias[v], i + 1);
    }
  }
  __syncthreads();
  if (!mine) return;
  uint32_t word[8], named = 0;
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) named |= word[i] = s_word[i0 + i];
  if (SPARSE && !named) return;
  if (SPARSE) {
    for (uint32_t t = 0; t < rows; ++t) {
      const uint64_t in = ((uint64_t)s * a.n_rows + t) * a.in_stride + v0 + i0;
      row.n_drafts = min(t, n_drafts);
#pragma unroll 1
      for (uint32_t i = 0; i < 8; ++i)
        if (const uint32_t w = s_word[i0 + i])
          store_from_f32<T>(a.out, in + i, lg_adjusted(load_as_f32<T>(a.in, in + i), w, v0 + i0 + i, s_bias[i0 + i], row));
    }
    return;
  }
  const auto finish = [&](uint32_t t, Raw& set) {
    row.n_drafts = min(t, n_drafts);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (T == TY_F32) x[i] = u2f(set.x[i]);
      else x[i] = from_bits16<T>((uint16_t)(set.x[i / 2] >> (16 * (i & 1))));
    }
    const uint32_t allowed = set.bits;
    if (t + 2 < rows) load(t + 2, set);
    if (named) {
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i)
        if (word[i]) x[i] = lg_adjusted(x[i], word[i], v0 + i0 + i, s_bias[i0 + i], row);
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) x[i] = allowed >> i & 1u ? x[i] : -INFINITY;
    const uint64_t out = ((uint64_t)s * a.n_rows + t) * a.out_stride + v0 + i0;
    char* dst = static_cast<char*>(a.out) + out * E;
    if (mine == 8 && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
      if constexpr (T == TY_F32) {
        f32x4v* q = reinterpret_cast<f32x4v*>(dst);
        q[0] = f32x4v{x[0], x[1], x[2], x[3]};
        q[1] = f32x4v{x[4], x[5], x[6], x[7]};
      } else {
        *reinterpret_cast<rk_u32x4*>(dst) = rk_pack8<T>(x);
      }
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i)
        if (i < mine) store_from_f32<T>(a.out, out + i, x[i]);
    }
  };
  for (uint32_t t = 0; t < rows; t += 2) {
    finish(t, sets[0]);
    if (t + 1 < rows) finish(t + 1, sets[1]);
  }
}

}  // namespace cm
