// kernels_logits.h -- logits before a token is drawn from them: penalties for repeated tokens, biases, masks.
//
//   x' = x / r where x > 0, else x r, for tokens that the row's text has (history and drafts before the row)
//   x' -= f count, x' -= p where count > 0, of the text's tokens behind the prompt (drafts are, always)
//   x' += bias of the token (the last one listed);  -infinity where the mask's bit is 0
// each step rounded in f32, the result once to the logits' type.
#pragma once
#include "kernels_paged.h"

namespace cm {

constexpr uint32_t LG_NT = 512;
constexpr uint32_t LG_BIASES = 32 * LG_NT;  // of a sequence at most
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
  uint32_t n_rows, vocab, slices, bias_stride, per, groups;  // per: rows of a workgroup
};

// What the lists say of a token (its word w, not 0) applied to its logit.
struct LogitsRow {
  float r, f, p;
  const uint32_t* drafts;
  uint32_t n_drafts;  // before the row
};
__device__ __forceinline__ float lg_adjusted(float x, uint32_t w, uint32_t token, uint32_t bias, const LogitsRow& a) {
  uint32_t count = w & LG_COUNT;
  if (w & LG_DRAFT)
    for (uint32_t j = 0; j < a.n_drafts; ++j) count += a.drafts[j] == token;
  if (count || (w & LG_SEEN)) x = x > 0.0f ? x / a.r : x * a.r;
  if (count) x = (x - a.f * (float)count) - a.p;
  if (w & LG_BIAS) x = x + u2f(bias);
  return x;
}

// One workgroup per (sequence, up to three rows, slice of the vocabulary): what the lists say of the slice's tokens goes
// to LDS once, then the rows, 8 logits a thread.  In place without a mask only the tokens that the lists name are read
// and written.  Bound: HBM where every logit is written, and the lists, which every slice reads from the L2.  32
// sequences of up to 6 rows of 151936 bf16 logits, 2000 tokens of history, 40 biases, masks: 28 us for 72 MB (20 us
// without the lists; f32 39 us for 143 MB); one row of 32000 in place: 4.8 us, a launch and three loads on each other.
template <int T, bool SPARSE>
__global__ __launch_bounds__(LG_NT) void k_adjust_logits(LogitsArgs a) {
  __shared__ uint32_t s_word[LG_SLICE];  // LG_COUNT: occurrences behind the prompt
  __shared__ uint32_t s_bias[LG_SLICE];  // where LG_BIAS is set: first the index of the last bias + 1, then its bits
  const uint32_t tid = threadIdx.x, unit = blockIdx.x / a.slices, v0 = (blockIdx.x - unit * a.slices) * LG_SLICE;
  const uint32_t s = unit / a.groups, t0 = (unit - s * a.groups) * a.per;  // first row
  const uint32_t n = min(LG_SLICE, a.vocab - v0);
  const uint32_t known = a.history ? (uint32_t)min((uint64_t)(a.history_lens ? a.history_lens[s] : ~0u), a.history_stride) : 0u;
  const uint32_t prompt = a.prompt_lens ? a.prompt_lens[s] : 0u;
  const uint32_t last = a.draft_lens ? min(a.draft_lens[s], a.n_rows - 1) : a.n_rows - 1;
  const uint32_t rows = min(last + 1, t0 + a.per), n_drafts = a.drafts && rows ? rows - 1 : 0u;
  if (t0 >= rows) return;
  const uint32_t biases = a.bias_tokens ? (a.bias_lens ? min(a.bias_lens[s], a.bias_stride) : a.bias_stride) : 0u;
  LogitsRow row{a.repetition ? a.repetition[s] : 1.0f, a.frequency ? a.frequency[s] : 0.0f,
                a.presence ? a.presence[s] : 0.0f, a.drafts + (size_t)s * (a.n_rows - 1), 0};
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
    load(t0, sets[0]);
    if (t0 + 1 < rows) load(t0 + 1, sets[1]);
  }
  // the first of the lists' tokens come before anything waits
  const uint32_t* history = a.history + s * a.history_stride;
  const uint32_t* bias_tokens = a.bias_tokens + (size_t)s * a.bias_stride;
  constexpr uint32_t H = 4;
  uint32_t v[H], draft = ~0u, bias = ~0u;
  const auto fetch = [&](uint32_t from) {
#pragma unroll
    for (uint32_t j = 0; j < H; ++j) v[j] = from + j * LG_NT < known ? history[from + j * LG_NT] - v0 : ~0u;
  };
  fetch(tid);
  if (tid < n_drafts) draft = row.drafts[tid] - v0;
  if (tid < biases) bias = bias_tokens[tid] - v0;
  for (uint32_t i = tid; i < LG_SLICE; i += LG_NT) {
    s_word[i] = 0;
    if (biases) s_bias[i] = 0;
  }
  __syncthreads();
  for (uint32_t from = tid; from < known; from += H * LG_NT) {
    if (from != tid) fetch(from);
#pragma unroll
    for (uint32_t j = 0; j < H; ++j) {
      if (v[j] >= n) continue;
      if (from + j * LG_NT < prompt) atomicOr(&s_word[v[j]], LG_SEEN);
      else atomicAdd(&s_word[v[j]], 1u);
    }
  }
  if (draft < n) atomicOr(&s_word[draft], LG_DRAFT);
  for (uint32_t i = tid; i < biases; i += LG_NT) {
    const uint32_t b = i == tid ? bias : bias_tokens[i] - v0;
    if (b >= n) continue;
    atomicOr(&s_word[b], LG_BIAS);
    atomicMax(&s_bias[b], i + 1);
  }
  __syncthreads();
  if (biases) {
    uint32_t wins = 0;  // entries i = tid + k LG_NT that are their token's last
    for (uint32_t k = 0; tid + k * LG_NT < biases; ++k) {
      if (k) bias = bias_tokens[tid + k * LG_NT] - v0;
      if (bias < n && s_bias[bias] == tid + k * LG_NT + 1) wins |= 1u << k;
    }
    __syncthreads();
    for (; wins; wins &= wins - 1) {
      const uint32_t i = tid + (__ffs(wins) - 1) * LG_NT;
      s_bias[bias_tokens[i] - v0] = f2u(a.bias_values[(size_t)s * a.bias_stride + i]);
    }
    __syncthreads();
  }
  if (!mine) return;
  uint32_t word[8], named = 0;
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) named |= word[i] = s_word[i0 + i];
  if (SPARSE && !named) return;
  if (SPARSE) {
    for (uint32_t t = t0; t < rows; ++t) {
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
  for (uint32_t t = t0; t < rows; t += 2) {
    finish(t, sets[0]);
    if (t + 1 < rows) finish(t + 1, sets[1]);
  }
}

}  // namespace cm
