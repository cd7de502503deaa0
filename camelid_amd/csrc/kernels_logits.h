// kernels_logits.h -- logits before a token is drawn from them: penalties for repeated tokens, biases, masks.
//
//   x' = x / r where x > 0, else x r, for tokens that the row's text has (history and drafts before the row)
//   x' -= f count, x' -= p where count > 0, of the text's tokens behind the prompt
//   x' += bias of the token (the last one listed);  -infinity where the mask's bit is 0
// each step rounded in f32, the result once to the logits' type.
#pragma once
#include "kernels_paged.h"

namespace cm {

constexpr uint32_t LG_NT = 256;
constexpr uint32_t LG_SLICE = 2048;  // tokens of a workgroup
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

// One workgroup per (sequence, slice of the vocabulary): what the lists say of the slice's tokens goes to LDS
// once, then the sequence's rows.
template <int T>
__global__ __launch_bounds__(LG_NT) void k_adjust_logits(LogitsArgs a) {
  __shared__ uint32_t s_word[LG_SLICE];  // LG_COUNT: occurrences behind the prompt
  __shared__ uint32_t s_bias[LG_SLICE];  // index of the last bias + 1
  const uint32_t tid = threadIdx.x, s = blockIdx.x / a.slices, v0 = (blockIdx.x - s * a.slices) * LG_SLICE;
  const uint32_t n = min(LG_SLICE, a.vocab - v0);
  for (uint32_t i = tid; i < LG_SLICE; i += LG_NT) s_word[i] = s_bias[i] = 0;
  __syncthreads();
  const uint32_t known = a.history ? (uint32_t)min((uint64_t)(a.history_lens ? a.history_lens[s] : ~0u), a.history_stride) : 0u;
  const uint32_t prompt = a.prompt_lens ? a.prompt_lens[s] : 0u;
  const uint32_t n_drafts = a.drafts ? min(a.draft_lens ? a.draft_lens[s] : a.n_rows - 1, a.n_rows - 1) : 0u;
  const uint32_t rows = (a.draft_lens ? min(a.draft_lens[s], a.n_rows - 1) : a.n_rows - 1) + 1;
  const uint32_t* drafts = a.drafts + (size_t)s * (a.n_rows - 1);
  for (uint32_t i = tid; i < known; i += LG_NT) {
    const uint32_t v = a.history[s * a.history_stride + i] - v0;
    if (v < n) {
      atomicOr(&s_word[v], LG_SEEN);
      if (i >= prompt) atomicAdd(&s_word[v], 1u);
    }
  }
  if (tid < n_drafts) {
    const uint32_t v = drafts[tid] - v0;
    if (v < n) atomicOr(&s_word[v], LG_DRAFT);
  }
  const uint32_t biases = a.bias_tokens ? (a.bias_lens ? min(a.bias_lens[s], a.bias_stride) : a.bias_stride) : 0u;
  for (uint32_t i = tid; i < biases; i += LG_NT) {
    const uint32_t v = a.bias_tokens[(size_t)s * a.bias_stride + i] - v0;
    if (v < n) {
      atomicOr(&s_word[v], LG_BIAS);
      atomicMax(&s_bias[v], i + 1);
    }
  }
  __syncthreads();
  const float r = a.repetition ? a.repetition[s] : 1.0f, f = a.frequency ? a.frequency[s] : 0.0f;
  const float p = a.presence ? a.presence[s] : 0.0f;
  for (uint32_t t = 0; t < rows; ++t) {
    const uint64_t row = (uint64_t)s * a.n_rows + t;
    for (uint32_t i = tid; i < n; i += LG_NT) {
      const uint32_t w = s_word[i];
      float x = load_as_f32<T>(a.in, row * a.in_stride + v0 + i);
      if (w) {
        uint32_t count = w & LG_COUNT;
        bool seen = w & LG_SEEN;
        if (w & LG_DRAFT)
          for (uint32_t j = 0; j < min(t, n_drafts); ++j)
            if (drafts[j] == v0 + i) {
              ++count;
              seen = true;
            }
        if (seen) x = x > 0.0f ? x / r : x * r;
        if (count) x = (x - f * (float)count) - p;
        if (w & LG_BIAS) x = x + a.bias_values[(size_t)s * a.bias_stride + s_bias[i] - 1];
      }
      if (a.mask && !(a.mask[row * a.mask_stride + ((v0 + i) >> 5)] >> ((v0 + i) & 31u) & 1u)) x = -INFINITY;
      store_from_f32<T>(a.out, row * a.out_stride + v0 + i, x);
    }
  }
}

}  // namespace cm
