// serving_args.h -- what the argument checks of the serving calls share.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

#include "errors.h"
#include "kernels_paged.h"
#include "launch_sizes.h"

namespace {

using cm::TY_BF16;
using cm::TY_F16;
using cm::TY_F32;
using cm::grid_ok;
using cm::up256;

inline int launched(const char* what) {
  const hipError_t st = hipGetLastError();
  return st == hipSuccess ? 0 : cm::fail_global(what, hipGetErrorString(st));
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

// Cache geometry, pages of `least` positions or more; false: the reason why it is refused in *why.
inline bool paged_geometry(cm::Paged* g, uint32_t n_seqs, uint32_t n_kv, uint32_t hd, uint32_t n_pages, uint32_t page_size,
                    const uint32_t* table, uint32_t stride, const uint32_t* lens, uint32_t* status, const char** why,
                    uint32_t least = 8) {
  *why = nullptr;
  if (hd != 64 && hd != 128 && hd != 256) *why = "head_dim must be 64, 128 or 256";
  else if (!n_kv || n_kv > 1024) *why = "n_kv must be in 1..=1024";
  else if (page_size < least || page_size > 4096 || (page_size & (page_size - 1)))
    *why = least == 8 ? "page_size must be a power of two in 8..=4096" : "page_size must be a power of two in 16..=4096";
  else if (!n_pages || !stride) *why = "n_pages and table_stride must be nonzero";
  else if ((uint64_t)stride * page_size > (1u << 24)) *why = "table_stride * page_size must be at most 2^24 positions";
  else if ((uint64_t)n_seqs * n_kv > (1u << 20)) *why = "n_seqs * n_kv must be at most 2^20";
  else if (!aligned4(table) || !aligned4(lens) || !aligned4(status)) *why = "table, lens and status must be 4-byte aligned";
  if (*why) return false;
  uint32_t shift = 3;
  while ((1u << shift) < page_size) ++shift;
  *g = cm::Paged{table, lens, status, stride, n_pages, shift, n_kv, hd, n_seqs};
  return true;
}

inline bool heads_ok(uint32_t n_heads, uint32_t n_kv) { return n_kv && n_heads && n_heads % n_kv == 0 && n_heads <= 4096; }
inline bool type_ok(uint32_t t) { return t == TY_F32 || t == TY_F16 || t == TY_BF16; }

}  // namespace
