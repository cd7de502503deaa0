// serving8.hip -- C entry points of serving over a paged cache held in 8 bits, of the bookkeeping of
// pages, and of logits before they are drawn from (include/camelid_hip.h).  As in serving.hip each call
// checks its arguments on the host, launches on the caller's stream, allocates nothing and waits for nothing,
// so it may be captured into a graph.
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../../include/camelid_hip.h"
#include "kernels_logits.h"
#include "kernels_paged8_attn.h"
#include "kernels_pages.h"
#include "serving_args.h"

namespace {

using cm::P8Sizes;
using cm::TY_E4M3;
using cm::TY_I8;

bool kv8_ok(uint32_t t) { return t == TY_I8 || t == TY_E4M3; }

// f with the integral constants of a head_dim, a cache type and a 16- or 32-bit type.
template <typename F>
void by_types(uint32_t hd, uint32_t kv_type, uint32_t type, F f) {
  const auto with_type = [&](auto d, auto k) {
    if (type == TY_F32) f(d, k, std::integral_constant<int, TY_F32>{});
    else if (type == TY_F16) f(d, k, std::integral_constant<int, TY_F16>{});
    else f(d, k, std::integral_constant<int, TY_BF16>{});
  };
  const auto with_kv = [&](auto d) {
    if (kv_type == TY_I8) with_type(d, std::integral_constant<int, TY_I8>{});
    else with_type(d, std::integral_constant<int, TY_E4M3>{});
  };
  if (hd == 64) with_kv(std::integral_constant<int, 64>{});
  else if (hd == 128) with_kv(std::integral_constant<int, 128>{});
  else with_kv(std::integral_constant<int, 256>{});
}

uint32_t log2_of(uint32_t power) {
  uint32_t n = 0;
  while ((1u << n) < power) ++n;
  return n;
}

template <int HD, int QT, int NR>
void p8_join(const cm::PaArgs& a, hipStream_t stream) {
  const uint32_t rows = a.n_new * a.group, sh = a.g.n_seqs * a.g.n_kv, cap = a.g.stride << a.g.shift;
  const auto join = [&](auto per, auto kernel) {
    const uint32_t row_groups = (rows + per.value - 1) / per.value;
    hipLaunchKernelGGL(kernel, dim3(sh * row_groups), dim3(cm::PA_NT), 0, stream, a, rows, row_groups, 0u, 8u);
  };
  if (NR > 2 || cap <= 16 * 4 * cm::P8_TILE || sh >= 256)
    join(std::integral_constant<uint32_t, cm::pj_parts(HD)>{}, cm::k_pa_join<HD, QT, NR, cm::pj_parts(HD)>);
  else
    join(std::integral_constant<uint32_t, 1>{}, cm::k_pa_join<HD, QT, NR, 1>);
}

bool p8_start(void (*kernel)(cm::P8Args), const cm::P8Args& p, const P8Sizes& z, uint32_t threads, size_t lds,
              hipStream_t stream) {
  if (lds > 64 * 1024) {
    const hipError_t st = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (st != hipSuccess) return cm::fail_global("paged8_attention", hipGetErrorString(st)) == 0;
  }
  hipLaunchKernelGGL(kernel, dim3(z.grid), dim3(threads), lds, stream, p);
  return true;
}

template <int HD, int KT, int QT, int NR>
bool p8_split(const cm::P8Args& p, const P8Sizes& z, hipStream_t stream) {
  const cm::PaArgs& a = p.a;
  // K and V that the batch's tables can hold, against the 256 MB of the memory-side cache (several row blocks read
  // them several times)
  const bool passing = z.blocks == 1 && ((uint64_t)a.g.n_seqs * a.g.n_kv * HD * 2 * a.g.stride << a.g.shift) > (256u << 20);
  constexpr size_t lds = (size_t)16 * NR * (4 * (HD + 4 + 2) + 2) * 4;
  if (!p8_start(passing ? cm::k_p8_split<HD, KT, QT, NR, true> : cm::k_p8_split<HD, KT, QT, NR, false>, p, z, cm::PA_NT, lds,
                stream))
    return false;
  if (z.join) p8_join<HD, QT, NR>(a, stream);
  return true;
}

template <int HD, int KT, int QT>
bool p8_launch(const cm::P8Args& p, const P8Sizes& z, hipStream_t stream) {
  if (z.prompt) {
    // 8 waves of 16 rows a workgroup hide each other's latency; f32 rows, which take twice the products, have enough
    // of those from some size on, and 4 waves of 32 rows read LDS half as often.  Heads of 128, f32: 3 prompts of up to
    // 1023 44.7 us with 8 waves and 56.1 with 4, 512 tokens at 1536 49 and 58, 2048 at 0 77 and 99, 1024 at 7168 267 and
    // 265, 512 at 32256 427 and 386, 4096 at 12288 1814 and 1628; bf16: 45 and 49, 46 and 48, 78 and 88, 223 and 232, 324
    // and 334, 1408 and 1407 (e4m3 1400 and 1347)
    const auto go = [&](auto waves) {
      return p8_start(cm::k_p8_prompt<HD, KT, QT, waves()>, p, z, 64 * waves(), cm::p8p_lds(HD), stream);
    };
    typedef std::integral_constant<int, 4> Four;
    typedef std::integral_constant<int, 8> Eight;
    bool ok;
    if constexpr (HD == 256) ok = go(Four{});
    else if constexpr (HD == 128 && QT == TY_F32) ok = z.tiles >= 16384 ? go(Four{}) : go(Eight{});
    else ok = go(Eight{});
    if (!ok) return false;
    if (z.join) p8_join<HD, QT, cm::p8p_rows(HD) / 16>(p.a, stream);
    return true;
  }
  if constexpr (HD <= 128)
    if (z.nr == 2) return p8_split<HD, KT, QT, 2>(p, z, stream);
  return p8_split<HD, KT, QT, 1>(p, z, stream);
}

}  // namespace

extern "C" {

int camelid_hip_paged8_rope_kv(const float* qkv, uint32_t n_seqs, uint32_t n_new, const uint32_t* new_lens,
                               uint32_t n_heads, uint32_t n_kv, uint32_t hd, uint32_t rope_dim, uint32_t split_half,
                               const float* cos_tab, const float* sin_tab, const float* q_norm, const float* k_norm,
                               float eps, void* q_out, uint32_t q_type, void* kc, void* vc, uint8_t* k_exp,
                               uint8_t* v_exp, uint32_t kv_type, uint32_t n_pages, uint32_t page_size,
                               const uint32_t* table, uint32_t table_stride, const uint32_t* lens, uint32_t* status,
                               void* stream) {
  const char* me = "paged8_rope_kv";
  if (!n_seqs || !n_new) return 0;
  if (!qkv || !q_out || !kc || !vc || !k_exp || !v_exp || !table || !lens) return cm::fail_global(me, "null argument");
  cm::Paged8 c{};
  const char* why;
  if (!paged_geometry(&c.g, n_seqs, n_kv, hd, n_pages, page_size, table, table_stride, lens, status, &why, 16))
    return cm::fail_global(me, why);
  if (!heads_ok(n_heads, n_kv)) return cm::fail_global(me, "n_heads must be a nonzero multiple of n_kv, at most 4096");
  if (rope_dim > hd || rope_dim % 2) return cm::fail_global(me, "rope_dim must be even and at most head_dim");
  if (rope_dim && (!cos_tab || !sin_tab)) return cm::fail_global(me, "null argument");
  if (!type_ok(q_type) || !kv8_ok(kv_type)) return cm::fail_global(me, "unknown type");
  if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(kc) || !aligned16(vc) || !aligned4(cos_tab) ||
      !aligned4(sin_tab) || !aligned4(q_norm) || !aligned4(k_norm) || !aligned4(new_lens))
    return cm::fail_global(me, "qkv, q_out and the cache must be 16-byte aligned, the rest 4-byte aligned");
  const bool whole = rope_dim == hd;
  const uint32_t roles = whole ? cm::r8_roles(hd, n_heads, n_kv) : n_heads + 2 * n_kv, blocks = cm::r8_blocks(n_new);
  const uint64_t grid = (uint64_t)n_seqs * blocks * roles;
  if (!grid_ok(grid, cm::R8_NT)) return cm::fail_global(me, "too many rows in one call");
  c.kc = static_cast<uint8_t*>(kc);
  c.vc = static_cast<uint8_t*>(vc);
  c.ke = k_exp;
  c.ve = v_exp;
  by_types(hd, kv_type, q_type, [&](auto d, auto k, auto q) {
    if (whole)
      hipLaunchKernelGGL((cm::k_paged8_rope_kv16<d(), q(), k()>), dim3((uint32_t)grid), dim3(cm::R8_NT), 0,
                         (hipStream_t)stream, c, qkv, n_new, new_lens, n_heads, split_half, cos_tab, sin_tab, q_norm,
                         k_norm, eps, q_out, roles, blocks);
    else
      hipLaunchKernelGGL((cm::k_paged8_rope_kv<q(), k()>), dim3((uint32_t)grid), dim3(cm::R8_NT), 0, (hipStream_t)stream,
                         c, qkv, n_new, new_lens, n_heads, rope_dim, split_half, cos_tab, sin_tab, q_norm, k_norm, eps,
                         q_out, blocks);
  });
  return launched(me);
}

int camelid_hip_paged8_read(const void* kc, const void* vc, const uint8_t* k_exp, const uint8_t* v_exp,
                            uint32_t kv_type, uint32_t n_pages, uint32_t page_size, uint32_t n_kv, uint32_t hd,
                            const uint32_t* table, uint32_t table_stride, const uint32_t* lens, uint32_t n_seqs,
                            void* k_out, void* v_out, uint32_t out_type, uint32_t out_positions, uint32_t* status,
                            void* stream) {
  const char* me = "paged8_read";
  if (!n_seqs || !out_positions) return 0;
  if (!kc || !vc || !k_exp || !v_exp || !table || !lens || !k_out || !v_out) return cm::fail_global(me, "null argument");
  cm::Paged8 c{};
  const char* why;
  if (!paged_geometry(&c.g, n_seqs, n_kv, hd, n_pages, page_size, table, table_stride, lens, status, &why, 16))
    return cm::fail_global(me, why);
  if (!type_ok(out_type) || !kv8_ok(kv_type)) return cm::fail_global(me, "unknown type");
  if (!aligned16(kc) || !aligned16(vc) || !aligned16(k_out) || !aligned16(v_out))
    return cm::fail_global(me, "the cache, k_out and v_out must be 16-byte aligned");
  const uint32_t reach = std::min(out_positions, table_stride * page_size);
  const uint32_t spans = (reach + cm::rd_span(hd) - 1) / cm::rd_span(hd);
  const uint64_t grid = (uint64_t)n_seqs * n_kv * spans * 2;
  if (!grid_ok(grid, cm::RD_NT)) return cm::fail_global(me, "too many positions in one call");
  c.kc = const_cast<uint8_t*>(static_cast<const uint8_t*>(kc));
  c.vc = const_cast<uint8_t*>(static_cast<const uint8_t*>(vc));
  c.ke = const_cast<uint8_t*>(k_exp);
  c.ve = const_cast<uint8_t*>(v_exp);
  by_types(hd, kv_type, out_type, [&](auto d, auto k, auto t) {
    hipLaunchKernelGGL((cm::k_paged8_read<d(), k(), t()>), dim3((uint32_t)grid), dim3(cm::RD_NT), 0, (hipStream_t)stream,
                       c, k_out, v_out, out_positions, spans);
  });
  return launched(me);
}

size_t camelid_hip_paged8_attention_workspace(uint32_t n_seqs, uint32_t n_new, uint32_t n_heads, uint32_t n_kv,
                                              uint32_t hd, uint32_t page_size, uint32_t table_stride) {
  if (!n_kv) return 0;
  return cm::p8_workspace(n_seqs, n_new, n_heads, n_kv, hd, (uint64_t)page_size * table_stride);
}

int camelid_hip_paged8_attention(const void* q, uint32_t q_type, uint32_t q_stride, uint32_t n_seqs, uint32_t n_new,
                                 const uint32_t* new_lens, uint32_t n_heads, uint32_t n_kv, uint32_t hd, const void* kc,
                                 const void* vc, const uint8_t* k_exp, const uint8_t* v_exp, uint32_t kv_type,
                                 uint32_t n_pages, uint32_t page_size, const uint32_t* table, uint32_t table_stride,
                                 const uint32_t* lens, float scale, void* out, uint32_t out_stride, void* workspace,
                                 size_t workspace_bytes, uint32_t* status, void* stream) {
  const char* me = "paged8_attention";
  if (!n_seqs || !n_new) return 0;
  if (!q || !kc || !vc || !k_exp || !v_exp || !table || !lens || !out || !workspace)
    return cm::fail_global(me, "null argument");
  cm::P8Args p{};
  cm::PaArgs& a = p.a;
  const char* why;
  if (!paged_geometry(&a.g, n_seqs, n_kv, hd, n_pages, page_size, table, table_stride, lens, status, &why, 16))
    return cm::fail_global(me, why);
  if (!heads_ok(n_heads, n_kv)) return cm::fail_global(me, "n_heads must be a nonzero multiple of n_kv, at most 4096");
  if (!type_ok(q_type) || !kv8_ok(kv_type)) return cm::fail_global(me, "unknown type");
  if (!std::isfinite(scale)) return cm::fail_global(me, "attention score scale must be finite");
  const uint32_t unit = q_type == TY_F32 ? 4 : 8;
  if (q_stride < (uint64_t)n_heads * hd || out_stride < (uint64_t)n_heads * hd || q_stride % unit || out_stride % unit)
    return cm::fail_global(me, "q_stride and out_stride must hold n_heads * head_dim elements and be whole 16-byte units");
  if (!aligned16(q) || !aligned16(out) || !aligned16(kc) || !aligned16(vc) || !aligned16(workspace) || !aligned4(new_lens))
    return cm::fail_global(me, "q, out, the cache and the workspace must be 16-byte aligned, the rest 4-byte aligned");
  if (workspace_bytes < camelid_hip_paged8_attention_workspace(n_seqs, n_new, n_heads, n_kv, hd, page_size, table_stride))
    return cm::fail_global(me, "workspace too small (camelid_hip_paged8_attention_workspace)");
  const uint64_t group = n_heads / n_kv;
  if (!grid_ok((uint64_t)n_seqs * n_kv * n_new * group, cm::PA_NT) || n_new * group * group >= (1ull << 32))
    return cm::fail_global(me, "too many rows in one call");
  const P8Sizes z = cm::p8_sizes(n_seqs, n_new, n_heads, n_kv, hd, (uint64_t)page_size * table_stride, q_type == TY_F32);
  if (!z.fits) return cm::fail_global(me, "n_seqs * n_kv * table_stride * page_size too large for one call");
  // (what the buffer is laid out by, apart from the formula that a caller is told)
  if (z.bytes > workspace_bytes) return cm::fail_global(me, "workspace too small for its own layout");
  // (every workgroup works the plan out from all lengths)
  if (n_seqs > 65535) return cm::fail_global(me, "at most 65535 sequences");
  char* ws = static_cast<char*>(workspace);
  p.ke = k_exp;
  p.ve = v_exp;
  a.kc = static_cast<const uint16_t*>(kc);
  a.vc = static_cast<const uint16_t*>(vc);
  a.q = q;
  a.new_lens = new_lens;
  a.out = out;
  a.part_ml = reinterpret_cast<float*>(ws);
  a.part_o = reinterpret_cast<float*>(ws + z.part_o);
  a.cuts = reinterpret_cast<uint2*>(ws + z.cuts);
  a.scale = scale;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.n_new = n_new;
  a.n_heads = n_heads;
  a.group = n_heads / n_kv;
  a.group_magic = a.group == 1 ? 0 : (uint32_t)(((1ull << 32) + a.group - 1) / a.group);
  a.at_once = z.at_once;
  a.blocks = z.blocks;
  a.part_rows = z.part_rows;
  bool ok = true;
  by_types(hd, kv_type, q_type, [&](auto d, auto k, auto t) {
    ok = p8_launch<d(), k(), t()>(p, z, (hipStream_t)stream);
  });
  return ok ? launched(me) : 1;
}

// ---- pages
static const char* pages_why(uint32_t n_seqs, uint32_t stride, uint32_t n_pages) {
  if (!n_pages || !stride) return "n_pages and table_stride must be nonzero";
  if (n_pages > 0x7fffffffu) return "n_pages must be below 2^31";
  if ((uint64_t)n_seqs * stride > 0x7fffffffull) return "n_seqs * table_stride must be below 2^31";
  if (n_seqs > (1u << 20)) return "n_seqs must be at most 2^20";
  return nullptr;
}
static bool page_size_ok(uint32_t p) { return p >= 8 && p <= 4096 && !(p & (p - 1)); }
static const char* const PAGE_SIZE = "page_size must be a power of two in 8..=4096";
static uint32_t page_chunks(uint32_t n_pages) { return (uint32_t)(((uint64_t)n_pages + cm::PG_CHUNK - 1) / cm::PG_CHUNK); }

size_t camelid_hip_pages_reserve_workspace(uint32_t n_seqs, uint32_t n_pages) {
  return 4 * up256((size_t)n_seqs * 4) + up256((size_t)page_chunks(n_pages) * 4) + up256((size_t)n_pages * 4);
}

int camelid_hip_pages_reserve(uint32_t* table, uint32_t table_stride, uint32_t* held, uint32_t n_seqs,
                              const uint32_t* first, const uint32_t* lens, uint32_t page_size, uint32_t* refs,
                              uint32_t n_pages, uint32_t* pairs, uint32_t max_pairs, uint32_t* n_pairs,
                              uint32_t* granted, void* workspace, size_t workspace_bytes, uint32_t* status,
                              void* stream) {
  const char* me = "pages_reserve";
  if (!n_seqs) return 0;
  if (!table || !held || !lens || !refs || !workspace || (first && !n_pairs) || (max_pairs && !pairs))
    return cm::fail_global(me, "null argument");
  if (const char* why = pages_why(n_seqs, table_stride, n_pages)) return cm::fail_global(me, why);
  if (!page_size_ok(page_size)) return cm::fail_global(me, PAGE_SIZE);
  if (!aligned16(workspace) || !aligned4(table) || !aligned4(held) || !aligned4(first) || !aligned4(lens) ||
      !aligned4(refs) || !aligned4(pairs) || !aligned4(n_pairs) || !aligned4(granted) || !aligned4(status))
    return cm::fail_global(me, "the workspace must be 16-byte aligned, the rest 4-byte aligned");
  if (workspace_bytes < camelid_hip_pages_reserve_workspace(n_seqs, n_pages))
    return cm::fail_global(me, "workspace too small (camelid_hip_pages_reserve_workspace)");
  cm::PagesArgs a{};
  a.table = table;
  a.held = held;
  a.first = first;
  a.lens = lens;
  a.refs = refs;
  a.pairs = pairs;
  a.n_pairs = n_pairs;
  a.granted = granted;
  a.status = status;
  const size_t row = up256((size_t)n_seqs * 4) / 4;
  a.need = static_cast<uint32_t*>(workspace);
  a.cows = a.need + row;
  a.before = a.cows + row;
  a.cows_before = a.before + row;
  a.chunk = a.cows_before + row;
  a.chunks = page_chunks(n_pages);
  a.free_list = a.chunk + up256((size_t)a.chunks * 4) / 4;
  a.stride = table_stride;
  a.n_seqs = n_seqs;
  a.shift = log2_of(page_size);
  a.n_pages = n_pages;
  a.max_pairs = max_pairs;
  if (n_seqs <= cm::PG_ONE_SEQS && n_pages <= cm::PG_ONE_PAGES && (uint64_t)n_seqs * table_stride <= cm::PG_ONE_ENTRIES) {
    hipLaunchKernelGGL(cm::k_pages_reserve, dim3(1), dim3(cm::PG_PLAN_NT), 0, (hipStream_t)stream, a);
    return launched(me);
  }
  hipLaunchKernelGGL(cm::k_pages_shrink, dim3(n_seqs), dim3(cm::PG_NT), 0, (hipStream_t)stream, a);
  hipLaunchKernelGGL(cm::k_pages_count, dim3(n_seqs + a.chunks), dim3(cm::PG_NT), 0, (hipStream_t)stream, a);
  hipLaunchKernelGGL(cm::k_pages_plan, dim3(a.chunks + 1), dim3(cm::PG_PLAN_NT), 0, (hipStream_t)stream, a);
  hipLaunchKernelGGL(cm::k_pages_grant, dim3(n_seqs), dim3(cm::PG_NT), 0, (hipStream_t)stream, a);
  return launched(me);
}

int camelid_hip_pages_fork(uint32_t* table, uint32_t table_stride, uint32_t* held, uint32_t n_seqs,
                           const uint32_t* parents, const uint32_t* children, uint32_t n_forks, const uint32_t* lens,
                           uint32_t page_size, uint32_t* refs, uint32_t n_pages, uint32_t* status, void* stream) {
  const char* me = "pages_fork";
  if (!n_forks) return 0;
  if (!table || !held || !parents || !children || !refs) return cm::fail_global(me, "null argument");
  if (const char* why = pages_why(n_seqs, table_stride, n_pages)) return cm::fail_global(me, why);
  if (!page_size_ok(page_size)) return cm::fail_global(me, PAGE_SIZE);
  if (n_forks > n_seqs) return cm::fail_global(me, "more forks than sequences");
  if (!aligned4(table) || !aligned4(held) || !aligned4(parents) || !aligned4(children) || !aligned4(lens) ||
      !aligned4(refs) || !aligned4(status))
    return cm::fail_global(me, "the buffers must be 4-byte aligned");
  hipLaunchKernelGGL(cm::k_pages_fork, dim3(n_forks), dim3(cm::PG_NT), 0, (hipStream_t)stream, table, table_stride, held,
                     n_seqs, parents, children, n_forks, lens, log2_of(page_size), refs, n_pages, status);
  return launched(me);
}

size_t camelid_hip_pages_compact_workspace(uint32_t n_pages) {
  return up256((size_t)page_chunks(n_pages) * 4) + 4 * up256((size_t)n_pages * 4);
}

int camelid_hip_pages_compact(const uint32_t* table, uint32_t table_stride, const uint32_t* held, uint32_t n_seqs,
                              const uint32_t* refs, uint32_t n_pages, uint32_t* table_out, uint32_t* refs_out,
                              uint32_t* pairs, uint32_t max_pairs, uint32_t* n_pairs, uint32_t* extent,
                              void* workspace, size_t workspace_bytes, uint32_t* status, void* stream) {
  const char* me = "pages_compact";
  if (!table || !held || !refs || !table_out || !refs_out || !n_pairs || !workspace || (max_pairs && !pairs))
    return cm::fail_global(me, "null argument");
  if (const char* why = pages_why(n_seqs, table_stride, n_pages)) return cm::fail_global(me, why);
  if (!aligned16(workspace) || !aligned4(table) || !aligned4(held) || !aligned4(refs) || !aligned4(table_out) ||
      !aligned4(refs_out) || !aligned4(pairs) || !aligned4(n_pairs) || !aligned4(extent) || !aligned4(status))
    return cm::fail_global(me, "the workspace must be 16-byte aligned, the rest 4-byte aligned");
  if (workspace_bytes < camelid_hip_pages_compact_workspace(n_pages))
    return cm::fail_global(me, "workspace too small (camelid_hip_pages_compact_workspace)");
  cm::CompactArgs a{};
  a.table = table;
  a.held = held;
  a.refs = refs;
  a.table_out = table_out;
  a.refs_out = refs_out;
  a.pairs = pairs;
  a.n_pairs = n_pairs;
  a.extent = extent;
  a.status = status;
  a.chunks = page_chunks(n_pages);
  const size_t row = up256((size_t)n_pages * 4) / 4;
  a.chunk = static_cast<uint32_t*>(workspace);
  a.old = a.chunk + up256((size_t)a.chunks * 4) / 4;
  a.rank = a.old + row;
  a.holes = a.rank + row;
  a.highs = a.holes + row;
  a.stride = table_stride;
  a.n_seqs = n_seqs;
  a.n_pages = n_pages;
  a.max_pairs = max_pairs;
  if (n_pages <= cm::PG_COUNT_PAGES) {
    hipLaunchKernelGGL(cm::k_compact_list<true>, dim3(a.chunks), dim3(cm::PG_PLAN_NT), 0, (hipStream_t)stream, a);
  } else {
    hipLaunchKernelGGL(cm::k_compact_count, dim3(a.chunks), dim3(cm::PG_NT), 0, (hipStream_t)stream, a);
    hipLaunchKernelGGL(cm::k_compact_list<false>, dim3(a.chunks), dim3(cm::PG_PLAN_NT), 0, (hipStream_t)stream, a);
  }
  hipLaunchKernelGGL(cm::k_compact_move, dim3(a.chunks + n_seqs), dim3(cm::PG_PLAN_NT), 0, (hipStream_t)stream, a);
  return launched(me);
}

int camelid_hip_pages_copy(void* const* buffers, const size_t* page_bytes, uint32_t n_buffers, uint32_t n_pages,
                           const uint32_t* pairs, uint32_t max_pairs, const uint32_t* n_pairs, uint32_t* status,
                           void* stream) {
  const char* me = "pages_copy";
  if (!n_buffers || !max_pairs) return 0;
  if (!buffers || !page_bytes || !pairs) return cm::fail_global(me, "null argument");
  if (!n_pages || n_pages > 0x7fffffffu) return cm::fail_global(me, "n_pages must be in 1 to 2^31 - 1");
  if (!aligned4(pairs) || !aligned4(n_pairs) || !aligned4(status))
    return cm::fail_global(me, "pairs, n_pairs and status must be 4-byte aligned");
  for (uint32_t i = 0; i < n_buffers; ++i)
    if (!buffers[i] && page_bytes[i]) return cm::fail_global(me, "null argument");
  // more than the caches hold passes them by (compacting 2048 pages of 256 KB: 56 us against 61), pages of which
  // one has just been read and the other is about to be do not (48 pages of 256 KB: 11 us against 18)
  uint64_t total = 0;
  for (uint32_t i = 0; i < n_buffers; ++i) total += page_bytes[i];
  const auto kernel = total * max_pairs >= (128u << 20) ? cm::k_pages_copy<true> : cm::k_pages_copy<false>;
  for (uint32_t i = 0; i < n_buffers; i += cm::PC_BUFFERS) {
    cm::PageCopyArgs a{};
    a.n_buffers = std::min(cm::PC_BUFFERS, n_buffers - i);
    for (uint32_t j = 0; j < a.n_buffers; ++j) {
      a.buffer[j] = static_cast<uint8_t*>(buffers[i + j]);
      a.bytes[j] = page_bytes[i + j];
    }
    a.pairs = pairs;
    a.n_pairs = n_pairs;
    a.status = status;
    a.max_pairs = max_pairs;
    a.n_pages = n_pages;
    hipLaunchKernelGGL(kernel, dim3(std::min(max_pairs, 512u) * a.n_buffers), dim3(cm::PC_NT), 0,
                       (hipStream_t)stream, a);
  }
  return launched(me);
}

// ---- logits
int camelid_hip_adjust_logits(const void* logits, size_t in_stride, void* out, size_t out_stride, uint32_t logits_type,
                              uint32_t n_seqs, uint32_t n_rows, uint32_t vocab, const uint32_t* history,
                              size_t history_stride, const uint32_t* history_lens, const uint32_t* prompt_lens,
                              const uint32_t* draft_tokens, const uint32_t* draft_lens, const float* repetition,
                              const float* frequency, const float* presence, const uint32_t* bias_tokens,
                              const float* bias_values, uint32_t bias_stride, const uint32_t* bias_lens,
                              const uint32_t* mask, size_t mask_stride, void* stream) {
  const char* me = "adjust_logits";
  if (!n_seqs || !n_rows) return 0;
  if (!logits || !out || (bias_tokens && !bias_values)) return cm::fail_global(me, "null argument");
  if (n_rows > 32) return cm::fail_global(me, "at most 32 rows per sequence");
  if (!vocab || vocab > (1u << 24)) return cm::fail_global(me, "vocab must be in 1..=2^24");
  if (!type_ok(logits_type)) return cm::fail_global(me, "unknown type");
  if (in_stride < vocab || out_stride < vocab) return cm::fail_global(me, "the strides must hold vocab elements");
  if (out == logits && in_stride != out_stride) return cm::fail_global(me, "in place the strides must be equal");
  if (mask && mask_stride < (vocab + 31) / 32) return cm::fail_global(me, "mask_stride must hold vocab bits");
  if (history && history_stride > (1u << 28)) return cm::fail_global(me, "history_stride must be at most 2^28");
  if (bias_tokens && bias_stride > cm::LG_BIASES) return cm::fail_global(me, "bias_stride must be at most 16384");
  const uintptr_t unit = logits_type == TY_F32 ? 3 : 1;
  if (((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(out)) & unit) || !aligned4(history) ||
      !aligned4(history_lens) || !aligned4(prompt_lens) || !aligned4(draft_tokens) || !aligned4(draft_lens) ||
      !aligned4(repetition) || !aligned4(frequency) || !aligned4(presence) || !aligned4(bias_tokens) ||
      !aligned4(bias_values) || !aligned4(bias_lens) || !aligned4(mask))
    return cm::fail_global(me, "the buffers must be aligned to their elements");
  cm::LogitsArgs a{logits, out, history, history_lens, prompt_lens, draft_tokens, draft_lens, repetition, frequency,
                   presence, bias_tokens, bias_values, bias_lens, mask, in_stride, out_stride, history_stride,
                   mask_stride, n_rows, vocab, (vocab + cm::LG_SLICE - 1) / cm::LG_SLICE, bias_stride, 0, 0};
  // rows of a workgroup: up to three, so that sequences with many do not keep the others waiting (32 x 6 of 151936, f32
  // 44.1 us with all, 38.2 with three, 43.4 with one, which reads the lists for each)
  a.per = std::min(n_rows, 3u);
  a.groups = (n_rows + a.per - 1) / a.per;
  const uint64_t grid = (uint64_t)n_seqs * a.groups * a.slices;
  if (!grid_ok(grid, cm::LG_NT)) return cm::fail_global(me, "too many rows in one call");
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((uint32_t)grid), dim3(cm::LG_NT), 0, (hipStream_t)stream, a);
  };
  const auto typed = [&](auto sparse) {
    if (logits_type == TY_F32) go(cm::k_adjust_logits<TY_F32, sparse()>);
    else if (logits_type == TY_F16) go(cm::k_adjust_logits<TY_F16, sparse()>);
    else go(cm::k_adjust_logits<TY_BF16, sparse()>);
  };
  if (out == logits && !mask) typed(std::true_type{});
  else typed(std::false_type{});
  return launched(me);
}

}  // extern "C"
