// serving.hip -- C entry points of batched serving over a paged cache (include/camelid_hip.h):
// RoPE + store, attention of new tokens, eviction, and verification of drafts by given random
// numbers.  Each call checks its arguments on the host, launches on the caller's stream, allocates
// nothing and waits for nothing, so it may be captured into a graph.
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../../include/camelid_hip.h"
#include "errors.h"
#include "kernels_paged_attn.h"
#include "kernels_verify.h"

namespace {

using cm::TY_BF16;
using cm::TY_F16;
using cm::TY_F32;

int launched(const char* what) {
  const hipError_t st = hipGetLastError();
  return st == hipSuccess ? 0 : cm::fail_global(what, hipGetErrorString(st));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
// A launch holds at most 2^32 - 1 threads.
bool grid_ok(uint64_t groups, uint32_t threads) { return groups * threads <= 0xffffffffull; }
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// Cache geometry; null: the reason why it is refused in *why.
bool paged_geometry(cm::Paged* g, uint32_t n_seqs, uint32_t n_kv, uint32_t hd, uint32_t n_pages, uint32_t page_size,
                    const uint32_t* table, uint32_t stride, const uint32_t* lens, uint32_t* status, const char** why) {
  *why = nullptr;
  if (hd != 64 && hd != 128 && hd != 256) *why = "head_dim must be 64, 128 or 256";
  else if (!n_kv || n_kv > 1024) *why = "n_kv must be in 1..=1024";
  else if (page_size < 8 || page_size > 4096 || (page_size & (page_size - 1)))
    *why = "page_size must be a power of two in 8..=4096";
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

bool heads_ok(uint32_t n_heads, uint32_t n_kv) { return n_kv && n_heads && n_heads % n_kv == 0 && n_heads <= 4096; }
bool type_ok(uint32_t t) { return t == TY_F32 || t == TY_F16 || t == TY_BF16; }
bool kv_type_ok(uint32_t t) { return t == TY_F16 || t == TY_BF16; }

// What a call of the attention needs: row blocks of 16 * nr query rows, workgroups, workspace.
struct PaSizes {
  uint32_t nr, blocks, part_rows, at_once, grid;
  bool join;                                  // some segment may be cut, or weights are kept
  bool fits;                                  // the plan's 32-bit counts hold
  size_t part_o, cuts, stats, scores, bytes;  // offsets of the workspace's parts, its size
};

PaSizes pa_sizes(uint64_t n_seqs, uint64_t n_new, uint64_t n_heads, uint64_t n_kv, uint32_t hd, uint64_t cap,
                 bool weights) {
  PaSizes z;
  const uint64_t rows = n_new * (n_heads / n_kv), cap_tiles = (cap + cm::PA_TILE - 1) / cm::PA_TILE;
  z.nr = rows > 16 && hd <= 128 ? 2 : 1;
  z.blocks = (uint32_t)((rows + 16 * z.nr - 1) / (16 * z.nr));
  z.part_rows = (uint32_t)std::min<uint64_t>(rows, 16 * z.nr);
  // 256 CUs; a seventh less, since cutting every segment evenly makes some more pieces
  z.at_once = 256 * cm::pa_per_cu((int)hd, (int)z.nr) * 7 / 8;
  const uint64_t segments = n_seqs * n_kv * z.blocks, most = 2048;
  // a segment has at most ceil(its tiles / 4) pieces, all of them together at most 2048 and one each
  const uint64_t pieces = std::min(most + segments, segments * ((cap_tiles + 3) / 4));
  z.fits = segments * cap_tiles < (1ull << 31) && grid_ok(pieces, cm::PA_NT);
  z.grid = (uint32_t)pieces;
  z.join = cap_tiles > 4 || weights;
  // cut segments have more tiles than the target: at most 2048 of them, twice as many pieces
  const size_t slots = cap_tiles > 4 ? (size_t)std::min(2 * most, pieces) : 0;
  z.part_o = up256(slots * z.part_rows * 8);
  z.cuts = z.part_o + up256(slots * z.part_rows * hd * 4);
  z.stats = z.cuts + up256(segments * 8);
  z.scores = z.stats + (weights ? up256(n_seqs * n_kv * rows * 8) : 0);
  z.bytes = z.scores + (weights ? up256(n_seqs * n_kv * rows * cap * 4) : 0);
  return z;
}

template <int HD, int KT, int QT, int NR>
bool pa_launch(const cm::PaArgs& a, const PaSizes& z, hipStream_t stream) {
  // K and V that the batch's tables can hold, against the 256 MB of the memory-side cache (several row
  // blocks read them several times).  One new token, 32 query heads, hd 128, f16: plain loads 28.9 us and
  // streaming loads 31.6 for 134 MB read again and again, 33.9 and 32.2 for 8 such caches in turn; 45.6 and
  // 47.9 for 269 MB, 54.9 and 49.7 for 4 of them; 101.8 and 91.7 for 538 MB
  const bool passing = z.blocks == 1 && ((uint64_t)a.g.n_seqs * a.g.n_kv * HD * 4 * a.g.stride << a.g.shift) > (256u << 20);
  const auto split = passing ? cm::k_pa_split<HD, KT, QT, NR, true> : cm::k_pa_split<HD, KT, QT, NR, false>;
  constexpr size_t lds = (size_t)16 * NR * (4 * (HD + 4 + 2) + 1) * 4;
  if (lds > 64 * 1024) {
    const hipError_t st = hipFuncSetAttribute(reinterpret_cast<const void*>(split),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (st != hipSuccess) return cm::fail_global("paged_attention", hipGetErrorString(st)) == 0;
  }
  hipLaunchKernelGGL(split, dim3(z.grid), dim3(cm::PA_NT), lds, stream, a);
  if (!z.join) return true;
  // tables of up to 16 pieces, or many segments (which make larger pieces): a row to one group of lanes (16x1100
  // with 5 drafts: 6.6 us against 7.6 with a workgroup a row, 83x2152 with 5: 123 us for the call against
  // 135); few longer ones: a workgroup a row (1x8199: 4.1 us against 6.6)
  const uint32_t rows = a.n_new * a.group, sh = a.g.n_seqs * a.g.n_kv;
  // weights: positions of a workgroup 256, or 64 with the rows dealt to its four waves where that makes less than
  // two workgroups a CU (5x940, 64 rows: 19.1 us for the call against 22.7; 1x46046, 56 rows: 65 against 47)
  const uint32_t cap = a.g.stride << a.g.shift, span_bits = (uint64_t)sh * ((cap + 255) >> 8) >= 512 ? 8 : 6;
  const uint32_t spans = a.weights ? (cap + (1u << span_bits) - 1) >> span_bits : 0;
  const auto join = [&](auto per, auto kernel) {
    const uint32_t row_groups = (rows + per.value - 1) / per.value;
    hipLaunchKernelGGL(kernel, dim3(sh * (row_groups + spans)), dim3(cm::PA_NT), 0, stream, a, rows, row_groups, spans,
                       span_bits);
  };
  if (cap <= 16 * 4 * cm::PA_TILE || sh >= 256)
    join(std::integral_constant<uint32_t, cm::pj_parts(HD)>{}, cm::k_pa_join<HD, QT, NR, cm::pj_parts(HD)>);
  else
    join(std::integral_constant<uint32_t, 1>{}, cm::k_pa_join<HD, QT, NR, 1>);
  return true;
}

template <int KT, int QT>
bool pa_launch_hd(const cm::PaArgs& a, const PaSizes& z, hipStream_t stream) {
  if (a.g.hd == 64) return z.nr == 1 ? pa_launch<64, KT, QT, 1>(a, z, stream) : pa_launch<64, KT, QT, 2>(a, z, stream);
  if (a.g.hd == 128) return z.nr == 1 ? pa_launch<128, KT, QT, 1>(a, z, stream) : pa_launch<128, KT, QT, 2>(a, z, stream);
  return pa_launch<256, KT, QT, 1>(a, z, stream);
}

}  // namespace

extern "C" {

int camelid_hip_paged_rope_kv(const float* qkv, uint32_t n_seqs, uint32_t n_new, const uint32_t* new_lens,
                              uint32_t n_heads, uint32_t n_kv, uint32_t hd, uint32_t rope_dim, uint32_t split_half,
                              const float* cos_tab, const float* sin_tab, const float* q_norm, const float* k_norm,
                              float eps, void* q_out, uint32_t q_type, void* kc, void* vc, uint32_t kv_type,
                              uint32_t n_pages, uint32_t page_size, const uint32_t* table, uint32_t table_stride,
                              const uint32_t* lens, uint32_t* status, void* stream) {
  const char* me = "paged_rope_kv";
  if (!n_seqs || !n_new) return 0;
  if (!qkv || !q_out || !kc || !vc || !table || !lens) return cm::fail_global(me, "null argument");
  cm::Paged g;
  const char* why;
  if (!paged_geometry(&g, n_seqs, n_kv, hd, n_pages, page_size, table, table_stride, lens, status, &why))
    return cm::fail_global(me, why);
  if (!heads_ok(n_heads, n_kv)) return cm::fail_global(me, "n_heads must be a nonzero multiple of n_kv, at most 4096");
  if (rope_dim > hd || rope_dim % 2) return cm::fail_global(me, "rope_dim must be even and at most head_dim");
  if (rope_dim && (!cos_tab || !sin_tab)) return cm::fail_global(me, "null argument");
  if (!type_ok(q_type) || !kv_type_ok(kv_type)) return cm::fail_global(me, "unknown type");
  if (q_type != TY_F32 && q_type != kv_type)
    return cm::fail_global(me, "16-bit q rows must have the cache's type");
  if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(kc) || !aligned16(vc) || !aligned4(cos_tab) ||
      !aligned4(sin_tab) || !aligned4(q_norm) || !aligned4(k_norm) || !aligned4(new_lens))
    return cm::fail_global(me, "qkv, q_out and the cache must be 16-byte aligned, the rest 4-byte aligned");
  const uint64_t rows = (uint64_t)n_seqs * n_new * (n_heads + n_kv);
  if (!grid_ok(rows, 64)) return cm::fail_global(me, "too many rows in one call");
  if (rope_dim == hd) {
    const uint32_t roles = cm::rk_roles(hd, n_heads, n_kv), granules = cm::rk_granules(n_new);
    const uint64_t grid = (uint64_t)n_seqs * granules * roles;
    if (!grid_ok(grid, cm::RK_NT)) return cm::fail_global(me, "too many rows in one call");
    const auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((uint32_t)grid), dim3(cm::RK_NT), 0, (hipStream_t)stream, g, qkv, n_new, new_lens,
                         n_heads, split_half, cos_tab, sin_tab, q_norm, k_norm, eps, q_out, static_cast<uint16_t*>(kc),
                         static_cast<uint16_t*>(vc), roles, granules);
    };
    const auto typed = [&](auto f32_f16, auto f16, auto f32_bf16, auto bf16) {
      if (kv_type == TY_F16) {
        if (q_type == TY_F32) go(f32_f16);
        else go(f16);
      } else {
        if (q_type == TY_F32) go(f32_bf16);
        else go(bf16);
      }
    };
    if (hd == 64)
      typed(cm::k_paged_rope_kv8<64, TY_F32, TY_F16>, cm::k_paged_rope_kv8<64, TY_F16, TY_F16>,
            cm::k_paged_rope_kv8<64, TY_F32, TY_BF16>, cm::k_paged_rope_kv8<64, TY_BF16, TY_BF16>);
    else if (hd == 128)
      typed(cm::k_paged_rope_kv8<128, TY_F32, TY_F16>, cm::k_paged_rope_kv8<128, TY_F16, TY_F16>,
            cm::k_paged_rope_kv8<128, TY_F32, TY_BF16>, cm::k_paged_rope_kv8<128, TY_BF16, TY_BF16>);
    else
      typed(cm::k_paged_rope_kv8<256, TY_F32, TY_F16>, cm::k_paged_rope_kv8<256, TY_F16, TY_F16>,
            cm::k_paged_rope_kv8<256, TY_F32, TY_BF16>, cm::k_paged_rope_kv8<256, TY_BF16, TY_BF16>);
    return launched(me);
  }
  // part of a head rotated: pairs fall anywhere
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((uint32_t)rows), dim3(64), 0, (hipStream_t)stream, g, qkv, n_new, new_lens,
                       n_heads, rope_dim, split_half, cos_tab, sin_tab, q_norm, k_norm, eps, q_out,
                       static_cast<uint16_t*>(kc), static_cast<uint16_t*>(vc));
  };
  if (kv_type == TY_F16) {
    if (q_type == TY_F32) go(cm::k_paged_rope_kv<TY_F32, TY_F16>);
    else go(cm::k_paged_rope_kv<TY_F16, TY_F16>);
  } else {
    if (q_type == TY_F32) go(cm::k_paged_rope_kv<TY_F32, TY_BF16>);
    else go(cm::k_paged_rope_kv<TY_BF16, TY_BF16>);
  }
  return launched(me);
}

size_t camelid_hip_paged_attention_workspace(uint32_t n_seqs, uint32_t n_new, uint32_t n_heads, uint32_t n_kv,
                                             uint32_t hd, uint32_t page_size, uint32_t table_stride,
                                             uint32_t with_weights) {
  if (!n_kv) return 0;
  const PaSizes z = pa_sizes(n_seqs, n_new, n_heads, n_kv, hd, (uint64_t)page_size * table_stride, with_weights != 0);
  return z.bytes;
}

int camelid_hip_paged_attention(const void* q, uint32_t q_type, uint32_t q_stride, uint32_t n_seqs, uint32_t n_new,
                                const uint32_t* new_lens, uint32_t n_heads, uint32_t n_kv, uint32_t hd, const void* kc,
                                const void* vc, uint32_t kv_type, uint32_t n_pages, uint32_t page_size,
                                const uint32_t* table, uint32_t table_stride, const uint32_t* lens, float scale,
                                void* out, uint32_t out_stride, float* weights, void* workspace,
                                size_t workspace_bytes, uint32_t* status, void* stream) {
  const char* me = "paged_attention";
  if (!n_seqs || !n_new) return 0;
  if (!q || !kc || !vc || !table || !lens || !out || !workspace) return cm::fail_global(me, "null argument");
  cm::Paged g;
  const char* why;
  if (!paged_geometry(&g, n_seqs, n_kv, hd, n_pages, page_size, table, table_stride, lens, status, &why))
    return cm::fail_global(me, why);
  if (!heads_ok(n_heads, n_kv)) return cm::fail_global(me, "n_heads must be a nonzero multiple of n_kv, at most 4096");
  if (n_new > CAMELID_MAX_VERIFY_K) return cm::fail_global(me, "at most 8 new tokens per sequence");
  if (!type_ok(q_type) || !kv_type_ok(kv_type)) return cm::fail_global(me, "unknown type");
  if (q_type != TY_F32 && q_type != kv_type)
    return cm::fail_global(me, "16-bit q rows must have the cache's type");
  if (!std::isfinite(scale)) return cm::fail_global(me, "attention score scale must be finite");
  if (q_type != TY_F32 && !std::isfinite(scale * cm::PA_LOG2E))
    return cm::fail_global(me, "scale times log2(e) must be finite for 16-bit q rows");
  const uint64_t groups = (uint64_t)n_seqs * n_kv * (n_new * (n_heads / n_kv) + (weights ? 1 + ((uint64_t)table_stride * page_size >> 6) : 0));
  if (!grid_ok(groups, cm::PA_NT)) return cm::fail_global(me, "too many rows in one call");
  const uint32_t unit = q_type == TY_F32 ? 4 : 8;
  if (q_stride < (uint64_t)n_heads * hd || out_stride < (uint64_t)n_heads * hd || q_stride % unit || out_stride % unit)
    return cm::fail_global(me, "q_stride and out_stride must hold n_heads * head_dim elements and be whole 16-byte units");
  if (!aligned16(q) || !aligned16(out) || !aligned16(kc) || !aligned16(vc) || !aligned16(workspace) ||
      !aligned4(weights) || !aligned4(new_lens))
    return cm::fail_global(me, "q, out, the cache and the workspace must be 16-byte aligned, the rest 4-byte aligned");
  if (workspace_bytes < camelid_hip_paged_attention_workspace(n_seqs, n_new, n_heads, n_kv, hd, page_size,
                                                              table_stride, weights != nullptr))
    return cm::fail_global(me, "workspace too small (camelid_hip_paged_attention_workspace)");
  const PaSizes z = pa_sizes(n_seqs, n_new, n_heads, n_kv, hd, (uint64_t)page_size * table_stride, weights != nullptr);
  if (!z.fits) return cm::fail_global(me, "n_seqs * n_kv * table_stride * page_size too large for one call");
  // every workgroup works the plan out from all lengths: 65535 sequences of 5 positions take 60 ms (4000: 0.18),
  // and it grows with the square
  if (n_seqs > 65535) return cm::fail_global(me, "at most 65535 sequences");
  char* ws = static_cast<char*>(workspace);
  cm::PaArgs a{};
  a.g = g;
  a.q = q;
  a.new_lens = new_lens;
  a.kc = static_cast<const uint16_t*>(kc);
  a.vc = static_cast<const uint16_t*>(vc);
  a.out = out;
  a.part_ml = reinterpret_cast<float*>(ws);
  a.part_o = reinterpret_cast<float*>(ws + z.part_o);
  a.cuts = reinterpret_cast<uint2*>(ws + z.cuts);
  a.stats = reinterpret_cast<float*>(ws + z.stats);
  a.scores = weights ? reinterpret_cast<float*>(ws + z.scores) : nullptr;
  a.weights = weights;
  a.scale = scale;
  a.p_bits = kv_type == TY_F16 ? 14.0f : -24.0f;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.n_new = n_new;
  a.n_heads = n_heads;
  a.group = n_heads / n_kv;
  a.group_magic = a.group == 1 ? 0 : (uint32_t)(((1ull << 32) + a.group - 1) / a.group);
  a.at_once = z.at_once;
  a.blocks = z.blocks;
  a.part_rows = z.part_rows;
  const bool ok = kv_type == TY_F16 ? (q_type == TY_F32 ? pa_launch_hd<TY_F16, TY_F32>(a, z, (hipStream_t)stream)
                                                        : pa_launch_hd<TY_F16, TY_F16>(a, z, (hipStream_t)stream))
                                    : (q_type == TY_F32 ? pa_launch_hd<TY_BF16, TY_F32>(a, z, (hipStream_t)stream)
                                                        : pa_launch_hd<TY_BF16, TY_BF16>(a, z, (hipStream_t)stream));
  return ok ? launched(me) : 1;
}

size_t camelid_hip_paged_evict_workspace(uint32_t n_seqs, uint32_t n_kv, uint32_t page_size, uint32_t table_stride,
                                         uint32_t keep) {
  (void)page_size;
  (void)table_stride;
  return up256((size_t)n_seqs * 8) + 3 * up256((size_t)n_seqs * n_kv * keep * 4);
}

int camelid_hip_paged_evict(void* kc, void* vc, uint32_t n_pages, uint32_t page_size, uint32_t n_kv, uint32_t hd,
                            const uint32_t* table, uint32_t table_stride, const uint32_t* lens, uint32_t n_seqs,
                            float* weights, uint32_t keep, uint32_t recent, uint32_t* lens_out, uint32_t* kept,
                            void* workspace, size_t workspace_bytes, uint32_t* status, void* stream) {
  const char* me = "paged_evict";
  if (!n_seqs) return 0;
  if (!kc || !vc || !table || !lens || !weights || !lens_out || !workspace) return cm::fail_global(me, "null argument");
  cm::Paged g;
  const char* why;
  if (!paged_geometry(&g, n_seqs, n_kv, hd, n_pages, page_size, table, table_stride, lens, status, &why))
    return cm::fail_global(me, why);
  if (!keep || keep > (1u << 24)) return cm::fail_global(me, "keep must be in 1..=2^24");
  if (recent > keep) return cm::fail_global(me, "recent must be at most keep");
  // dims of a workgroup of the move: as many as still let all kept rows be one chunk, else 8, of V 16 where that
  // leaves two workgroups a CU (4 x 8 rows of V with 8 dims: 31.8 us for the call, with 16: 33.0)
  uint32_t ks = 0, vs = 0;
  while (hd >> (4 + ks) && keep <= (1u << cm::EM_K_LOG2) >> (ks + 1)) ++ks;
  while (hd >> (4 + vs) && keep <= cm::EM_G >> (vs + 1)) ++vs;
  if (!vs && (uint64_t)n_seqs * n_kv * hd >= 512 * 16) vs = 1;
  const uint64_t movers = (uint64_t)n_seqs * n_kv * ((hd >> (3 + ks)) + (hd >> (3 + vs)));
  if (!grid_ok(movers, cm::EM_NT)) return cm::fail_global(me, "n_seqs * n_kv * head_dim too large for one call");
  if ((uint64_t)n_pages * page_size > 0xffffffffull)
    return cm::fail_global(me, "n_pages * page_size must be below 2^32");
  if (!aligned16(kc) || !aligned16(vc) || !aligned16(workspace) || !aligned4(weights) || !aligned4(lens_out) ||
      !aligned4(kept))
    return cm::fail_global(me, "the cache and the workspace must be 16-byte aligned, the rest 4-byte aligned");
  if (workspace_bytes < camelid_hip_paged_evict_workspace(n_seqs, n_kv, page_size, table_stride, keep))
    return cm::fail_global(me, "workspace too small (camelid_hip_paged_evict_workspace)");
  cm::EvictPlan plan;
  char* ws = static_cast<char*>(workspace);
  plan.old_lens = reinterpret_cast<uint32_t*>(ws);
  plan.new_lens = plan.old_lens + n_seqs;
  ws += up256((size_t)n_seqs * 8);
  const size_t rows = up256((size_t)n_seqs * n_kv * keep * 4);
  plan.slot = reinterpret_cast<uint32_t*>(ws);
  plan.from = reinterpret_cast<uint32_t*>(ws + rows);
  plan.granule = reinterpret_cast<uint32_t*>(ws + 2 * rows);
  // rows of at most 512, 2048, 8192 and 16384 positions have their weights read once
  const uint32_t cap = page_size * table_stride;
  const auto select = [&](auto kernel, uint32_t threads) {
    hipLaunchKernelGGL(kernel, dim3(n_seqs * n_kv), dim3(threads), 0, (hipStream_t)stream, g, weights, keep, recent, plan,
                       kept);
  };
  if (cap <= 512) select(cm::k_evict_select<2, 256>, 256);
  else if (cap <= 2048) select(cm::k_evict_select<2, 1024>, 1024);
  else if (cap <= 8192) select(cm::k_evict_select<8, 1024>, 1024);
  else select(cm::k_evict_select<16, 1024>, 1024);
  const auto go = [&](auto kernel, uint32_t f) {
    const size_t lds = cm::em_lds(f);
    if (lds >= 64 * 1024) {
      const hipError_t st = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
      if (st != hipSuccess) return cm::fail_global(me, hipGetErrorString(st));
    }
    hipLaunchKernelGGL(kernel, dim3((uint32_t)movers), dim3(cm::EM_NT), lds, (hipStream_t)stream, g,
                       static_cast<uint16_t*>(kc), static_cast<uint16_t*>(vc), keep, plan, lens_out, ks, vs);
    return launched(me);
  };
  // few workgroups (one or two a CU) with many rows take them in larger chunks (8 x 14511 rows of one of two
  // sequences: 73 us for the call against 78, 1 x 8 x 14027: 56 against 59)
  if (!ks && !vs && movers <= 256) return go(cm::k_evict_move<4>, 4);
  if (!ks && !vs && movers <= 512) return go(cm::k_evict_move<2>, 2);
  return go(cm::k_evict_move<1>, 1);
}

static uint32_t vd_shares(uint32_t vocab) { return (vocab + cm::VD_SHARE - 1) / cm::VD_SHARE; }
static size_t vd_parts_bytes(uint64_t n_seqs, uint64_t n_draft, uint32_t vocab) {
  return up256(n_seqs * (2 * n_draft + 1) * vd_shares(vocab) * sizeof(cm::VdPart));
}

size_t camelid_hip_verify_drafts_workspace(uint32_t n_seqs, uint32_t n_draft, uint32_t vocab) {
  return vd_parts_bytes(n_seqs, n_draft, vocab) + up256((size_t)n_seqs * vd_shares(vocab) * 8) +
         (size_t)n_seqs * (cm::VD_MAX_ROWS + 1) * sizeof(cm::VdPart);
}

int camelid_hip_verify_drafts(const void* target, const void* draft_logits, uint32_t logits_type,
                              const uint32_t* draft_tokens, const uint32_t* draft_lens, uint32_t n_seqs,
                              uint32_t n_draft, uint32_t vocab, const float* temperature, const float* uniforms,
                              uint32_t* accepted, uint32_t* tokens_out, float* logprobs_out, void* workspace,
                              size_t workspace_bytes, void* stream) {
  const char* me = "verify_drafts";
  if (!n_seqs) return 0;
  if (!target || !temperature || !uniforms || !accepted || !tokens_out || !workspace || (n_draft && !draft_tokens))
    return cm::fail_global(me, "null argument");
  if (n_draft > 31) return cm::fail_global(me, "at most 31 drafts per sequence");
  if (!vocab || vocab > (1u << 24)) return cm::fail_global(me, "vocab must be in 1..=2^24");
  if (n_seqs > 65535) return cm::fail_global(me, "at most 65535 sequences");
  if (!type_ok(logits_type)) return cm::fail_global(me, "unknown type");
  const uintptr_t unit = logits_type == TY_F32 ? 3 : 1;
  if (((reinterpret_cast<uintptr_t>(target) | reinterpret_cast<uintptr_t>(draft_logits)) & unit) ||
      !aligned16(workspace) || !aligned4(draft_tokens) || !aligned4(draft_lens) || !aligned4(temperature) ||
      !aligned4(uniforms) || !aligned4(accepted) || !aligned4(tokens_out) || !aligned4(logprobs_out))
    return cm::fail_global(me, "the workspace must be 16-byte aligned, the rest aligned to its elements");
  if (workspace_bytes < camelid_hip_verify_drafts_workspace(n_seqs, n_draft, vocab))
    return cm::fail_global(me, "workspace too small (camelid_hip_verify_drafts_workspace)");
  cm::VdArgs a{};
  a.target = target;
  a.draft = n_draft ? draft_logits : nullptr;
  a.tokens = draft_tokens;
  a.draft_lens = draft_lens;
  a.temperature = temperature;
  a.uniforms = uniforms;
  a.parts = static_cast<cm::VdPart*>(workspace);
  a.rest = reinterpret_cast<double*>(static_cast<char*>(workspace) + vd_parts_bytes(n_seqs, n_draft, vocab));
  a.judged = reinterpret_cast<cm::VdPart*>(reinterpret_cast<char*>(a.rest) + up256((size_t)n_seqs * vd_shares(vocab) * 8));
  a.accepted = accepted;
  a.out = tokens_out;
  a.logprobs = logprobs_out;
  a.n_draft = n_draft;
  a.vocab = vocab;
  a.shares = vd_shares(vocab);
  const uint64_t rows = a.draft ? 2 * n_draft + 1 : n_draft + 1, groups = (a.shares + 3) / 4;
  if (!grid_ok(n_seqs * rows * groups, cm::VD_NT)) return cm::fail_global(me, "too many rows in one call");
  // shares of a wave: one while the chip holds all waves at once (about 4096), up to 4
  const uint32_t per = (uint32_t)std::min<uint64_t>(4, std::max<uint64_t>(1, n_seqs * rows * a.shares / 4096));
  const auto go = [&](auto stats, auto rest, auto pick) {
    hipLaunchKernelGGL(stats, dim3((uint32_t)(n_seqs * rows * ((a.shares + 4 * per - 1) / (4 * per)))), dim3(cm::VD_NT),
                       0, (hipStream_t)stream, a, per);
    if (a.draft)
      hipLaunchKernelGGL(rest, dim3((uint32_t)(n_seqs * groups)), dim3(cm::VD_NT), 0, (hipStream_t)stream, a);
    hipLaunchKernelGGL(pick, dim3(n_seqs), dim3(cm::VD_NT), 0, (hipStream_t)stream, a);
  };
  if (logits_type == TY_F32) go(cm::k_vd_stats<TY_F32>, cm::k_vd_rest<TY_F32>, cm::k_vd_pick<TY_F32>);
  else if (logits_type == TY_F16) go(cm::k_vd_stats<TY_F16>, cm::k_vd_rest<TY_F16>, cm::k_vd_pick<TY_F16>);
  else go(cm::k_vd_stats<TY_BF16>, cm::k_vd_rest<TY_BF16>, cm::k_vd_pick<TY_BF16>);
  return launched(me);
}

}  // extern "C"
