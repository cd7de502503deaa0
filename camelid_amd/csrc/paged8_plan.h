// paged8_plan.h -- how the attention over an 8-bit cache is cut, and what workspace that takes: the sizes that its
// kernels (kernels_paged8_attn.h) and its entry point share; plain C++.
#pragma once
#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "../../include/camelid_hip.h"
#include "launch_sizes.h"

namespace cm {

constexpr uint32_t P8_TILE = 64;  // positions
// Workgroups of a CU that the split's plan counts on and that the compiler is held to.  (Registers and LDS take one more,
// but for f32 rows over heads of 256.)
constexpr int p8_per_cu(int hd, int nr) { return hd == 64 ? 4 - nr : hd == 128 ? 3 - nr : 1; }
// Prompts: rows of a block, and tiles up to which segments stay whole.
constexpr int p8p_rows(int hd) { return hd == 256 ? 64 : 128; }
constexpr uint32_t P8P_WHOLE = 64;

// What a call of the attention needs: row blocks of 16 * nr query rows, workgroups, workspace.
struct P8Sizes {
  uint32_t nr, blocks, part_rows, at_once, grid;
  bool prompt;                 // the prompts' kernel
  uint64_t tiles;              // of all row blocks, as the tables have room
  bool join;                   // some segment may be cut
  bool fits;                   // the plan's 32-bit counts hold
  size_t part_o, cuts, bytes;  // offsets of the workspace's parts, its size
};

inline P8Sizes p8_sizes(uint64_t n_seqs, uint64_t n_new, uint64_t n_heads, uint64_t n_kv, uint32_t hd, uint64_t cap,
                        bool f32_rows) {
  P8Sizes z;
  const uint64_t rows = n_new * (n_heads / n_kv), cap_tiles = (cap + P8_TILE - 1) / P8_TILE;
  // The prompts' kernel converts K and V once for a block of rows and keeps its operands in LDS; the split reads and
  // converts them once for each 32 rows (16 for heads of 256), but cuts finer and waits at no barrier.  From a whole
  // block on (two for heads of 256): 16 sequences of 4096 positions, 8 KV heads of 64 / 128 / 256, prompts' kernel and split:
  // 64 rows 49 and 39 / 68 and 64 / 111 and 133 us, 96 rows 50 and 49 / 73 and 85 / 187 and 239, 128 rows 51 and
  // 59 / 80 and 104 / 190 and 215, 256 rows 88 and 98 / 132 and 170 / 343 and 370 (groups of 1 and 8 alike; with
  // one row more than a block the split wins again: 43 tokens of groups of 3 81 and 71 / 119 and 120 / 274 and 232).
  // One sequence: the split by 1 to 3 us from 64 to 512 rows (128: 18 and 15 / 22 and 22 / 27 and 26).
  z.prompt = n_new > CAMELID_MAX_VERIFY_K && rows >= 128;
  z.nr = z.prompt ? p8p_rows((int)hd) / 16 : rows > 16 && hd <= 128 ? 2 : 1;
  z.blocks = (uint32_t)((rows + 16 * z.nr - 1) / (16 * z.nr));
  z.part_rows = (uint32_t)std::min<uint64_t>(rows, 16 * z.nr);
  // a piece has at least `least` tiles, or all; pieces altogether are at most `most` and one for each segment
  const uint64_t segments = n_seqs * n_kv * z.blocks;
  z.tiles = segments * cap_tiles;
  uint64_t least = !z.prompt || z.tiles <= 2048 ? 4 : 16;
  const uint64_t most = z.prompt ? 512 : 2048;
  // prompts whose pieces of 16 would be one for each CU at most, where two fit (not f32's 8 waves), and most of whose
  // pieces do not end at the diagonal: 512 tokens at 1536 46 us against 49, 256 at 3840 45 against 47; f32 57 against 50
  if (least == 16 && !f32_rows && segments < 256 && segments * ((cap_tiles + 15) / 16) <= 256 && cap >= 2 * n_new)
    least = 8;
  // prompts without much before them (the tables have no room for it; the kernel looks at the lengths, too): not cut
  if (least == 16 && cap < 2 * n_new && segments >= 256) least = P8P_WHOLE;
  // the split's: 256 CUs; a seventh less, since cutting every segment evenly makes some more pieces
  z.at_once = z.prompt ? (uint32_t)least : 256 * p8_per_cu((int)hd, (int)z.nr) * 7 / 8;
  const uint64_t pieces = std::min(most + segments, segments * ((cap_tiles + least - 1) / least));
  z.fits = z.tiles < (1ull << 31) && grid_ok(pieces, 512);
  z.grid = (uint32_t)pieces;
  z.join = cap_tiles > least;
  // cut segments have more tiles than the target: at most `most` of them, twice as many pieces
  const size_t slots = z.join ? (size_t)std::min(2 * most, pieces) : 0;
  z.part_o = up256(slots * z.part_rows * 8);
  z.cuts = z.part_o + up256(slots * z.part_rows * hd * 4);
  z.bytes = z.cuts + up256(segments * 8);
  return z;
}

// Workspace of calls of at most these sizes: parts of at most `slots` pieces, and a word pair for each segment; the
// most that either kernel takes up to n_new.
inline size_t p8_workspace(uint64_t n_seqs, uint64_t n_new, uint64_t n_heads, uint64_t n_kv, uint32_t hd, uint64_t cap) {
  const uint64_t group = std::max<uint64_t>(n_heads / n_kv, 1), cap_tiles = (cap + P8_TILE - 1) / P8_TILE;
  const auto most = [&](uint64_t rows, uint64_t block, uint64_t slots) {
    const uint64_t segments = n_seqs * n_kv * ((rows + block - 1) / block), part_rows = std::min(rows, block);
    slots = cap_tiles > 4 ? std::min(slots, segments * ((cap_tiles + 3) / 4)) : 0;
    return up256(slots * part_rows * 8) + up256(slots * part_rows * hd * 4) + up256(segments * 8);
  };
  const uint64_t few = std::min(n_new, std::max<uint64_t>(CAMELID_MAX_VERIFY_K, 127 / group)) * group;
  size_t bytes = std::max(most(std::min<uint64_t>(few, 16), 16, 4096), most(few, few > 16 && hd <= 128 ? 32 : 16, 4096));
  if (n_new > CAMELID_MAX_VERIFY_K && n_new * group >= 128)
    bytes = std::max(bytes, most(n_new * group, p8p_rows((int)hd), 1024));
  return bytes;
}

}  // namespace cm
