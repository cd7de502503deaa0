// launch_sizes.h -- what launches and workspaces are made of; plain C++.
#pragma once
#include <cstddef>
#include <cstdint>

namespace cm {

// A launch holds at most 2^32 - 1 threads.
inline bool grid_ok(uint64_t groups, uint32_t threads) { return groups <= 0xffffffffull / threads; }
inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace cm
