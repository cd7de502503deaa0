// kernels_pages.h -- who holds which page of a cache: rows of page ids that grow, shrink, are forked and
// made their own, pages moved to the front of the pool, and the copies that follow from it.
//
// refs[page] counts the table entries (of the first held[s] of row s) that name the page; 0: free.  All of
// it is integers in an order that is laid down, so every call has one result: the k-th page needed, in the
// order of sequences and entries, is the k-th free one in ascending order.
#pragma once
#include "kernels_paged.h"

namespace cm {

constexpr uint32_t PG_NT = 256;
constexpr uint32_t PG_CHUNK = 1024;  // pages of a workgroup that counts or lists them
constexpr uint32_t PG_COW = 0x80000000u;  // mark of an entry to be replaced, between two launches
enum { PG_NO_PAGE = 4, PG_BAD_FORK = 8 };  // CAMELID_PAGED_NO_PAGE, CAMELID_PAGED_BAD_FORK

// Exclusive prefix sum of a workgroup's x, and the sum.
struct PgScan {
  uint32_t before, total;
};
template <uint32_t NT>
__device__ __forceinline__ PgScan pg_scan(uint32_t x, uint32_t* s_wave) {
  const uint32_t lane = threadIdx.x & 63u, w = threadIdx.x >> 6, inc = ev_wave_scan(x);
  __syncthreads();  // (the caller's last use of s_wave)
  if (lane == 63) s_wave[w] = inc;
  __syncthreads();
  PgScan r{inc - x, 0};
  for (uint32_t i = 0; i < NT / 64; ++i) {
    if (i < w) r.before += s_wave[i];
    r.total += s_wave[i];
  }
  return r;
}

struct PagesArgs {
  uint32_t* table;
  uint32_t* held;
  const uint32_t* first;  // may be null: nothing is going to be written
  const uint32_t* lens;
  uint32_t* refs;
  uint32_t* pairs;
  uint32_t* n_pairs;
  uint32_t* granted;
  uint32_t* status;
  uint32_t* need;    // [n_seqs] pages needed, PG_COW: left alone
  uint32_t* cows;    // [n_seqs] of them: replaced ones
  uint32_t* before;  // [n_seqs] pages needed by the sequences before, ~0: not granted
  uint32_t* cows_before;
  uint32_t* chunk;   // [chunks] free pages
  uint32_t* free_list;
  uint32_t stride, n_seqs, shift, n_pages, max_pairs, chunks;
};

__device__ __forceinline__ void pages_flag(uint32_t* status, uint32_t bit) {
  if (status) atomicOr(status, bit);
}

// 1: entries that a row no longer needs let go.  A workgroup per sequence.
__device__ __forceinline__ uint32_t pages_wanted(const PagesArgs& a, uint32_t s) {
  return (uint32_t)(((uint64_t)a.lens[s] + (1u << a.shift) - 1) >> a.shift);
}
__global__ __launch_bounds__(PG_NT) void k_pages_shrink(PagesArgs a) {
  __shared__ uint32_t s_bad;
  const uint32_t s = blockIdx.x, tid = threadIdx.x, held = a.held[s], want = pages_wanted(a, s);
  if (tid == 0) s_bad = held > a.stride || want > a.stride ? PG_BAD_LENGTH : 0u;
  __syncthreads();
  const uint32_t* row = a.table + (size_t)s * a.stride;
  if (!s_bad) {
    bool bad = false;
    for (uint32_t j = tid; j < held; j += PG_NT) bad |= row[j] >= a.n_pages;
    if (bad) s_bad = PG_BAD_PAGE;
  }
  __syncthreads();
  if (s_bad) {
    if (tid == 0) {
      pages_flag(a.status, s_bad);
      a.need[s] = PG_COW;
    }
    return;
  }
  for (uint32_t j = want + tid; j < held; j += PG_NT) atomicSub(&a.refs[row[j]], 1u);
  if (tid == 0) {
    a.need[s] = 0;
    if (want < held) a.held[s] = want;
  }
}

// 2: pages that each row needs (its entries to be replaced marked), and free pages of each chunk.
__global__ __launch_bounds__(PG_NT) void k_pages_count(PagesArgs a) {
  __shared__ uint32_t s_sum;
  const uint32_t tid = threadIdx.x;
  if (tid == 0) s_sum = 0;
  __syncthreads();
  uint32_t n = 0;
  if (blockIdx.x >= a.n_seqs) {
    const uint32_t c = blockIdx.x - a.n_seqs, p0 = c * PG_CHUNK;
    for (uint32_t i = tid; i < PG_CHUNK; i += PG_NT) n += p0 + i < a.n_pages && a.refs[p0 + i] == 0;
    if (n) atomicAdd(&s_sum, n);
    __syncthreads();
    if (tid == 0) a.chunk[c] = s_sum;
    return;
  }
  const uint32_t s = blockIdx.x;
  if (a.need[s] & PG_COW) return;
  const uint32_t held = a.held[s], want = pages_wanted(a, s);
  uint32_t* row = a.table + (size_t)s * a.stride;
  if (a.first && a.first[s] < a.lens[s]) {
    for (uint32_t j = (a.first[s] >> a.shift) + tid; j < held; j += PG_NT) {
      if (a.refs[row[j]] > 1) {
        row[j] |= PG_COW;
        ++n;
      }
    }
  }
  if (n) atomicAdd(&s_sum, n);
  __syncthreads();
  if (tid == 0) {
    a.cows[s] = s_sum;
    a.need[s] = s_sum + (want - held);
  }
}

// 3: the free pages listed; by one more workgroup the sequences' shares of them.
constexpr uint32_t PG_PLAN_NT = 1024;
__global__ __launch_bounds__(PG_PLAN_NT) void k_pages_plan(PagesArgs a) {
  __shared__ uint32_t s_wave[PG_PLAN_NT / 64];
  const uint32_t tid = threadIdx.x;
  // free pages before this chunk, or (the last workgroup) of the pool
  uint32_t mine = 0;
  for (uint32_t i = tid; i < min(blockIdx.x, a.chunks); i += PG_PLAN_NT) mine += a.chunk[i];
  const uint32_t base = pg_scan<PG_PLAN_NT>(mine, s_wave).total;
  if (blockIdx.x < a.chunks) {
    const uint32_t p0 = blockIdx.x * PG_CHUNK;
    uint32_t at = base;
    for (uint32_t i = 0; i < PG_CHUNK; i += PG_PLAN_NT) {
      const uint32_t p = p0 + i + tid;
      const bool free = p < a.n_pages && a.refs[p] == 0;
      const PgScan r = pg_scan<PG_PLAN_NT>(free, s_wave);
      if (free) a.free_list[at + r.before] = p;
      at += r.total;
    }
    return;
  }
  uint32_t pages = 0, cows = 0, told = 0;
  for (uint32_t i = 0; i < a.n_seqs; i += PG_PLAN_NT) {
    const uint32_t s = i + tid;
    const bool live = s < a.n_seqs && !(a.need[s] & PG_COW);
    const uint32_t need = live ? a.need[s] : 0u, cow = live ? a.cows[s] : 0u;
    const PgScan n = pg_scan<PG_PLAN_NT>(need, s_wave), c = pg_scan<PG_PLAN_NT>(cow, s_wave);
    const uint32_t to = cows + c.before + cow;
    const bool ok = live && (need == 0 || (pages + n.before + need <= base && (cow == 0 || to <= a.max_pairs)));
    if (s < a.n_seqs) {
      a.before[s] = ok ? pages + n.before : ~0u;
      a.cows_before[s] = cows + c.before;
      if (a.granted) a.granted[s] = ok;
      if (live && !ok) pages_flag(a.status, PG_NO_PAGE);
    }
    if (ok && cow) told = to;
    pages += n.total;
    cows += c.total;
  }
  if (!a.n_pairs) return;
  __shared__ uint32_t s_told;
  if (tid == 0) s_told = 0;
  __syncthreads();
  atomicMax(&s_told, told);
  __syncthreads();
  if (tid == 0) *a.n_pairs = s_told;
}

// 4: the rows' new entries.  A workgroup per sequence.
__global__ __launch_bounds__(PG_NT) void k_pages_grant(PagesArgs a) {
  __shared__ uint32_t s_wave[PG_NT / 64];
  const uint32_t s = blockIdx.x, tid = threadIdx.x;
  if (a.need[s] & PG_COW) return;
  const uint32_t held = a.held[s], want = pages_wanted(a, s), before = a.before[s];
  uint32_t* row = a.table + (size_t)s * a.stride;
  if (a.need[s] == 0) return;
  uint32_t rank = 0;
  if (a.cows[s]) {
    for (uint32_t j0 = a.first[s] >> a.shift; j0 < held; j0 += PG_NT) {
      const uint32_t j = j0 + tid, e = j < held ? row[j] : 0u;
      const bool cow = e & PG_COW;
      const PgScan r = pg_scan<PG_NT>(cow, s_wave);
      if (cow) {
        const uint32_t old = e & ~PG_COW;
        if (before == ~0u) {
          row[j] = old;
        } else {
          const uint32_t k = rank + r.before, page = a.free_list[before + k], at = a.cows_before[s] + k;
          a.pairs[2 * at] = old;
          a.pairs[2 * at + 1] = page;
          row[j] = page;
          a.refs[page] = 1;
          atomicSub(&a.refs[old], 1u);
        }
      }
      rank += r.total;
    }
  }
  if (before == ~0u) return;
  for (uint32_t j = held + tid; j < want; j += PG_NT) {
    const uint32_t page = a.free_list[before + rank + (j - held)];
    row[j] = page;
    a.refs[page] = 1;
  }
  if (tid == 0 && want > held) a.held[s] = want;
}

// The four steps by one workgroup with barriers in the place of launches, for small batches and pools: a thread per
// entry.  Bound: latency, 7 to 9 us for 64 rows over 1500 pages; the four launches take 13, and four times a
// launch's host time.  A step of 64 rows of 160 entries over 8192 pages with nothing shared: 16 us.  What other waves changed is waited for and read past the L1.
constexpr uint32_t PG_ONE_SEQS = 1024, PG_ONE_PAGES = 8192, PG_ONE_ENTRIES = 16384;
__device__ __forceinline__ uint32_t pg_read(const uint32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__global__ __launch_bounds__(PG_PLAN_NT) void k_pages_reserve(PagesArgs a) {
  constexpr uint32_t NT = PG_PLAN_NT, PER = PG_ONE_PAGES / NT;
  __shared__ uint32_t s_wave[NT / 64], s_held[PG_ONE_SEQS], s_want[PG_ONE_SEQS], s_write[PG_ONE_SEQS], s_bad[PG_ONE_SEQS];
  __shared__ uint32_t s_cows[PG_ONE_SEQS], s_before[PG_ONE_SEQS], s_cows_before[PG_ONE_SEQS];
  __shared__ uint32_t s_mark[PG_ONE_ENTRIES / 32], s_free[PG_ONE_PAGES], s_told;
  const uint32_t tid = threadIdx.x, entries = a.n_seqs * a.stride;
  for (uint32_t i = tid; i < PG_ONE_ENTRIES / 32; i += NT) s_mark[i] = 0;
  if (tid == 0) s_told = 0;
  if (tid < a.n_seqs) {
    const uint32_t held = a.held[tid], want = pages_wanted(a, tid);
    s_held[tid] = held;
    s_want[tid] = want;
    s_write[tid] = a.first && a.first[tid] < a.lens[tid] ? a.first[tid] >> a.shift : ~0u;  // first entry to be written
    s_bad[tid] = held > a.stride || want > a.stride ? PG_BAD_LENGTH : 0u;
    s_cows[tid] = 0;
  }
  __syncthreads();
  // 1: entries that a row no longer needs
  for (uint32_t i = tid; i < entries; i += NT) {
    const uint32_t s = i / a.stride, j = i - s * a.stride;
    if (j < s_held[s] && a.table[i] >= a.n_pages && s_bad[s] == 0) s_bad[s] = PG_BAD_PAGE;
  }
  __syncthreads();
  for (uint32_t i = tid; i < entries; i += NT) {
    const uint32_t s = i / a.stride, j = i - s * a.stride;
    if (!s_bad[s] && j >= s_want[s] && j < s_held[s]) atomicSub(&a.refs[a.table[i]], 1u);
  }
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  // 2: entries to be replaced marked; the free pages in ascending order (thread i: PER pages side by side)
  for (uint32_t i = tid; i < entries; i += NT) {
    const uint32_t s = i / a.stride, j = i - s * a.stride;
    if (!s_bad[s] && j >= s_write[s] && j < min(s_held[s], s_want[s]) && pg_read(&a.refs[a.table[i]]) > 1) {
      atomicOr(&s_mark[i >> 5], 1u << (i & 31u));
      atomicAdd(&s_cows[s], 1u);
    }
  }
  uint32_t mine = 0, mask = 0;
#pragma unroll
  for (uint32_t i = 0; i < PER; ++i) {
    const uint32_t p = tid * PER + i;
    if (p < a.n_pages && pg_read(&a.refs[p]) == 0) {
      mask |= 1u << i;
      ++mine;
    }
  }
  const PgScan free = pg_scan<NT>(mine, s_wave);
  for (uint32_t i = 0, k = free.before; i < PER; ++i)
    if (mask >> i & 1u) s_free[k++] = tid * PER + i;
  __syncthreads();
  // 3: the sequences' shares
  const bool here = tid < a.n_seqs, live = here && !s_bad[tid];
  const uint32_t held = live ? min(s_held[tid], s_want[tid]) : 0u, cow = live ? s_cows[tid] : 0u;
  const uint32_t need = live ? cow + s_want[tid] - held : 0u;
  const PgScan n = pg_scan<NT>(need, s_wave), c = pg_scan<NT>(cow, s_wave);
  const bool ok = live && (need == 0 || (n.before + need <= free.total && (cow == 0 || c.before + cow <= a.max_pairs)));
  if (here) {
    s_before[tid] = ok ? n.before : ~0u;
    s_cows_before[tid] = c.before;
    if (live) a.held[tid] = ok ? s_want[tid] : held;
    if (a.granted) a.granted[tid] = ok;
    if (!ok) pages_flag(a.status, live ? PG_NO_PAGE : s_bad[tid]);
    if (ok && cow) atomicMax(&s_told, c.before + cow);
  }
  __syncthreads();
  if (a.n_pairs && tid == 0) *a.n_pairs = s_told;
  // 4: the rows' new entries
  for (uint32_t i = tid; i < entries; i += NT) {
    const uint32_t s = i / a.stride, j = i - s * a.stride, before = s_before[s];
    if (before == ~0u) continue;
    if (s_mark[i >> 5] >> (i & 31u) & 1u) {
      uint32_t rank = 0;  // marked entries of the row before this one
      for (uint32_t k = s * a.stride; k < i;) {
        const uint32_t bits = s_mark[k >> 5] >> (k & 31u), most = min(32 - (k & 31u), i - k);
        rank += __popc(most < 32 ? bits & ((1u << most) - 1u) : bits);
        k += most;
      }
      const uint32_t old = a.table[i], page = s_free[before + rank], at = s_cows_before[s] + rank;
      a.pairs[2 * at] = old;
      a.pairs[2 * at + 1] = page;
      a.table[i] = page;
      a.refs[page] = 1;
      atomicSub(&a.refs[old], 1u);
    } else if (j >= s_held[s] && j < s_want[s]) {
      const uint32_t page = s_free[before + s_cows[s] + (j - s_held[s])];
      a.table[i] = page;
      a.refs[page] = 1;
    }
  }
}

// ---------------------------------------------------------------------------
// Children get their parents' pages.  A workgroup per (parent, child) pair; a pair whose child holds pages or is
// named twice, or whose parent is a child itself, does nothing but flag: what the others do does not depend on
// their order then.
__global__ __launch_bounds__(PG_NT) void k_pages_fork(uint32_t* __restrict__ table, uint32_t stride,
                                                      uint32_t* __restrict__ held, uint32_t n_seqs,
                                                      const uint32_t* __restrict__ parents,
                                                      const uint32_t* __restrict__ children, uint32_t n_forks,
                                                      const uint32_t* __restrict__ lens, uint32_t shift,
                                                      uint32_t* __restrict__ refs, uint32_t n_pages,
                                                      uint32_t* status) {
  __shared__ uint32_t s_bad;
  const uint32_t i = blockIdx.x, tid = threadIdx.x, from = parents[i], to = children[i];
  if (tid == 0) s_bad = from >= n_seqs || to >= n_seqs || from == to ? PG_BAD_FORK : 0u;
  __syncthreads();
  if (!s_bad) {
    bool bad = false;
    for (uint32_t j = tid; j < n_forks; j += PG_NT) bad |= children[j] == from || (j != i && children[j] == to);
    if (bad) s_bad = PG_BAD_FORK;
  }
  __syncthreads();
  uint32_t n = 0;
  if (!s_bad) {
    n = held[from];
    const uint32_t had = held[to];
    if (lens) n = min(n, (uint32_t)(((uint64_t)lens[from] + (1u << shift) - 1) >> shift));
    __syncthreads();
    if (tid == 0 && (had || held[from] > stride)) s_bad = had ? PG_BAD_FORK : PG_BAD_LENGTH;
    __syncthreads();
  } else {
    __syncthreads();
    __syncthreads();
  }
  const uint32_t* src = table + (size_t)from * stride;
  if (!s_bad) {
    bool bad = false;
    for (uint32_t j = tid; j < n; j += PG_NT) bad |= src[j] >= n_pages;
    __syncthreads();
    if (bad) s_bad = PG_BAD_PAGE;
  } else {
    __syncthreads();
  }
  __syncthreads();
  if (s_bad) {
    if (tid == 0) pages_flag(status, s_bad);
    return;
  }
  uint32_t* dst = table + (size_t)to * stride;
  for (uint32_t j = tid; j < n; j += PG_NT) {
    const uint32_t page = src[j];
    dst[j] = page;
    atomicAdd(&refs[page], 1u);
  }
  if (tid == 0) held[to] = n;
}

// ---------------------------------------------------------------------------
// Pages in use moved to [0, n_live): the i-th hole there (ascending) takes the i-th highest page in use.
struct CompactArgs {
  const uint32_t* table;
  const uint32_t* held;
  const uint32_t* refs;
  uint32_t* table_out;
  uint32_t* refs_out;
  uint32_t* pairs;
  uint32_t* n_pairs;
  uint32_t* extent;
  uint32_t* status;
  uint32_t* chunk;  // [chunks] pages in use
  uint32_t* old;    // [n_pages] refs as they were
  uint32_t* rank;   // [n_pages] of a page in use at or behind n_live: pages in use above it
  uint32_t* holes;  // [n_pages]
  uint32_t* highs;  // [n_pages]
  uint32_t stride, n_seqs, n_pages, max_pairs, chunks;
};

__global__ __launch_bounds__(PG_NT) void k_compact_count(CompactArgs a) {
  __shared__ uint32_t s_sum;
  const uint32_t tid = threadIdx.x, p0 = blockIdx.x * PG_CHUNK;
  if (tid == 0) s_sum = 0;
  __syncthreads();
  uint32_t n = 0;
  for (uint32_t i = tid; i < PG_CHUNK; i += PG_NT) {
    if (p0 + i >= a.n_pages) break;
    const uint32_t r = a.refs[p0 + i];
    a.old[p0 + i] = r;
    n += r != 0;
  }
  if (n) atomicAdd(&s_sum, n);
  __syncthreads();
  if (tid == 0) a.chunk[blockIdx.x] = s_sum;
}

// Pages in use before a chunk, and of the pool.
__device__ __forceinline__ PgScan compact_sums(const CompactArgs& a, uint32_t c, uint32_t* s_wave) {
  uint32_t below = 0, all = 0;
  for (uint32_t i = threadIdx.x; i < a.chunks; i += PG_PLAN_NT) {
    const uint32_t n = a.chunk[i];
    all += n;
    if (i < c) below += n;
  }
  const uint32_t b = pg_scan<PG_PLAN_NT>(below, s_wave).total;
  return PgScan{b, pg_scan<PG_PLAN_NT>(all, s_wave).total};
}

// COUNT: no k_compact_count before it; every workgroup counts the pool by itself.  Up to 8192 pages, which takes less
// than a launch: compaction and copy of 2048 pages of 16 KB 22.4 us against 25.1, of 8192 42.6 against 46.0.
constexpr uint32_t PG_COUNT_PAGES = 8192;
template <bool COUNT>
__global__ __launch_bounds__(PG_PLAN_NT) void k_compact_list(CompactArgs a) {
  static_assert(PG_CHUNK == PG_PLAN_NT, "a page a thread");
  __shared__ uint32_t s_wave[PG_PLAN_NT / 64];
  const uint32_t tid = threadIdx.x, p = blockIdx.x * PG_CHUNK + tid;
  uint32_t count = 0;
  PgScan sum;
  if constexpr (COUNT) {
    uint32_t below = 0, all = 0;
#pragma unroll
    for (uint32_t i = 0; i < PG_COUNT_PAGES / PG_PLAN_NT; ++i) {
      const uint32_t r = i * PG_PLAN_NT + tid < a.n_pages ? a.refs[i * PG_PLAN_NT + tid] : 0u;
      all += r != 0;
      if (i < blockIdx.x) below += r != 0;
      if (i == blockIdx.x) count = r;
    }
    const uint32_t b = pg_scan<PG_PLAN_NT>(below, s_wave).total;
    sum = PgScan{b, pg_scan<PG_PLAN_NT>(all, s_wave).total};
    if (p < a.n_pages) a.old[p] = count;
  } else {
    sum = compact_sums(a, blockIdx.x, s_wave);
    if (p < a.n_pages) count = a.old[p];
  }
  const uint32_t n_live = sum.total;
  const bool used = count != 0;
  const PgScan r = pg_scan<PG_PLAN_NT>(used, s_wave);
  if (COUNT && tid == 0) a.chunk[blockIdx.x] = r.total;
  const uint32_t below = sum.before + r.before;  // pages in use below p
  if (p >= a.n_pages) return;
  if (used && p >= n_live) {
    const uint32_t above = n_live - 1 - below;
    a.rank[p] = above;
    a.highs[above] = p;
  } else if (!used && p < n_live) {
    a.holes[p - below] = p;
  }
}

__global__ __launch_bounds__(PG_PLAN_NT) void k_compact_move(CompactArgs a) {
  __shared__ uint32_t s_wave[PG_PLAN_NT / 64];
  // holes below n_live: n_live - (pages in use below n_live)
  const uint32_t n_live = compact_sums(a, 0, s_wave).total;
  const uint32_t edge = n_live / PG_CHUNK;
  uint32_t below = compact_sums(a, edge, s_wave).before, in = 0;
  for (uint32_t p = edge * PG_CHUNK + threadIdx.x; p < n_live; p += PG_PLAN_NT) in += a.old[p] != 0;
  below += pg_scan<PG_PLAN_NT>(in, s_wave).total;
  const uint32_t total = n_live - below, moves = min(total, a.max_pairs);
  if (blockIdx.x < a.chunks) {
    for (uint32_t i = threadIdx.x; i < PG_CHUNK; i += PG_PLAN_NT) {
      const uint32_t p = blockIdx.x * PG_CHUNK + i;
      if (p >= a.n_pages) break;
      uint32_t r = a.old[p];
      if (r && p >= n_live && a.rank[p] < moves) r = 0;
      if (!a.old[p] && p < n_live) continue;  // (a hole: written by its pair, or below)
      a.refs_out[p] = r;
    }
    // pairs of this workgroup's share, and their holes' counts
    for (uint32_t k = blockIdx.x * PG_CHUNK + threadIdx.x; k < min(total, (blockIdx.x + 1) * PG_CHUNK); k += PG_PLAN_NT) {
      const uint32_t from = a.highs[k], to = a.holes[k];
      a.refs_out[to] = k < moves ? a.old[from] : 0u;
      if (k < moves) {
        a.pairs[2 * k] = from;
        a.pairs[2 * k + 1] = to;
      }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      *a.n_pairs = moves;
      if (a.extent) *a.extent = moves < total ? a.highs[moves] + 1 : n_live;
    }
    return;
  }
  // rows of the table
  const uint32_t s = blockIdx.x - a.chunks, held = a.held[s];
  const uint32_t* row = a.table + (size_t)s * a.stride;
  uint32_t* out = a.table_out + (size_t)s * a.stride;
  if (held > a.stride && threadIdx.x == 0) pages_flag(a.status, PG_BAD_LENGTH);
  for (uint32_t j = threadIdx.x; j < a.stride; j += PG_PLAN_NT) {
    uint32_t page = row[j];
    if (j < held && held <= a.stride) {
      if (page >= a.n_pages) pages_flag(a.status, PG_BAD_PAGE);
      else if (page >= n_live && a.old[page] && a.rank[page] < moves) page = a.holes[a.rank[page]];
    }
    out[j] = page;
  }
}

// ---------------------------------------------------------------------------
// Pages copied in every buffer, a workgroup a (pair, buffer).  Bound: HBM: 67 MB read and written (64 pairs of 16
// buffers of 32 KB) in 10.8 us, 268 MB (512 pairs of 16 of 16 KB) in 56 us, past the caches.
constexpr uint32_t PC_BUFFERS = 128;  // of one launch
constexpr uint32_t PC_NT = 256;
struct PageCopyArgs {
  uint8_t* buffer[PC_BUFFERS];
  uint64_t bytes[PC_BUFFERS];
  const uint32_t* pairs;
  const uint32_t* n_pairs;  // may be null: max_pairs
  uint32_t* status;
  uint32_t max_pairs, n_pages, n_buffers;
};
template <bool STREAM>
__global__ __launch_bounds__(PC_NT) void k_pages_copy(PageCopyArgs a) {
  const uint32_t n = a.n_pairs ? min(*a.n_pairs, a.max_pairs) : a.max_pairs;
  const uint32_t b = blockIdx.x % a.n_buffers;
  for (uint32_t k = blockIdx.x / a.n_buffers; k < n; k += gridDim.x / a.n_buffers) {
    const uint32_t from = a.pairs[2 * k], to = a.pairs[2 * k + 1];
    if (from >= a.n_pages || to >= a.n_pages) {
      if (threadIdx.x == 0) pages_flag(a.status, PG_BAD_PAGE);
      continue;
    }
    const uint8_t* src = a.buffer[b] + from * a.bytes[b];
    uint8_t* dst = a.buffer[b] + to * a.bytes[b];
    if (((reinterpret_cast<uintptr_t>(a.buffer[b]) | a.bytes[b]) & 15u) == 0) {
      const uint64_t units = a.bytes[b] / 16;
      const rk_u32x4* from16 = reinterpret_cast<const rk_u32x4*>(src);
      rk_u32x4* to16 = reinterpret_cast<rk_u32x4*>(dst);
      for (uint64_t i = threadIdx.x; i < units; i += 4 * PC_NT) {  // 4 a thread on their way
        rk_u32x4 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + j * PC_NT < units) x[j] = STREAM ? __builtin_nontemporal_load(from16 + i + j * PC_NT) : from16[i + j * PC_NT];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + j * PC_NT < units) {
            if (STREAM) __builtin_nontemporal_store(x[j], to16 + i + j * PC_NT);
            else to16[i + j * PC_NT] = x[j];
          }
      }
    } else {
      for (uint64_t i = threadIdx.x; i < a.bytes[b]; i += PC_NT) dst[i] = src[i];
    }
  }
}

}  // namespace cm
