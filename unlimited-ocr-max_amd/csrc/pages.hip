// The pages of the KV pool: copies, forks, growth and release, compaction (the pool and
// its page lists of unlimited_ocr_max/kv_cache.py:1-36, :210-335, which the reference
// keeps on the host).
//
//   pool    kv_blocks [pages][2 (k, v)][layers][P][slot floats]; the last page is the null page
//   lookup  [requests][cols]: column c of a row is the page of its logical rows [cP, cP + P);
//           an entry outside [0, pages - 1) is unset (unset entries are written as pages - 1)
//   counts  [pages]: the entries that name each page; <= 0: free
//
// A fork, a resize and a compaction are scans over the counts and the table by one
// workgroup, in a fixed order, so that which page an entry gets does not depend on
// timing.  Each output may be its input.  What they decide to copy goes, as (source,
// destination, rows) triples, to a second launch over the whole device; or, where the
// outputs are other tensors and the tables small, every workgroup makes the same scans
// and then its share of the copies.
#include <algorithm>

#include "uocr_device.h"
#include "uocr_kernels.h"

namespace uocr {

namespace {

constexpr int kTableThreads = 1024;
constexpr int kTableWaves = kTableThreads / kWave;
// Elements of a thread at a time, whose loads are under way together.  Few: each kernel's code is fetched cold, and more
// of it costs more than more rounds do.  A resize of 8 requests in 81 pages / of 256 of 32 pages in 6001, in us: 2
// 3.6 / 11.2, 4 4.1 / 10.8, 16 9.8 / 15.1.
constexpr int kPer = 2;
constexpr int kRound = kPer * kTableThreads;
constexpr int kCopyThreads = 256;

// Up to these sizes counts, lists and the rest of a table kernel's state are in LDS (145 KB of 160), else in memory.
constexpr int kLdsPages = 16384, kLdsRows = 4096;

// Where a table kernel works.  kEvery: every workgroup of the grid works the tables out for itself, in LDS, the first
// writes them, and all make the copies, with no launch between.  The tables' outputs are then other tensors than their
// inputs (which the others may still read), and the sizes those of one round.
enum Where { kMemory, kLds, kEvery };
constexpr int kEveryGroups = 512;  // two to a CU
template <Where kAt>
constexpr int kHeld = kAt == kMemory ? 1 : kAt == kLds ? kLdsPages : kRound;

// f(u, e) for this thread's elements e < n of the round that starts at e0.
template <typename F>
__device__ __forceinline__ void each(int64_t e0, int64_t n, F f) {
#pragma unroll
  for (int u = 0; u < kPer; ++u)
    if (e0 + u * kTableThreads < n) {
      const int64_t e = e0 + u * kTableThreads + threadIdx.x;
      if (e < n) f(u, (int)e);
    }
}

static_assert(kPer * kTableWaves <= kWave, "a lane has a total");

// Of every element of a round whose flag (bit u) is set, how many before it are (in element order), and their number.
__device__ __forceinline__ void ranks(uint32_t flags, int (&rank)[kPer], int* totals, int& all) {
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), lane = lane_id();
  uint64_t set[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    set[u] = __ballot(flags >> u & 1);
    if (lane == 0) totals[u * kTableWaves + w] = __popcll(set[u]);
  }
  __syncthreads();
  // element order is that of the totals
  const int mine = lane < kPer * kTableWaves ? totals[lane] : 0, upto = wave_scan_i(mine);
  all = __builtin_amdgcn_readlane(upto, 63);
#pragma unroll
  for (int u = 0; u < kPer; ++u)
    rank[u] = __builtin_amdgcn_readlane(upto - mine, u * kTableWaves + w) + lanes_below(set[u]);
  __syncthreads();
}

// Counts in memory change by atomics, which act past the CU's L1: they are read the same way.
template <bool kLds>
__device__ __forceinline__ int32_t count_of(int32_t* c) {
  if constexpr (kLds) return *c;
  return __hip_atomic_load(c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <bool kLds>
__device__ __forceinline__ void set_count(int32_t* c, int32_t v) {
  if constexpr (kLds)
    *c = v;
  else
    __hip_atomic_store(c, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <bool kLds>
__device__ __forceinline__ void release(int32_t* c) {  // never below zero
  constexpr int kScope = kLds ? __HIP_MEMORY_SCOPE_WORKGROUP : __HIP_MEMORY_SCOPE_AGENT;
  int32_t old = __hip_atomic_load(c, __ATOMIC_RELAXED, kScope);
  while (old > 0 && !__hip_atomic_compare_exchange_strong(c, &old, old - 1, __ATOMIC_RELAXED, __ATOMIC_RELAXED, kScope)) {
  }
}

// The call's counts to where they are worked on (in memory: counts_out, which may hold them already).
template <bool kLds>
__device__ __forceinline__ void load_counts(const PageTables& t, int pages, int32_t* counts) {
  if (!kLds && counts == t.counts) return;
  for (int64_t p0 = 0; p0 < pages; p0 += kRound) {
    int32_t v[kPer];
    each(p0, pages, [&](int u, int p) { v[u] = ldg(t.counts + p); });
    each(p0, pages, [&](int u, int p) { set_count<kLds>(counts + p, v[u]); });
  }
}

// The free pages in ascending order into `list`; returns their number (to every thread).
template <bool kLds>
__device__ __forceinline__ int list_free(int32_t* counts, int null, int32_t* list, int* totals) {
  int found = 0;
  for (int64_t p0 = 0; p0 < null; p0 += kRound) {
    uint32_t free = 0;
    each(p0, null, [&](int u, int p) { free |= (uint32_t)(count_of<kLds>(counts + p) <= 0) << u; });
    int rank[kPer], all;
    ranks(free, rank, totals, all);
    each(p0, null, [&](int u, int p) {
      if (free >> u & 1) list[found + rank[u]] = p;
    });
    found += all;
  }
  __syncthreads();
  return found;
}

__device__ __forceinline__ int pages_for(int32_t rows, const Divide& by_page, int cols) {
  return rows <= 0 ? 0 : min(by_page(rows - 1) + 1, cols);
}

// Every request gets exactly the pages of its length: entries past them are released,
// then missing ones are taken, in (request, column) order, from the free pages in
// ascending order (the released ones among them).
//
// One scan over the counts and one over the entries, in rounds of 2048 elements; what bounds it is latency: where each
// is one round, a trip to memory for the counts, lengths and entries together and one for the results (8 requests in 81
// pages: 3.5 us on the device), else a trip for each round (256 requests of 32 pages in a pool of 6001, three rounds of
// counts and four of entries: 11.1).
template <bool kLds>
__global__ void __launch_bounds__(kTableThreads) k_resize(PageTables t, int pages, Divide by_page, Divide by_cols,
                                                          const int32_t* __restrict__ lengths, int32_t* missing,
                                                          int32_t* list_mem) {
  __shared__ __attribute__((aligned(16))) int totals[kPer * kTableWaves];
  __shared__ int32_t lds_counts[kLds ? kLdsPages : 1], lds_list[kLds ? kLdsPages : 1], lds_need[kLdsRows];
  int32_t* counts = kLds ? lds_counts : t.counts_out;
  int32_t* list = kLds ? lds_list : list_mem;
  const int null = pages - 1;
  const int64_t entries = (int64_t)t.requests * t.cols;
  const bool once = entries <= kRound;
  uint32_t old[kPer];
  if (once) each(0, entries, [&](int u, int e) { old[u] = ldg(t.lookup + e); });
  const bool listed = t.requests <= kLdsRows;
  if (listed)
    for (int n = (int)threadIdx.x; n < t.requests; n += kTableThreads)
      lds_need[n] = pages_for(ldg(lengths + n), by_page, t.cols);
  load_counts<kLds>(t, pages, counts);
  __syncthreads();
  // whether an entry lies below its request's length
  auto needed = [&](int e) {
    const int n = by_cols(e);
    return e - n * t.cols < (listed ? lds_need[n] : pages_for(ldg(lengths + n), by_page, t.cols));
  };
  for (int64_t e0 = 0; e0 < entries; e0 += kRound) {
    if (!once) each(e0, entries, [&](int u, int e) { old[u] = ldg(t.lookup + e); });
    each(e0, entries, [&](int u, int e) {
      if (old[u] < (uint32_t)null && !needed(e)) release<kLds>(counts + old[u]);
    });
  }
  __syncthreads();
  const int free = list_free<kLds>(counts, null, list, totals);
  int taken = 0;
  for (int64_t e0 = 0; e0 < entries; e0 += kRound) {
    if (!once) each(e0, entries, [&](int u, int e) { old[u] = ldg(t.lookup + e); });
    uint32_t want = 0;
    each(e0, entries, [&](int u, int e) {
      const bool need = needed(e), set = old[u] < (uint32_t)null;
      want |= (uint32_t)(need && !set) << u;
      if (!need || !set) old[u] = (uint32_t)null;
    });
    int rank[kPer], all;
    ranks(want, rank, totals, all);
    each(e0, entries, [&](int u, int e) {
      const int r = taken + rank[u];
      if ((want >> u & 1) && r < free) {
        old[u] = (uint32_t)list[r];
        set_count<kLds>(counts + old[u], 1);
      }
      t.lookup_out[e] = old[u];
    });
    taken += all;
  }
  if (threadIdx.x == 0) missing[0] = max(0, taken - free);
  if constexpr (kLds) {
    __syncthreads();
    for (int p = (int)threadIdx.x; p < pages; p += kTableThreads) t.counts_out[p] = counts[p];
  }
}

struct Move {
  int src, dst, rows;
};
struct Copies {
  f32x4* pool;
  int planes, P, slot4;
};
// The copies that a fork or a compaction comes to: (page, plane, segment) triples over the grid.  Destinations are
// distinct and no page is both a source and a destination.
template <int kThreads, typename F>
__device__ __forceinline__ void copy_moves(const Copies& c, int moves, const F& move) {
  constexpr int kAtOnce = 4, kSegment = kAtOnce * kThreads;  // float4s of one plane that a workgroup copies at a time
  const int64_t plane4 = (int64_t)c.P * c.slot4;
  const int segments = (int)((plane4 + kSegment - 1) / kSegment);
  const int64_t items = (int64_t)moves * c.planes * segments;
  for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const int seg = (int)(i % segments);
    const int64_t mp = i / segments;
    const int plane = (int)(mp % c.planes);
    const Move m = move((int)(mp / c.planes));
    const int64_t end = (int64_t)m.rows * c.slot4;
    const f32x4* src = c.pool + ((int64_t)m.src * c.planes + plane) * plane4;
    f32x4* dst = c.pool + ((int64_t)m.dst * c.planes + plane) * plane4;
    const int64_t e0 = (int64_t)seg * kSegment + threadIdx.x;
    f32x4 v[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
      if (e0 + u * kThreads < end) v[u] = *(const UOCR_GLOBAL f32x4*)(src + e0 + u * kThreads);
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
      if (e0 + u * kThreads < end) *(UOCR_GLOBAL f32x4*)(dst + e0 + u * kThreads) = v[u];
  }
}

struct ForkScratch {
  int32_t* moves;   // [0]: pages to copy
  int32_t* plan;    // [3 * count * cols]: source, destination, rows
  int32_t* fresh;   // [count * cols]: the children's new entries
  int32_t* winner;  // [requests]: the last pair whose child the row is
  int32_t* list;    // [pages]: the free pages
};

// Each child's row becomes its parent's, as the table was before the call: pages wholly
// below shared_rows are shared, the others up to the length are copied to pages that were
// free before the call, in (pair, column) order from the lowest; then the child's old
// pages are released.  Bound by latency, as k_resize is.
template <Where kAt>
__global__ void __launch_bounds__(kTableThreads) k_fork(PageTables t, int pages, int P, Divide by_page, Divide by_cols,
                                                        const int32_t* __restrict__ parents,
                                                        const int32_t* __restrict__ children,
                                                        const int32_t* __restrict__ lengths,
                                                        const int32_t* __restrict__ shared_rows, int count,
                                                        int32_t* missing, ForkScratch w, Copies copies) {
  constexpr bool kLds = kAt != kMemory;
  const bool writes = kAt != kEvery || blockIdx.x == 0;
  __shared__ __attribute__((aligned(16))) int totals[kPer * kTableWaves];
  __shared__ int32_t lds_counts[kHeld<kAt>], lds_list[kHeld<kAt>], lds_winner[kLds ? kLdsRows : 1];
  __shared__ int32_t lds_from[kAt == kEvery ? kRound : 1], lds_rows[kAt == kEvery ? kRound : 1];
  int32_t* counts = kLds ? lds_counts : t.counts_out;
  int32_t* list = kLds ? lds_list : w.list;
  int32_t* winner = kLds ? lds_winner : w.winner;
  constexpr int kScope = kLds ? __HIP_MEMORY_SCOPE_WORKGROUP : __HIP_MEMORY_SCOPE_AGENT;
  const int null = pages - 1, tid = (int)threadIdx.x;
  if (t.lookup_out != t.lookup && writes)
    for (int64_t e0 = 0; e0 < (int64_t)t.requests * t.cols; e0 += kRound) {
      uint32_t v[kPer];
      each(e0, (int64_t)t.requests * t.cols, [&](int u, int e) { v[u] = ldg(t.lookup + e); });
      each(e0, (int64_t)t.requests * t.cols, [&](int u, int e) { t.lookup_out[e] = v[u]; });
    }
  load_counts<kLds>(t, pages, counts);
  for (int n = tid; n < t.requests; n += kTableThreads) set_count<kLds>(winner + n, -1);
  __syncthreads();
  for (int c = tid; c < count; c += kTableThreads) {
    const int child = ldg(children + c);
    if ((uint32_t)child < (uint32_t)t.requests) __hip_atomic_fetch_max(winner + child, c, __ATOMIC_RELAXED, kScope);
  }
  const int free = list_free<kLds>(counts, null, list, totals);  // its barriers are the winners' too
  const int64_t entries = (int64_t)count * t.cols;
  const bool once = entries <= kRound;
  auto child_of = [&](int c) {  // the pair's child, or -1 where the pair does not count
    const int parent = ldg(parents + c), child = ldg(children + c);
    return (uint32_t)parent < (uint32_t)t.requests && (uint32_t)child < (uint32_t)t.requests && parent != child &&
                   count_of<kLds>(winner + child) == c
               ? child
               : -1;
  };
  int32_t page[kPer];
  int taken = 0;
  for (int64_t e0 = 0; e0 < entries; e0 += kRound) {
    uint32_t share = 0, copy = 0;
    each(e0, entries, [&](int u, int e) {
      const int c = by_cols(e), col = e - c * t.cols;
      const uint32_t old = child_of(c) < 0 ? null : ldg(t.lookup + (int64_t)ldg(parents + c) * t.cols + col);
      const bool held = old < (uint32_t)null && col < pages_for(ldg(lengths + c), by_page, t.cols);
      const bool whole = col < by_page(max(ldg(shared_rows + c), 0));
      share |= (uint32_t)(held && whole) << u;
      copy |= (uint32_t)(held && !whole) << u;
      page[u] = held ? (int32_t)old : null;
    });
    int rank[kPer], all;
    ranks(copy, rank, totals, all);
    each(e0, entries, [&](int u, int e) {
      const int64_t r = taken + rank[u];
      if (share >> u & 1) __hip_atomic_fetch_add(counts + page[u], 1, __ATOMIC_RELAXED, kScope);
      if (copy >> u & 1) {
        const int old = page[u], c = by_cols(e);
        page[u] = null;
        if (r < free) {
          page[u] = list[r];
          const int rows = min(P, ldg(lengths + c) - (e - c * t.cols) * P);
          if constexpr (kAt == kEvery) {  // to the free page r
            lds_from[r] = old;
            lds_rows[r] = rows;
          } else {
            w.plan[3 * r] = old;
            w.plan[3 * r + 1] = page[u];
            w.plan[3 * r + 2] = rows;
          }
          set_count<kLds>(counts + page[u], 1);
        }
      }
      if (!once) w.fresh[e] = page[u];
    });
    taken += all;
  }
  __syncthreads();  // every new entry is counted, and every row read, before an old one is released
  if constexpr (kAt == kEvery) {
    copy_moves<kTableThreads>(copies, min(taken, free), [&](int m) { return Move{lds_from[m], list[m], lds_rows[m]}; });
    if (!writes) return;
  }
  for (int64_t e = tid; e < entries; e += kTableThreads) {
    const int c = by_cols((int)e), child = child_of(c);
    const uint32_t old = child < 0 ? null : ldg(t.lookup + (int64_t)child * t.cols + (e - c * t.cols));
    if (old < (uint32_t)null) release<kLds>(counts + old);
  }
  for (int64_t e0 = 0; e0 < entries; e0 += kRound)
    each(e0, entries, [&](int u, int e) {  // in place: the entries that this thread read above
      const int c = by_cols(e), child = child_of(c);
      int now = page[u];
      if (!once) now = w.fresh[e];
      if (child >= 0) t.lookup_out[(int64_t)child * t.cols + (e - c * t.cols)] = (uint32_t)now;
    });
  if (tid == 0) {
    if constexpr (kAt != kEvery) w.moves[0] = min(taken, free);
    missing[0] = max(0, taken - free);
  }
  if constexpr (kLds) {
    __syncthreads();
    for (int p = (int)threadIdx.x; p < pages; p += kTableThreads) t.counts_out[p] = counts[p];
  }
}

// The pages in use move to the front: with L of them, those at or past L go, in ascending
// order, to the free ones below L in ascending order.  With b(p) the used pages below p,
// the free page p < L is hole p - b(p), and the used page p >= L goes to hole b(p) - b(L).
template <Where kAt>
__global__ void __launch_bounds__(kTableThreads) k_compact(PageTables t, int pages, int P, int32_t* remap,
                                                           int32_t* moves, int32_t* plan, int32_t* holes_mem,
                                                           Copies copies) {
  constexpr bool kLds = kAt != kMemory;
  const bool writes = kAt != kEvery || blockIdx.x == 0;
  __shared__ __attribute__((aligned(16))) int totals[kPer * kTableWaves];
  __shared__ int32_t lds_remap[kHeld<kAt>], lds_holes[kLds ? kHeld<kAt> / 2 : 1];
  __shared__ int32_t lds_from[kAt == kEvery ? kRound / 2 : 1];
  __shared__ int below_live;
  int32_t* holes = kLds ? lds_holes : holes_mem;
  const int null = pages - 1, tid = (int)threadIdx.x;
  int32_t v[kPer];
  int rank[kPer], live = 0;
  uint32_t used = 0;
  for (int64_t p0 = 0; p0 < null; p0 += kRound) {
    used = 0;
    each(p0, null, [&](int u, int p) { v[u] = ldg(t.counts + p); });
    each(p0, null, [&](int u, int) { used |= (uint32_t)(v[u] > 0) << u; });
    int all;
    ranks(used, rank, totals, all);
    live += all;
  }
  int before = 0;
  for (int64_t p0 = 0; p0 < null; p0 += kRound) {
    if (null > kRound) {  // else the round above was the only one
      used = 0;
      each(p0, null, [&](int u, int p) { v[u] = t.counts[p]; });
      each(p0, null, [&](int u, int) { used |= (uint32_t)(v[u] > 0) << u; });
      int all;
      ranks(used, rank, totals, all);
#pragma unroll
      for (int u = 0; u < kPer; ++u) rank[u] += before;
      before += all;
    }
    each(p0, null, [&](int u, int p) {
      if (p == live) below_live = rank[u];
      if (p < live && !(used >> u & 1)) holes[p - rank[u]] = p;
    });
    __syncthreads();
    each(p0, null, [&](int u, int p) {
      const bool in_use = used >> u & 1;
      int now = in_use ? p : -1;
      if (in_use && p >= live) {
        const int64_t i = rank[u] - below_live;
        now = holes[i];
        if constexpr (kAt == kEvery) {
          lds_from[i] = p;
        } else {
          plan[3 * i] = p;
          plan[3 * i + 1] = now;
          plan[3 * i + 2] = P;
        }
        if (writes) {
          t.counts_out[now] = v[u];
          t.counts_out[p] = 0;
        }
      } else if ((in_use || p >= live) && t.counts_out != t.counts && writes) {
        t.counts_out[p] = v[u];
      }
      if constexpr (kLds) lds_remap[p] = now;
      if (writes) remap[p] = now;
    });
  }
  __syncthreads();
  const int count = live < null ? live - below_live : 0;
  if (tid == 0 && writes) {
    remap[null] = null;
    if (t.counts_out != t.counts) t.counts_out[null] = t.counts[null];
    if constexpr (kAt != kEvery) moves[0] = count;
  }
  if constexpr (kAt == kEvery) {
    copy_moves<kTableThreads>(copies, count, [&](int m) { return Move{lds_from[m], holes[m], P}; });
    if (!writes) return;
  }
  for (int64_t e0 = 0; e0 < (int64_t)t.requests * t.cols; e0 += kRound) {
    uint32_t page[kPer];
    each(e0, (int64_t)t.requests * t.cols, [&](int u, int e) { page[u] = ldg(t.lookup + e); });
    each(e0, (int64_t)t.requests * t.cols, [&](int u, int e) {
      const int32_t now = page[u] >= (uint32_t)null ? null : kLds ? lds_remap[page[u]] : remap[page[u]];
      t.lookup_out[e] = (uint32_t)(now < 0 ? null : now);
    });
  }
}

// The planned copies, a launch of their own.
__global__ void __launch_bounds__(kCopyThreads) k_copy_plan(Copies c, const int32_t* __restrict__ moves,
                                                            const int32_t* __restrict__ plan) {
  copy_moves<kCopyThreads>(c, ldc(moves), [&](int m) {
    const int32_t* p = plan + 3 * (int64_t)m;
    return Move{ldc(p), ldc(p + 1), ldc(p + 2)};
  });
}

// Copies in the order of the pairs: a thread does its element of every pair, one pair after the other, so a page may be
// both written and read.  Bound by memory: 24 pages of 12 layers part filled 76.7 us, which is
// 4.92 TB/s of reads and writes, what a plain copy reaches; one page 5.3 us.  More loads of a thread under way (two to
// eight elements, or pairs that do not meet) are no faster or slower, 5.0 to 11.6 us
// for one page, 75.8 to 151 us for 24, 11 to 52 us (here 9.7) for 24 of one layer: the waves of a CU are enough.
__global__ void __launch_bounds__(kCopyThreads) k_copy_pages(f32x4* pool, int pages, int planes, int64_t plane4,
                                                             int slot4, const int32_t* __restrict__ src,
                                                             const int32_t* __restrict__ dst,
                                                             const int32_t* __restrict__ rows, int count) {
  const int64_t e = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x, page4 = planes * plane4;
  for (int plane = (int)blockIdx.y; plane < planes; plane += (int)gridDim.y) {
    UOCR_GLOBAL f32x4* at = (UOCR_GLOBAL f32x4*)pool + plane * plane4 + e;
    for (int i = 0; i < count; ++i) {
      const int a = ldc(src + i), b = ldc(dst + i);
      if ((uint32_t)a >= (uint32_t)pages || (uint32_t)b >= (uint32_t)pages) continue;
      const int64_t end = rows == nullptr ? plane4 : min(plane4, (int64_t)ldc(rows + i) * slot4);
      if (e < end) at[b * page4] = at[a * page4];
    }
  }
}

Copies copies_of(const PagePool& p) { return {(f32x4*)p.kv_blocks, 2 * p.layers, p.page_size, p.slot / 4}; }
hipError_t launch_plan(const PagePool& p, const int32_t* moves, const int32_t* plan, hipStream_t s) {
  UOCR_LAUNCH("copy_plan", k_copy_plan, dim3(2048), dim3(kCopyThreads), 0, s, copies_of(p), moves, plan);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_copy_pages(const PagePool& p, const int32_t* src, const int32_t* dst, const int32_t* rows,
                             int count, hipStream_t s) {
  if (count == 0) return hipSuccess;
  const int64_t plane4 = (int64_t)p.page_size * (p.slot / 4);
  const int planes = 2 * p.layers;
  const dim3 grid((unsigned)((plane4 + kCopyThreads - 1) / kCopyThreads), (unsigned)std::min(planes, 65535));
  UOCR_LAUNCH("copy_pages", k_copy_pages, grid, dim3(kCopyThreads), 0, s, (f32x4*)p.kv_blocks, p.pages, planes, plane4,
              p.slot / 4, src, dst, rows, count);
  return hipGetLastError();
}

namespace {
bool in_lds(int64_t pages, int64_t requests) { return pages <= kLdsPages && requests <= kLdsRows; }
// One launch, against the tables' and then the copies' (us, the host's call included; on the device): a fork of three
// requests 14.3 for 18.8 (6.8 for 4.5 + 1.8), a compaction of 6 requests 11.8 for 16.1 (10.8 for 3.4 + 6.4), of 24 and
// 12 layers 247 for 279 (250 for 4.9 + 273).
bool by_every(int64_t pages, int64_t requests, int64_t entries, bool in_place) {
  return !in_place && pages <= kRound && requests <= kLdsRows && entries <= kRound;
}
}  // namespace

bool in_place(const PageTables& t) {
  return t.counts == t.counts_out || (t.requests > 0 && t.lookup == t.lookup_out);
}

size_t fork_workspace_bytes(int64_t pages, int64_t requests, int64_t cols, int64_t count, bool in_place) {
  const int64_t entries = count * cols;
  if (by_every(pages, requests, entries, in_place)) return 0;
  return sizeof(int32_t) * (4 + 3 * entries + (entries > kRound ? entries : 0) +
                            (in_lds(pages, requests) ? 0 : requests + pages));
}

hipError_t launch_fork_pages(const PagePool& p, const PageTables& t, const int32_t* parents, const int32_t* children,
                             const int32_t* lengths, const int32_t* shared_rows, int count, int32_t* missing,
                             void* workspace, hipStream_t s) {
  const int64_t entries = (int64_t)count * t.cols;
  const bool every = by_every(p.pages, t.requests, entries, in_place(t));
  ForkScratch w{};
  if (!every) {
    w.moves = (int32_t*)workspace;
    w.plan = w.moves + 4;
    w.fresh = w.plan + 3 * entries;
    w.winner = w.fresh + (entries > kRound ? entries : 0);
    w.list = w.winner + t.requests;
  }
  const auto kernel = every ? k_fork<kEvery> : in_lds(p.pages, t.requests) ? k_fork<kLds> : k_fork<kMemory>;
  UOCR_LAUNCH("fork_tables", kernel, dim3(every && count > 0 ? kEveryGroups : 1), dim3(kTableThreads), 0, s, t, p.pages,
              p.page_size, divide_by(p.page_size), divide_by(t.cols), parents, children, lengths, shared_rows, count,
              missing, w, copies_of(p));
  if (every || count == 0) return hipGetLastError();
  return launch_plan(p, w.moves, w.plan, s);
}

size_t resize_workspace_bytes(int64_t pages) { return in_lds(pages, 0) ? 0 : sizeof(int32_t) * pages; }

hipError_t launch_resize_pages(const PagePool& p, const PageTables& t, const int32_t* lengths, int32_t* missing,
                               void* workspace, hipStream_t s) {
  const auto kernel = in_lds(p.pages, 0) ? k_resize<true> : k_resize<false>;
  UOCR_LAUNCH("resize_tables", kernel, dim3(1), dim3(kTableThreads), 0, s, t, p.pages, divide_by(p.page_size),
              divide_by(t.cols), lengths, missing, (int32_t*)workspace);
  return hipGetLastError();
}

// At most half of the pages move.
size_t compact_workspace_bytes(int64_t pages, bool in_place) {
  if (by_every(pages, 0, 0, in_place)) return 0;
  return sizeof(int32_t) * (4 + (in_lds(pages, 0) ? 3 : 4) * (pages / 2 + 1));
}

hipError_t launch_compact_pages(const PagePool& p, const PageTables& t, int32_t* remap, void* workspace,
                                hipStream_t s) {
  const bool every = by_every(p.pages, 0, 0, in_place(t));
  int32_t* moves = (int32_t*)workspace;
  int32_t* plan = every ? nullptr : moves + 4;
  int32_t* holes = every || in_lds(p.pages, 0) ? nullptr : plan + 3 * ((int64_t)p.pages / 2 + 1);
  const auto kernel = every ? k_compact<kEvery> : in_lds(p.pages, 0) ? k_compact<kLds> : k_compact<kMemory>;
  UOCR_LAUNCH("compact_tables", kernel, dim3(every ? kEveryGroups : 1), dim3(kTableThreads), 0, s, t, p.pages,
              p.page_size, remap, moves, plan, holes, copies_of(p));
  return every ? hipGetLastError() : launch_plan(p, moves, plan, s);
}

}  // namespace uocr
