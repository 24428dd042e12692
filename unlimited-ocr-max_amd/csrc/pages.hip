// The pages of the KV pool: copies, forks, growth and release, compaction (the pool and
// its page lists of unlimited_ocr_max/kv_cache.py:1-36, :210-335, which the reference
// keeps on the host).
//
//   pool    kv_blocks [pages][2 (k, v)][layers][P][slot floats]; the last page is the null page
//   lookup  [requests][cols]: column c of a row is the page of its logical rows [cP, cP + P);
//           an entry outside [0, pages - 1) is unset (unset entries are written as pages - 1)
//   counts  [pages]: the entries that name each page; <= 0: free
//
// The table kernels are one workgroup each: a fork, a resize and a compaction are scans
// over the counts and the table in a fixed order, so that which page an entry gets does
// not depend on timing.  What they decide to copy goes, as (source, destination, rows)
// triples, to a second launch over the whole device.
#include "uocr_device.h"
#include "uocr_kernels.h"

namespace uocr {

namespace {

constexpr int kTableThreads = 1024;
constexpr int kTableWaves = kTableThreads / kWave;
constexpr int kCopyThreads = 256;
constexpr int kSegment = 4 * kCopyThreads;  // float4s of one plane that a workgroup copies at a time

// The rank of this thread among the workgroup's threads whose flag is set, and their number.
__device__ __forceinline__ int block_rank(bool flag, int* totals, int& all) {
  const uint64_t set = __ballot(flag);
  if (lane_id() == 0) totals[threadIdx.x / kWave] = __popcll(set);
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kTableWaves; ++w) {
    before += w < (int)threadIdx.x / kWave ? totals[w] : 0;
    all += totals[w];
  }
  __syncthreads();
  return before + lanes_below(set);
}

// Counts change by atomics, which act past the CU's L1: they are read the same way.
__device__ __forceinline__ int32_t count_of(int32_t* c) {
  return __hip_atomic_load(c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void set_count(int32_t* c, int32_t v) {
  __hip_atomic_store(c, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void release(int32_t* c) {  // never below zero
  int32_t old = count_of(c);
  while (old > 0 && !__hip_atomic_compare_exchange_strong(c, &old, old - 1, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                                          __HIP_MEMORY_SCOPE_AGENT)) {
  }
}

// The free pages in ascending order into `list`; returns their number (to every thread).
__device__ __forceinline__ int list_free(int32_t* counts, int null, int32_t* list, int* totals) {
  int found = 0;
  for (int p0 = 0; p0 < null; p0 += kTableThreads) {
    const int p = p0 + (int)threadIdx.x;
    const bool free = p < null && count_of(counts + p) <= 0;
    int all;
    const int rank = block_rank(free, totals, all);
    if (free) list[found + rank] = p;
    found += all;
  }
  return found;
}

__device__ __forceinline__ int pages_for(int32_t rows, int P, int cols) {
  return rows <= 0 ? 0 : min((rows - 1) / P + 1, cols);
}

// Every request gets exactly the pages of its length: entries past them are released,
// then missing ones are taken, in (request, column) order, from the free pages in
// ascending order (the released ones among them).
__global__ void __launch_bounds__(kTableThreads) k_resize(PageTables t, int pages, int P,
                                                          const int32_t* __restrict__ lengths, int32_t* missing,
                                                          int32_t* list) {
  __shared__ int totals[kTableWaves];
  const int null = pages - 1, tid = (int)threadIdx.x;
  const int64_t entries = (int64_t)t.requests * t.cols;
  if (t.counts_out != t.counts)
    for (int p = tid; p < pages; p += kTableThreads) set_count(t.counts_out + p, t.counts[p]);
  __syncthreads();
  for (int64_t e = tid; e < entries; e += kTableThreads) {
    const uint32_t page = t.lookup[e];
    const bool set = page < (uint32_t)null;
    const bool need = (int)(e % t.cols) < pages_for(lengths[e / t.cols], P, t.cols);
    if (set && !need) release(t.counts_out + page);
    t.lookup_out[e] = set && need ? page : (uint32_t)null;
  }
  __syncthreads();
  const int free = list_free(t.counts_out, null, list, totals);
  __syncthreads();
  int taken = 0;
  for (int64_t e0 = 0; e0 < entries; e0 += kTableThreads) {
    const int64_t e = e0 + tid;
    // this thread wrote the entry above
    const bool want = e < entries && t.lookup_out[e] == (uint32_t)null &&
                      (int)(e % t.cols) < pages_for(lengths[e / t.cols], P, t.cols);
    int all;
    const int rank = taken + block_rank(want, totals, all);
    if (want && rank < free) {
      t.lookup_out[e] = (uint32_t)list[rank];
      set_count(t.counts_out + list[rank], 1);
    }
    taken += all;
  }
  if (tid == 0) missing[0] = max(0, taken - free);
}

struct ForkScratch {
  int32_t* moves;   // [0]: pages to copy
  int32_t* winner;  // [requests]: the last pair whose child the row is
  int32_t* list;    // [pages]: the free pages
  int32_t* fresh;   // [count * cols]: the children's new entries
  int32_t* plan;    // [3 * count * cols]: source, destination, rows
};

__device__ __forceinline__ bool fork_pair(const PageTables& t, const ForkScratch& w, const int32_t* parents,
                                          const int32_t* children, int c, int& parent, int& child) {
  parent = parents[c];
  child = children[c];
  return (uint32_t)parent < (uint32_t)t.requests && (uint32_t)child < (uint32_t)t.requests && parent != child &&
         w.winner[child] == c;
}

// Each child's row becomes its parent's, as the table was before the call: pages wholly
// below shared_rows are shared, the others up to the length are copied to pages that were
// free before the call, in (pair, column) order from the lowest; then the child's old
// pages are released.
__global__ void __launch_bounds__(kTableThreads) k_fork(PageTables t, int pages, int P,
                                                        const int32_t* __restrict__ parents,
                                                        const int32_t* __restrict__ children,
                                                        const int32_t* __restrict__ lengths,
                                                        const int32_t* __restrict__ shared_rows, int count,
                                                        int32_t* missing, ForkScratch w) {
  __shared__ int totals[kTableWaves];
  const int null = pages - 1, tid = (int)threadIdx.x;
  if (t.counts_out != t.counts)
    for (int p = tid; p < pages; p += kTableThreads) set_count(t.counts_out + p, t.counts[p]);
  if (t.lookup_out != t.lookup)
    for (int64_t e = tid; e < (int64_t)t.requests * t.cols; e += kTableThreads) t.lookup_out[e] = t.lookup[e];
  for (int n = tid; n < t.requests; n += kTableThreads) set_count(w.winner + n, -1);
  __syncthreads();
  for (int c = tid; c < count; c += kTableThreads)
    if ((uint32_t)children[c] < (uint32_t)t.requests)
      __hip_atomic_fetch_max(w.winner + children[c], c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const int free = list_free(t.counts_out, null, w.list, totals);
  __syncthreads();
  const int64_t entries = (int64_t)count * t.cols;
  int taken = 0;
  for (int64_t e0 = 0; e0 < entries; e0 += kTableThreads) {
    const int64_t e = e0 + tid;
    const int c = (int)(min(e, entries - 1) / t.cols), col = (int)(e % t.cols);
    int parent, child;
    const bool pair = e < entries && fork_pair(t, w, parents, children, c, parent, child);
    const uint32_t old = pair ? t.lookup[(int64_t)parent * t.cols + col] : (uint32_t)null;
    const bool held = old < (uint32_t)null && col < pages_for(lengths[c], P, t.cols);
    const bool share = held && col < max(shared_rows[c], 0) / P;
    const bool copy = held && !share;
    int all;
    const int rank = taken + block_rank(copy, totals, all);
    uint32_t page = share ? old : (uint32_t)null;
    if (copy && rank < free) {
      page = (uint32_t)w.list[rank];
      w.plan[3 * (int64_t)rank] = (int32_t)old;
      w.plan[3 * (int64_t)rank + 1] = (int32_t)page;
      w.plan[3 * (int64_t)rank + 2] = min(P, lengths[c] - col * P);
      set_count(t.counts_out + page, 1);
    }
    if (share) __hip_atomic_fetch_add(t.counts_out + page, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (e < entries) w.fresh[e] = (int32_t)page;
    taken += all;
  }
  __syncthreads();  // every new entry is counted before an old one is released
  for (int64_t e = tid; e < entries; e += kTableThreads) {
    const int c = (int)(e / t.cols), col = (int)(e % t.cols);
    int parent, child;
    if (!fork_pair(t, w, parents, children, c, parent, child)) continue;
    const int64_t at = (int64_t)child * t.cols + col;
    const uint32_t old = t.lookup[at];  // in place: this thread alone writes the entry
    if (old < (uint32_t)null) release(t.counts_out + old);
    t.lookup_out[at] = (uint32_t)w.fresh[e];
  }
  if (tid == 0) {
    w.moves[0] = min(taken, free);
    missing[0] = max(0, taken - free);
  }
}

// The pages in use move to the front: with L of them, those at or past L go, in ascending
// order, to the free ones below L in ascending order.
__global__ void __launch_bounds__(kTableThreads) k_compact(PageTables t, int pages, int P, int32_t* remap,
                                                           int32_t* moves, int32_t* plan) {
  __shared__ int totals[kTableWaves];
  const int null = pages - 1, tid = (int)threadIdx.x;
  int live = 0;
  for (int p0 = 0; p0 < null; p0 += kTableThreads) {
    int all;
    block_rank(p0 + tid < null && t.counts[min(p0 + tid, null)] > 0, totals, all);
    live += all;
  }
  int from = 0, to = 0;
  for (int p0 = 0; p0 < null; p0 += kTableThreads) {
    const int p = p0 + tid;
    const bool used = p < null && t.counts[min(p, null)] > 0;
    const bool source = used && p >= live, hole = p < null && !used && p < live;
    int n_from, n_to;
    const int i = from + block_rank(source, totals, n_from), j = to + block_rank(hole, totals, n_to);
    if (source) {
      plan[3 * (int64_t)i] = p;
      plan[3 * (int64_t)i + 2] = P;
    }
    if (hole) plan[3 * (int64_t)j + 1] = p;
    if (p < null) remap[p] = used ? p : -1;
    if (p < null && t.counts_out != t.counts) t.counts_out[p] = t.counts[p];
    from += n_from;
    to += n_to;
  }
  if (tid == 0) {
    remap[null] = null;
    if (t.counts_out != t.counts) t.counts_out[null] = t.counts[null];
    moves[0] = from;
  }
  __syncthreads();
  for (int i = tid; i < from; i += kTableThreads) {
    const int src = plan[3 * (int64_t)i], dst = plan[3 * (int64_t)i + 1];
    const int32_t held = t.counts[src];
    remap[src] = dst;
    t.counts_out[dst] = held;
    t.counts_out[src] = 0;
  }
  __syncthreads();
  for (int64_t e = tid; e < (int64_t)t.requests * t.cols; e += kTableThreads) {
    const uint32_t page = t.lookup[e];
    const int32_t now = page < (uint32_t)null ? remap[page] : null;
    t.lookup_out[e] = (uint32_t)(now < 0 ? null : now);
  }
}

// The planned copies: (page, plane, segment) triples over the grid.  Destinations are
// distinct and no page is both a source and a destination.
__global__ void __launch_bounds__(kCopyThreads) k_copy_plan(f32x4* pool, int planes, int P, int slot4,
                                                            const int32_t* __restrict__ moves,
                                                            const int32_t* __restrict__ plan) {
  const int64_t plane4 = (int64_t)P * slot4;
  const int segments = (int)((plane4 + kSegment - 1) / kSegment);
  const int64_t items = (int64_t)ldc(moves) * planes * segments;
  for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const int seg = (int)(i % segments);
    const int64_t mp = i / segments;
    const int plane = (int)(mp % planes);
    const int32_t* m = plan + 3 * (mp / planes);
    const int64_t end = (int64_t)ldc(m + 2) * slot4;
    const f32x4* src = pool + ((int64_t)ldc(m) * planes + plane) * plane4;
    f32x4* dst = pool + ((int64_t)ldc(m + 1) * planes + plane) * plane4;
    const int64_t e0 = (int64_t)seg * kSegment + threadIdx.x;
    f32x4 v[kSegment / kCopyThreads];
#pragma unroll
    for (int u = 0; u < kSegment / kCopyThreads; ++u)
      if (e0 + u * kCopyThreads < end) v[u] = *(const UOCR_GLOBAL f32x4*)(src + e0 + u * kCopyThreads);
#pragma unroll
    for (int u = 0; u < kSegment / kCopyThreads; ++u)
      if (e0 + u * kCopyThreads < end) *(UOCR_GLOBAL f32x4*)(dst + e0 + u * kCopyThreads) = v[u];
  }
}

// Copies in the order of the pairs: a thread does its elements of every pair, one pair
// after the other, so a page may be both written and read.
__global__ void __launch_bounds__(kCopyThreads) k_copy_pages(f32x4* pool, int pages, int planes, int P, int slot4,
                                                             const int32_t* src, const int32_t* dst,
                                                             const int32_t* rows, int count) {
  const int64_t plane4 = (int64_t)P * slot4, page4 = planes * plane4;
  const int64_t e = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x;
  if (e >= page4) return;
  const int slot = (int)(e % plane4 / slot4);
  for (int i = 0; i < count; ++i) {
    const int a = ldg(src + i), b = ldg(dst + i);
    if ((uint32_t)a >= (uint32_t)pages || (uint32_t)b >= (uint32_t)pages) continue;
    if (rows != nullptr && slot >= ldg(rows + i)) continue;
    pool[b * page4 + e] = pool[a * page4 + e];
  }
}

hipError_t launch_plan(const PagePool& p, const int32_t* moves, const int32_t* plan, hipStream_t s) {
  UOCR_LAUNCH("copy_plan", k_copy_plan, dim3(2048), dim3(kCopyThreads), 0, s, (f32x4*)p.kv_blocks, 2 * p.layers,
              p.page_size, p.slot / 4, moves, plan);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_copy_pages(const PagePool& p, const int32_t* src, const int32_t* dst, const int32_t* rows,
                             int count, hipStream_t s) {
  const int64_t page4 = (int64_t)2 * p.layers * p.page_size * (p.slot / 4);
  if (count == 0) return hipSuccess;
  UOCR_LAUNCH("copy_pages", k_copy_pages, dim3((unsigned)((page4 + kCopyThreads - 1) / kCopyThreads)),
              dim3(kCopyThreads), 0, s, (f32x4*)p.kv_blocks, p.pages, 2 * p.layers, p.page_size, p.slot / 4, src, dst,
              rows, count);
  return hipGetLastError();
}

size_t fork_workspace_bytes(int64_t pages, int64_t requests, int64_t cols, int64_t count) {
  return sizeof(int32_t) * (4 + requests + pages + 4 * count * cols);
}

hipError_t launch_fork_pages(const PagePool& p, const PageTables& t, const int32_t* parents, const int32_t* children,
                             const int32_t* lengths, const int32_t* shared_rows, int count, int32_t* missing,
                             void* workspace, hipStream_t s) {
  ForkScratch w{};
  w.moves = (int32_t*)workspace;
  w.winner = w.moves + 4;
  w.list = w.winner + t.requests;
  w.fresh = w.list + p.pages;
  w.plan = w.fresh + (int64_t)count * t.cols;
  UOCR_LAUNCH("fork_tables", k_fork, dim3(1), dim3(kTableThreads), 0, s, t, p.pages, p.page_size, parents, children,
              lengths, shared_rows, count, missing, w);
  if (count == 0) return hipGetLastError();
  return launch_plan(p, w.moves, w.plan, s);
}

size_t resize_workspace_bytes(int64_t pages) { return sizeof(int32_t) * pages; }

hipError_t launch_resize_pages(const PagePool& p, const PageTables& t, const int32_t* lengths, int32_t* missing,
                               void* workspace, hipStream_t s) {
  UOCR_LAUNCH("resize_tables", k_resize, dim3(1), dim3(kTableThreads), 0, s, t, p.pages, p.page_size, lengths, missing,
              (int32_t*)workspace);
  return hipGetLastError();
}

// At most half of the pages move.
size_t compact_workspace_bytes(int64_t pages) { return sizeof(int32_t) * (4 + 3 * (pages / 2 + 1)); }

hipError_t launch_compact_pages(const PagePool& p, const PageTables& t, int32_t* remap, void* workspace,
                                hipStream_t s) {
  int32_t* moves = (int32_t*)workspace;
  int32_t* plan = moves + 4;
  UOCR_LAUNCH("compact_tables", k_compact, dim3(1), dim3(kTableThreads), 0, s, t, p.pages, p.page_size, remap, moves,
              plan);
  return launch_plan(p, moves, plan, s);
}

}  // namespace uocr
