// Trees of drafted tokens: the rows that a node sees, and what follows the model's answers.
//
// A request's chunk is its tree: node 0 the root (the last token that is certain), node i a drafted token whose parent
// is an earlier node.  With the model's answer to every node, the accepted path goes from the root to the first child
// whose token is its parent's answer, and so on; the nodes' rows in the pool, cached + i, then move together to cached,
// cached + 1, ...  The first 64 nodes count.
#include "chunk_device.h"
#include "uocr_kernels.h"

namespace uocr {

namespace {

constexpr int kNodes = 64;  // a lane each
constexpr int kThreads = 256;

struct Request {
  int first, end;
};
__device__ __forceinline__ Request request_of(const int32_t* offsets, int n, int tokens) {
  return {ldg(offsets + n), min(ldg(offsets + n + 1), tokens)};
}

// One wave a request: every node's ancestors by pointers that double their reach.  Bound by its launch.
__global__ void __launch_bounds__(kWave) k_draft_masks(int64_t* masks, const int32_t* parents, const int32_t* offsets, int tokens) {
  const Request q = request_of(offsets, (int)blockIdx.x, tokens);
  if (q.first < 0) return;
  const int lane = lane_id(), length = q.end - q.first;
  int up = lane > 0 && lane < length ? ldg(parents + q.first + lane) : -1;
  if (up >= lane) up = -1;
  uint64_t mask = 1ull << lane;
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    const int at = max(up, 0);
    const uint64_t above = (uint64_t)(uint32_t)__shfl((int)(mask >> 32), at, kWave) << 32 | (uint32_t)__shfl((int)mask, at, kWave);
    const int next = __shfl(up, at, kWave);
    if (up >= 0) {
      mask |= above;
      up = next;
    }
  }
  if (lane < length) stg(masks + q.first + lane, (int64_t)mask);
  for (int i0 = kNodes; i0 < length; i0 += kNodes) {  // further tokens see what a parent among the first sees
    const int i = i0 + lane, p = i < length ? ldg(parents + q.first + i) : -1, at = p >= 0 && p < kNodes ? p : 0;
    const uint64_t above = (uint64_t)(uint32_t)__shfl((int)(mask >> 32), at, kWave) << 32 | (uint32_t)__shfl((int)mask, at, kWave);
    if (i < length) stg(masks + q.first + i, p >= 0 && p < kNodes ? (int64_t)above : 0);
  }
}

// A workgroup has a request, a layer's k or v, and 256 16-byte pieces of its rows; every wave follows the path for
// itself (a step is a broadcast and a ballot).  Each row moves towards the front and the path ascends, so a thread
// reads every row before it is overwritten.  Bound by trips to memory, the path's words, then the table's, then the rows: 3 us
// for one tree over 12 layers, 6 for 24 trees.
constexpr int kAtOnce = 8;  // rows whose loads are under way together
__global__ void __launch_bounds__(kThreads) k_accept_drafts(AcceptDrafts p, Divide by_page) {
  const int n = (int)blockIdx.x, lane = lane_id();
  const Request q = request_of(p.offsets, n, p.tokens);
  const int length = q.first < 0 ? 0 : max(q.end - q.first, 0);
  const bool node = lane < length;
  const int parent = node ? ldg(p.parents + q.first + lane) : -1, token = node ? ldg(p.drafted + q.first + lane) : 0;
  const int answer = node ? ldg(p.answers + q.first + lane) : -1;
  const int cached = (int)min(ldg(p.cache_lengths + n), (uint32_t)p.max_rows);
  uint64_t path = length > 0 ? 1 : 0;
  int at = 0;
  while (path != 0) {
    const int want = __builtin_amdgcn_readlane(answer, at);
    const uint64_t next = __ballot(node && lane > at && parent == at && token == want);
    if (next == 0) break;
    at = __builtin_ctzll(next);
    path |= 1ull << at;
  }
  const int count = __popcll(path);
  if (blockIdx.y == 0 && blockIdx.z == 0) {  // the request's words
    if (threadIdx.x == 0) {
      stg(p.counts + n, count);
      stg(p.next + n, __builtin_amdgcn_readlane(answer, at));
      stg(p.lengths_out + n, (uint32_t)cached + (uint32_t)count);
    }
    if (threadIdx.x < kWave) {  // node `lane` of the path at its place
      if (path >> lane & 1) stg(p.path + q.first + lanes_below(path), lane);
      if (node && lane >= count) stg(p.path + q.first + lane, -1);
    }
    for (int i = kNodes + (int)threadIdx.x; i < length; i += kThreads) stg(p.path + q.first + i, -1);
    if (n == 0)  // tokens of no chunk
      for (int i = (int)threadIdx.x; i < min(q.first, p.tokens); i += kThreads) stg(p.path + i, -1);
    if (n == (int)gridDim.x - 1)
      for (int i = max(q.end, 0) + (int)threadIdx.x; i < p.tokens; i += kThreads) stg(p.path + i, -1);
  }
  const int piece = (int)blockIdx.z * kThreads + (int)threadIdx.x;
  if (piece >= p.slot_bytes / 16) return;
  const int64_t plane = (int64_t)blockIdx.y * p.page_size * p.slot_bytes + 16 * (int64_t)piece;
  const int64_t page_bytes = 2 * (int64_t)p.layers * p.page_size * p.slot_bytes;
  const auto row = [&](int r) {
    const int col = by_page(r);
    const uint32_t page = min(ldc(p.lookup + (int64_t)n * p.lookup_cols + col), (uint32_t)(p.pages - 1));
    return p.pool + (int64_t)page * page_bytes + plane + (int64_t)(r - col * p.page_size) * p.slot_bytes;
  };
  // nodes that are where they belong already come first; rows that the table does not address stay
  int i = path == ~0ull ? kNodes : __builtin_ctzll(~path);
  uint64_t left = i == kNodes ? 0 : path >> i << i;
  if (p.max_rows - cached < kNodes) left &= (1ull << (p.max_rows - cached)) - 1;
  for (int rows = __popcll(left); rows > 0; rows -= kAtOnce, i += kAtOnce) {
    f32x4 v[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {  // (behind the last row, the last again)
      v[u] = *(const UOCR_GLOBAL f32x4*)row(cached + __builtin_ctzll(left));
      left = (left & (left - 1)) != 0 ? left & (left - 1) : left;
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
      if (u < rows) *(UOCR_GLOBAL f32x4*)row(cached + i + u) = v[u];
  }
}

}  // namespace

hipError_t launch_draft_masks(int64_t* masks, const int32_t* parents, const int32_t* offsets, int requests, int tokens,
                              hipStream_t s) {
  if (requests == 0 || tokens == 0) return hipSuccess;
  UOCR_LAUNCH("draft_masks", k_draft_masks, dim3((unsigned)requests), dim3(kWave), 0, s, masks, parents, offsets, tokens);
  return hipGetLastError();
}

hipError_t launch_accept_drafts(const AcceptDrafts& p, int requests, hipStream_t s) {
  if (requests == 0) return hipSuccess;
  const dim3 grid((unsigned)requests, (unsigned)(2 * p.layers), (unsigned)((p.slot_bytes / 16 + kThreads - 1) / kThreads));
  UOCR_LAUNCH("accept_drafts", k_accept_drafts, grid, dim3(kThreads), 0, s, p, divide_by(p.page_size));
  return hipGetLastError();
}

}  // namespace uocr
