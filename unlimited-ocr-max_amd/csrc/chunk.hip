// Attention of a chunk of new tokens over the KV page pool: the prompt's form of
// the decode op (unlimited_ocr_max/decoder.py:425-437, store_k/v_cache_ragged then
// flash_attention_ragged under the causal mask; the pool and its row mapping of
// unlimited_ocr_max/kv_cache.py:1-36).
//
// N requests; request n's chunk is token rows [off[n], off[n + 1]) and follows its
// c_n cached rows.  Token i of it is the request's logical row c_n + i: its k and v
// are stored there, and it attends rows [0, c_n + i]:
//   out = sum_r softmax_r(scale * q.k_r) v_r      (fp32, D = 128).
//
// k_chunk_store writes the new rows into the pool (rotating q and k first where
// they come unrotated; the rotated q waits in out), so the attention reads every
// row from the pool.
//
// k_chunk_rows: one wave per (token, head), a float2 of the head dim per lane, one
// pass with a running maximum and sum.
#include "uocr_device.h"
#include "uocr_kernels.h"

namespace uocr {

namespace {

constexpr int kD = 128;
constexpr int kWavesRows = 4;   // waves (token, head pairs) of a k_chunk_rows workgroup
constexpr int kKeysAtOnce = 8;  // rows whose loads are in flight together

struct ChunkArgs {
  float* pool;
  int64_t page_stride;  // floats per page: 2 * layers * P * heads * D
  int64_t kv_stride;    // floats between the k and v halves of a page
  int64_t layer_off;    // floats to the layer
  int64_t slot_stride;  // floats per slot: heads * D
  int P;
  int heads;
  int pages;     // page ids at or past this are clamped to the last page (the null page)
  int max_rows;  // lookup_cols * P: rows a lookup row can address
  const uint32_t* lookup;
  int lookup_cols;
  int requests;
  const uint32_t* cache_lengths;
  const int32_t* offsets;  // [requests + 1]
  int tokens;
  int attend_max;
  int64_t in_stride;  // floats between rows of q / k_new / v_new
};

// The request whose chunk holds token t, its first token and its cached rows; false
// where none does.  Offsets are device data: whatever they hold, the request is in range.
__device__ __forceinline__ bool request_of(const ChunkArgs& a, int t, int& n, int& first, int64_t& row) {
  int lo = 0, hi = a.requests;  // the last n < requests with off[n] <= t (an empty chunk's offset is its successor's)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (ldg(a.offsets + mid) <= t) lo = mid;
    else hi = mid;
  }
  n = lo;
  first = ldg(a.offsets + n);
  if (first < 0 || first > t || ldg(a.offsets + n + 1) <= t) return false;
  const uint32_t cached = min(ldg(a.cache_lengths + n), (uint32_t)a.max_rows);
  row = (int64_t)cached + (t - first);
  return true;
}

__device__ __forceinline__ float* row_ptr(const ChunkArgs& a, int n, int h, int r, int kv) {
  const uint32_t page = min(ldg(a.lookup + (int64_t)n * a.lookup_cols + r / a.P), (uint32_t)(a.pages - 1));
  return a.pool + (int64_t)page * a.page_stride + kv * a.kv_stride + a.layer_off +
         (int64_t)(r % a.P) * a.slot_stride + (int64_t)h * kD;
}

// Thread (token, head, d < 64): the pair (d, d + 64) of k and v into the pool, and, given
// positions, of q into out, q and k rotated with k_rope's arithmetic (each product and the
// sum rounded, no contraction).
__global__ void __launch_bounds__(256) k_chunk_store(ChunkArgs a, float* __restrict__ out, const float* q,
                                                     const float* k_new, const float* v_new,
                                                     const int32_t* __restrict__ positions,
                                                     const float* __restrict__ cos_t,
                                                     const float* __restrict__ sin_t, int table_rows) {
#pragma clang fp contract(off)
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int d = (int)(i % 64);
  const int64_t th = i / 64;  // token * heads + head
  if (th >= (int64_t)a.tokens * a.heads) return;
  const int t = (int)(th / a.heads), h = (int)(th % a.heads);
  int n, first;
  int64_t row;
  if (!request_of(a, t, n, first, row)) return;
  const int64_t src = (int64_t)t * a.in_stride + (int64_t)h * kD;
  float kl = ldg(k_new + src + d), kh = ldg(k_new + src + d + 64);
  const float vl = ldg(v_new + src + d), vh = ldg(v_new + src + d + 64);
  if (positions != nullptr) {
    const int pos = min(max(ldg(positions + t), 0), table_rows - 1);
    const float cl = ldg(cos_t + (int64_t)pos * kD + d), ch = ldg(cos_t + (int64_t)pos * kD + d + 64);
    const float sl = ldg(sin_t + (int64_t)pos * kD + d), sh = ldg(sin_t + (int64_t)pos * kD + d + 64);
    const float l = kl, u = kh;
    kl = l * cl + (-u) * sl;
    kh = u * ch + l * sh;
    const float ql = ldg(q + src + d), qu = ldg(q + src + d + 64);
    out[th * kD + d] = ql * cl + (-qu) * sl;
    out[th * kD + d + 64] = qu * ch + ql * sh;
  }
  if (row >= a.max_rows) return;  // past what the lookup row addresses: not stored
  float* kp = row_ptr(a, n, h, (int)row, 0);
  kp[d] = kl;
  kp[d + 64] = kh;
  kp[a.kv_stride + d] = vl;
  kp[a.kv_stride + d + 64] = vh;
}

__global__ void __launch_bounds__(64 * kWavesRows) k_chunk_rows(ChunkArgs a, float* out, const float* q,
                                                                int64_t q_stride, float scale) {
  const int64_t th = (int64_t)blockIdx.x * kWavesRows + threadIdx.x / 64;
  if (th >= (int64_t)a.tokens * a.heads) return;
  const int t = (int)(th / a.heads), h = (int)(th % a.heads), lane = lane_id();
  int n, first;
  int64_t row;
  if (!request_of(a, t, n, first, row)) return;
  const int len = (int)min(row + 1, (int64_t)a.attend_max);
  const float* qp = q + (int64_t)t * q_stride + (int64_t)h * kD + 2 * lane;
  const float q0 = qp[0], q1 = qp[1];
  float m = -__builtin_huge_valf(), l = 0.0f, o0 = 0.0f, o1 = 0.0f;
  for (int r0 = 0; r0 < len; r0 += kKeysAtOnce) {
    float s[kKeysAtOnce], v0[kKeysAtOnce], v1[kKeysAtOnce];
    float mb = -__builtin_huge_valf();
#pragma unroll
    for (int j = 0; j < kKeysAtOnce; ++j) {
      const float* kp = row_ptr(a, n, h, min(r0 + j, len - 1), 0) + 2 * lane;
      s[j] = __builtin_fmaf(q1, ldg(kp + 1), q0 * ldg(kp));
      v0[j] = ldg(kp + a.kv_stride);
      v1[j] = ldg(kp + a.kv_stride + 1);
    }
#pragma unroll
    for (int j = 0; j < kKeysAtOnce; ++j) {
      s[j] = tree_sum(s[j]) * scale;
      if (r0 + j < len) mb = fmaxf(mb, s[j]);
    }
    const float mn = fmaxf(m, mb);
    const float keep = m == mn ? 1.0f : expf(m - mn);
    l *= keep;
    o0 *= keep;
    o1 *= keep;
#pragma unroll
    for (int j = 0; j < kKeysAtOnce; ++j) {
      if (r0 + j >= len) continue;  // rows past the attended ones may hold anything
      const float p = expf(s[j] - mn);
      l += p;
      o0 = __builtin_fmaf(p, v0[j], o0);
      o1 = __builtin_fmaf(p, v1[j], o1);
    }
    m = mn;
  }
  float* op = out + th * kD + 2 * lane;
  op[0] = o0 / l;
  op[1] = o1 / l;
}

}  // namespace

size_t chunk_workspace_bytes(int64_t, int64_t, int, int) { return 0; }

hipError_t launch_chunk_attention(const ChunkAttention& p, hipStream_t s) {
  if (p.tokens == 0 || p.requests == 0) return hipSuccess;
  if (p.head_dim != kD || p.page_size < 1 || p.pages < 1) return hipErrorInvalidValue;
  ChunkArgs a{};
  a.pool = p.kv_blocks;
  a.slot_stride = (int64_t)p.heads * kD;
  a.layer_off = (int64_t)p.layer * p.page_size * a.slot_stride;
  a.kv_stride = (int64_t)p.layers * p.page_size * a.slot_stride;
  a.page_stride = 2 * a.kv_stride;
  a.P = p.page_size;
  a.heads = p.heads;
  a.pages = p.pages;
  a.max_rows = p.lookup_cols * p.page_size;
  a.lookup = p.lookup;
  a.lookup_cols = p.lookup_cols;
  a.requests = (int)p.requests;
  a.cache_lengths = p.cache_lengths;
  a.offsets = p.chunk_offsets;
  a.tokens = (int)p.tokens;
  a.attend_max = p.attend_max;
  a.in_stride = p.in_stride;
  const int64_t pairs = p.tokens * p.heads;
  UOCR_LAUNCH("chunk_store", k_chunk_store, dim3((unsigned)((pairs * 64 + 255) / 256)), dim3(256), 0, s, a, p.out,
              p.q, p.k_new, p.v_new, p.positions, p.cos_table, p.sin_table, p.table_rows);
  const bool rotated = p.positions != nullptr;
  UOCR_LAUNCH("chunk_rows", k_chunk_rows, dim3((unsigned)((pairs + kWavesRows - 1) / kWavesRows)),
              dim3(64 * kWavesRows), 0, s, a, p.out, rotated ? p.out : p.q,
              rotated ? (int64_t)p.heads * kD : p.in_stride, p.scale);
  return hipGetLastError();
}

}  // namespace uocr
