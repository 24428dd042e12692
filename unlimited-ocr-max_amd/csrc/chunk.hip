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
// k_chunk_tiles (256 queries a workgroup) and k_chunk_few (32) run the two products on the fp16 matrix instruction,
// each operand as a pair of halves, and keep a running maximum and sum of every query (below).
#include <algorithm>

#include "uocr_device.h"
#include "uocr_kernels.h"

namespace uocr {

namespace {

constexpr int kD = 128;

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

// ------------------------------------------------------------------ fp32 products on the fp16 matrix instruction
//
// An operand x (times a power of two that brings its group's largest to [2^14, 2^15)) is held
// as hi = fp16(x), lo = fp16(x - hi): 22 bits, or 2^-39 of the group's largest where
// that is more.  hi hi + hi lo + lo hi leaves out lo lo, 2^-22 of the product at most.

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kInf = __builtin_huge_valf();
constexpr int kBlock = 32;    // rows (keys) a wave takes at a time: the rows of one matrix instruction
constexpr int kMinExp = 15;   // exponents of a group's scale: 2^(141 - e) is a normal fp32
constexpr int kMaxExp = 254;
constexpr int kLift = 7;      // weights are held as 2^kLift p: they stay above fp16's smallest
constexpr float kSlack = 8.0f;  // a maximum may lag by 2^8 before the sums are rescaled: 2^15 p at most
constexpr int kNear = 6;      // binades between value groups that the weights take up
constexpr int kRoom = 60;     // binades that a sum may stand above the values now added to it
constexpr int kSpread = 12;   // binades between the rows of one group beside hidden rows
constexpr int kAbove = 2;     // binades of the walk's scales above its first block's largest,
constexpr int kBelow = 10;    // and below the scale that a group's largest may be
constexpr int kFlag = 1 << 16;  // a group that the fp16 pairs cannot hold
constexpr int kFrag = 64 * 8;   // halves of an operand: 8 of each lane
constexpr int kMaxSplitRows = 1 << 16;  // rows of one workgroup: a bit each of their blocks in LDS

__device__ __forceinline__ uint32_t split2(float a, float b, uint32_t& lo) {
  f16x2 h;
  h.x = (_Float16)a;
  h.y = (_Float16)b;
  const uint32_t hi = __builtin_bit_cast(uint32_t, h);
  float ra, rb;  // a - hi exactly: one instruction that widens the half itself
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(hi), "v"(a));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rb) : "v"(hi), "v"(b));
  f16x2 l;
  l.x = (_Float16)ra;
  l.y = (_Float16)rb;
  lo = __builtin_bit_cast(uint32_t, l);
  return hi;
}
__device__ __forceinline__ f16x8 halves(u32x4 v) { return __builtin_bit_cast(f16x8, v); }
__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// max(m, |a|, |b|), NaN if one is.
__device__ __forceinline__ float amax3(float m, float a, float b) {
  float r;
  asm("v_maximum3_f32 %0, %1, |%2|, |%3|" : "=v"(r) : "v"(m), "v"(a), "v"(b));
  return r;
}
// Reductions in which every lane gets the result: over lanes 16 or 32 apart, and over 16 lanes in a row.
template <int OFF>
__device__ __forceinline__ uint32_t other(uint32_t v) {  // of the lane whose number differs in bit OFF, or this one's
  if constexpr (OFF == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return lane_id() < 32 ? r[1] : r[0];
  } else {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return (lane_id() & 16) == 0 ? r[1] : r[0];
  }
}
__device__ __forceinline__ float other32(float v) { return __uint_as_float(other<32>(__float_as_uint(v))); }
template <int ROR>
__device__ __forceinline__ uint32_t ror(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + ROR, 0xf, 0xf, false);
}
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = max(v, ror<8>(v));
  v = max(v, ror<4>(v));
  v = max(v, ror<2>(v));
  return max(v, ror<1>(v));
}
__device__ __forceinline__ uint32_t row_min(uint32_t v) {
  v = min(v, ror<8>(v));
  v = min(v, ror<4>(v));
  v = min(v, ror<2>(v));
  return min(v, ror<1>(v));
}
// The lane's number as the compiler cannot know it: what is computed from it inside a loop is computed there,
// and takes no register around the loop.
__device__ __forceinline__ int lane_now() {
  int l = lane_id();
  asm volatile("" : "+v"(l));
  return l;
}
__device__ __forceinline__ float pow2_of(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ int clamp_exp(uint32_t bits) {
  return min(max((int)(bits >> 23), kMinExp), kMaxExp);
}

// A wave's 32 queries of one head: lanes l and l + 32 hold query l % 32.  The products are
// S^T = K Q^T and O^T = V^T P^T, so a lane's 16 results of S^T are scores of its query, in
// the very order in which the second product wants the weights:
//   S^T register r of lane l: key 8 (r / 4) + 4 (l / 32) + r % 4;
//   slots j of step t of a B (or A) operand: the same with r = 8 t + j.
// O^T register r of o[u]: column d = 4 (8 (r / 4) + 4 (l / 32) + r % 4) + u.
struct Queries {
  f16x8 hi[8];  // the lo parts wait in LDS
  float unit;   // |scale| log2 e
  int exp;     // of the query's scale
  int limit;   // rows the query attends
  float m, l;  // running maximum (log2), sum of the weights (times 2^kLift)
  int ev;      // o is in units of 2^(ev - 141)
  int most;    // the largest exponent of the values so far
  f32x16 o[4];
};

__device__ __forceinline__ void load_queries(Queries& w, _Float16* qlo, const float* row, float scale, int limit) {
  const int h = lane_id() >> 5;
  f32x4 x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = *(const UOCR_GLOBAL f32x4*)(row + 8 * i + 4 * h);
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = amax3(amax3(m, x[i].x, x[i].y), x[i].z, x[i].w);
  const uint32_t bits = max(__float_as_uint(m), other<32>(__float_as_uint(m)));
  w.exp = clamp_exp(bits);
  const float up = __builtin_copysignf(pow2_of(141 - w.exp), scale);  // the scale's sign goes into the query
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    u32x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x4 v = x[2 * t + i] * up;
      uint32_t a, b;
      hi[2 * i] = split2(v.x, v.y, a);
      hi[2 * i + 1] = split2(v.z, v.w, b);
      lo[2 * i] = a;
      lo[2 * i + 1] = b;
    }
    w.hi[t] = halves(hi);
    *(f16x8*)(qlo + t * kFrag + lane_id() * 8) = halves(lo);
  }
  w.unit = __builtin_fabsf(scale) * 1.44269504f;
  w.limit = limit;
  w.m = -kInf;
  w.l = 0.0f;
  w.ev = w.most = kMinExp;
#pragma unroll
  for (int u = 0; u < 4; ++u) w.o[u] = f32x16{};
}

// Brings a lane's unit to where values of exponent eb can be added: at or above it, and not more
// than kNear below, as far as the sum of larger ones (2^kRoom at most) stays in range.
__device__ __forceinline__ void set_unit(Queries& w, int eb, bool attends) {
  w.most = attends ? max(w.most, eb) : w.most;
  const int need = max(eb, w.most - kRoom);
  const bool move = attends && (need > w.ev || need < w.ev - kNear);
  if (__ballot(move) == 0) return;
  const float f = move ? __builtin_ldexpf(1.0f, w.ev - need) : 1.0f;
#pragma unroll
  for (int u = 0; u < 4; ++u) w.o[u] *= f;
  w.ev = move ? need : w.ev;
}

// Moves a lane's running maximum to mx, where that is more by kSlack; returns what to take off its scores.
__device__ __forceinline__ float move_max(Queries& w, float mx) {
  mx = fmaxf(mx, other32(mx));
  const bool up = mx > w.m + kSlack;
  if (__ballot(up) != 0) {
    const float alpha = up ? __builtin_amdgcn_exp2f(w.m - mx) : 1.0f;
    w.m = up ? mx : w.m;
    w.l *= alpha;
#pragma unroll
    for (int u = 0; u < 4; ++u) w.o[u] *= alpha;
  }
  return w.m == -kInf ? 0.0f : w.m;
}

// A block that the fp16 pairs cannot hold (a value that is not finite, or rows of unlike sizes beside
// hidden ones), in fp32 and one key at a time.  stash: 32 floats a lane.
__device__ __forceinline__ void slow_block(Queries& w, const float* q, float scale, const float* k,
                                           int64_t kv_stride, int64_t slot_stride, int live, float* stash) {
  const int h = lane_id() >> 5;
  float y[16], mx = -kInf;
#pragma unroll 1
  for (int r = 0; r < 16; ++r) {
    const int key = 8 * (r / 4) + 4 * h + r % 4;
    float s = 0.0f;
    if (key < live) {
#pragma unroll 1
      for (int d = 0; d < kD; ++d) s = __builtin_fmaf(ldg(q + d), ldg(k + (int64_t)key * slot_stride + d), s);
    }
    stash[r * kWave] = key < live ? s * scale * 1.44269504f : -kInf;
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    y[r] = stash[r * kWave];
    mx = fmaxf(mx, y[r]);
  }
  const float mu = move_max(w, mx);
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const float p = __builtin_amdgcn_exp2f(y[r] - mu + (float)kLift);
    w.l += p;
    const float theirs = other32(p);
    stash[(8 * (r / 4) + r % 4) * kWave] = h == 0 ? p : theirs;  // by key, for this lane's query
    stash[(8 * (r / 4) + 4 + r % 4) * kWave] = h == 0 ? theirs : p;
  }
  const float* v = k + kv_stride;
  uint32_t most = 0;  // of the attended rows' finite values
#pragma unroll 1
  for (int i = 0; i < live * 64; ++i) {
    const uint32_t x = __float_as_uint(ldg(v + (int64_t)(i / 64) * slot_stride + 64 * h + i % 64)) & 0x7fffffffu;
    if (x < 0x7f800000u) most = max(most, x);
  }
  most = max(most, other<32>(most));
  set_unit(w, clamp_exp(most), live > 0);
  const float down = pow2_of(141 - w.ev);
#pragma unroll 1
  for (int key = 0; key < live; ++key) {
    const float p = stash[key * kWave];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const f32x4 x = *(const UOCR_GLOBAL f32x4*)(v + (int64_t)key * slot_stride + 4 * (8 * (i / 4) + 4 * h + i % 4));
#pragma unroll
      for (int u = 0; u < 4; ++u) w.o[u][i] = __builtin_fmaf(p, x[u] * down, w.o[u][i]);
    }
  }
}

struct Weights {
  f16x8 hi[2], lo[2];
};
// The products of a block, operands read a step ahead: o += P V (vf(t, u, part) gives the operands of V^T), and S^T (kf(t,
// part) those of K, ql(t) the lo parts of the queries).
template <class VF>
__device__ __forceinline__ void add_values(Queries& w, const Weights& p, const VF& vf) {
  f16x8 hi[2], lo[2];
  hi[0] = vf(0, 0, 0);
  lo[0] = vf(0, 0, 1);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int t = i / 4, u = i % 4;
    if (i < 7) {
      hi[(i + 1) & 1] = vf((i + 1) / 4, (i + 1) % 4, 0);
      lo[(i + 1) & 1] = vf((i + 1) / 4, (i + 1) % 4, 1);
    }
    __builtin_amdgcn_sched_barrier(0);
    w.o[u] = mfma(hi[i & 1], p.lo[t], w.o[u]);
    w.o[u] = mfma(lo[i & 1], p.hi[t], w.o[u]);
    w.o[u] = mfma(hi[i & 1], p.hi[t], w.o[u]);
    __builtin_amdgcn_sched_barrier(0);
  }
}
template <class KF, class QL>
__device__ __forceinline__ f32x16 scores(const Queries& w, const KF& kf, const QL& ql) {
  f32x16 s = {};
  f16x8 hi[2], lo[2], q[2];
  hi[0] = kf(0, 0);
  q[0] = ql(0);
  lo[0] = kf(0, 1);
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    if (t < 7) {
      hi[(t + 1) & 1] = kf(t + 1, 0);
      q[(t + 1) & 1] = ql(t + 1);
      lo[(t + 1) & 1] = kf(t + 1, 1);
    }
    __builtin_amdgcn_sched_barrier(0);
    s = mfma(hi[t & 1], q[t & 1], s);
    s = mfma(lo[t & 1], w.hi[t], s);
    s = mfma(hi[t & 1], w.hi[t], s);
    __builtin_amdgcn_sched_barrier(0);
  }
  return s;
}

// A block's scores with the rows that a lane's query does not attend at -inf.
__device__ __forceinline__ void hide(f32x16& s, int live, int lane) {
  if (__ballot(live < kBlock) == 0) return;
  const int mine = live - 4 * (lane >> 5);
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (8 * (r / 4) + r % 4 >= mine) s[r] = -kInf;
}
__device__ __forceinline__ float scale_of(const Queries& w, int ek) {  // > 0: hidden rows stay at -inf
  return __builtin_amdgcn_fmed3f(__builtin_ldexpf(w.unit, w.exp + (ek - 282)), 1e-37f, 3.4e38f);
}
// The largest score of the lane's query in the block's 16 rows that the lane holds.
__device__ __forceinline__ float largest_of(const f32x16& s) {
  float m[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) m[g] = fmaxf(fmaxf(s[4 * g], s[4 * g + 1]), fmaxf(s[4 * g + 2], s[4 * g + 3]));
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}
// The block's weights 2^(c s + lift) as fp16 pairs; returns their sum.
__device__ __forceinline__ float weigh(const f32x16& s, float c, float lift, Weights& out) {
  float sum = 0.0f;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    u32x4 hi, lo;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * t + 2 * j], c, lift));
      const float b = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * t + 2 * j + 1], c, lift));
      uint32_t rest;
      hi[j] = split2(a, b, rest);
      lo[j] = rest;
      sum += a + b;
    }
    out.hi[t] = halves(hi);
    out.lo[t] = halves(lo);
  }
  return sum;
}

// Where a block's groups are at scales of their own (or an earlier block moved a lane's unit).  Before the
// weights: the scores at the walk's scale, and the units of the sums.  Returns whether the block is the slow
// path's.
__device__ __forceinline__ bool apart_scores(Queries& w, f32x16& s, const int* meta, int kunit, int vunit, bool attends) {
  int any = 0, most = 0, least = kMaxExp, far = 0;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int wk = meta[g], wv = meta[4 + g];
    const int ek = wk == 0 ? kunit : wk & (kFlag - 1), ev = wv == 0 ? vunit : wv & (kFlag - 1);
    any |= wk | wv;
    most = max(most, ev);
    least = min(least, ev);
    far = max(far, ek - kunit);
#pragma unroll
    for (int r = 4 * g; r < 4 * g + 4; ++r) s[r] = __builtin_ldexpf(s[r], ek - kunit);
  }
  const bool slow = __ballot(any >= kFlag || most - least > kNear || far > kRoom) != 0;
  set_unit(w, most, attends && !slow);
  return slow;
}
// Then the weights take up the binades from w.ev to their value group's scale: the scores are moved so that the
// weights come out so, and the sum of the weights has what they lack.
__device__ __forceinline__ void apart_weights(Queries& w, f32x16& s, const int* meta, int vunit, float c, float lift) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int wv = meta[4 + g], by = min((wv == 0 ? vunit : wv & (kFlag - 1)) - w.ev, 0);
    const float lack = __builtin_ldexpf(1.0f, -by) - 1.0f, move = (float)by / c;
#pragma unroll
    for (int r = 4 * g; r < 4 * g + 4; ++r) {
      s[r] += move;
      w.l = __builtin_fmaf(lack, __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, lift)), w.l);
    }
  }
}

// ------------------------------------------------------------------ tiles of queries

// The query tiles of all chunks, numbered without a sum over the requests: tile j of request
// n is slot floor(off[n] / rows) + n + j, which no other tile is.
struct QueryTile {
  int n, first, end;  // the request, its first token and the one behind its last
  int t0;             // the tile's first token
  int cached;
};
__device__ __forceinline__ bool query_tile(const ChunkArgs& a, int rows_log2, int slot, QueryTile& q) {
  // the last n with floor(off[n] / rows) + n <= slot: 64 probes at a time
  int lo = 0, hi = a.requests;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, i = lo + lane_id() * step;
    const bool below = i < hi && (ldg(a.offsets + min(i, hi - 1)) >> rows_log2) + (int64_t)i <= slot;
    const int found = max(1, __popcll(__ballot(below)));
    lo = min(lo + (found - 1) * step, hi - 1);
    hi = min(hi, lo + step);
  }
  q.n = __builtin_amdgcn_readfirstlane(lo);
  q.first = ldc(a.offsets + q.n);
  q.end = min(ldc(a.offsets + q.n + 1), a.tokens);
  const int64_t j = (int64_t)slot - ((int64_t)(q.first >> rows_log2) + q.n);
  if (q.first < 0 || j < 0 || ((int64_t)q.first + (j << rows_log2)) >= q.end) return false;
  q.t0 = q.first + (int)(j << rows_log2);
  q.cached = (int)min(ldc(a.cache_lengths + q.n), (uint32_t)a.max_rows);
  return true;
}
// Rows that token t of the request attends.
__device__ __forceinline__ int rows_of(const ChunkArgs& a, const QueryTile& q, int t) {
  return (int)min((int64_t)q.cached + (t - q.first) + 1, (int64_t)a.attend_max);
}

// Results of one wave: into out, or, where the rows of the tile are split, normalised into part with
// their weight's logarithm, [split][token][head][D] and [split][token][head].
__device__ __forceinline__ void store_queries(const Queries& w, const ChunkArgs& a, int t, bool live, int head,
                                              int split, bool whole, float* out, float* part, float* weights) {
  const int h = lane_id() >> 5;
  const float l = w.l + other32(w.l);
  const float f = 1.0f / l;
  const int64_t th = (int64_t)t * a.heads + head;
  float* dst = (whole ? out + th * kD : part + ((int64_t)split * a.tokens * a.heads + th) * kD) + 16 * h;
  if (!live) return;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    f32x4 v;
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = __builtin_ldexpf(w.o[u][r] * f, w.ev - 141);
    *(UOCR_GLOBAL f32x4*)(dst + 32 * (r / 4) + 4 * (r % 4)) = v;
  }
  if (!whole && h == 0)  // no row attended: no weight
    weights[(int64_t)split * a.tokens * a.heads + th] = l == 0.0f ? -kInf : w.m + __builtin_amdgcn_logf(l);
}

// k_chunk_tiles: 8 waves of 32 queries each walk the rows together, a block of 32 at a time.  4 more bring the
// rows, two blocks ahead, turn them into fp16 pairs and write them to LDS as the matrix operands they will
// be, an operand's 64 lanes side by side.
constexpr int kTileWaves = 8;   // that attend
constexpr int kStageWaves = 4;  // that convert: one a SIMD, beside two that attend
constexpr int kTileLog2 = 8;    // queries of a workgroup
constexpr int kKHalves = 8 * 2 * kFrag;      // [step][part][lane][8]
constexpr int kVHalves = 2 * 4 * 2 * kFrag;  // [step][u][part][lane][8]
constexpr int kQHalves = 8 * kFrag;          // a wave's queries' lo parts, [step][lane][8]
constexpr int kLdsHalves = 2 * kKHalves + 3 * kVHalves + kTileWaves * kQHalves;

// 8 rows of a block on their way from memory to the operands in LDS: keys (lane: row l % 8, columns 32 j +
// 4 (l / 8), whose step is 2 j + l / 32) or values (lane: columns 4 (l % 32) on, rows 4 (l / 32) + j).
template <bool kValues>
struct Stage {
  f32x4 x[4];
  float m, up;
  uint32_t bits;
  int e, word;
  uint32_t at;  // this lane's offset in bytes from the block's first row

  __device__ __forceinline__ static int row_in_group(int lane) { return kValues ? 4 * (lane >> 5) : lane & 7; }
  __device__ __forceinline__ static uint32_t column(int lane) { return 16u * (kValues ? lane & 31 : lane >> 3); }
  // 32 rows are below 2^31 bytes: 32 bits of offset a lane, from a scalar base
  __device__ __forceinline__ void load(const float* base, int64_t kv_stride, uint32_t row_bytes, int group, int last,
                                       int lane) {
    const char* from = (const char*)(kValues ? base + kv_stride : base);
    if (last >= kBlock - 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[j] = kValues ? *(const UOCR_GLOBAL f32x4*)(from + (at + j * row_bytes))
                       : *(const UOCR_GLOBAL f32x4*)(from + at + 128 * j);
    } else {  // rows past the last are its copies, zeroed before they are converted
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = min(8 * group + row_in_group(lane) + (kValues ? j : 0), last);
        x[j] = *(const UOCR_GLOBAL f32x4*)(from + ((uint32_t)row * row_bytes + column(lane) + (kValues ? 0u : 128u * j)));
      }
    }
  }
  __device__ __forceinline__ void clear_past(int group, int last, int lane) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (8 * group + row_in_group(lane) + (kValues ? j : 0) > last) x[j] = f32x4{};
  }
  __device__ __forceinline__ void largest() {
    m = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = amax3(amax3(m, x[j].x, x[j].y), x[j].z, x[j].w);
  }
  __device__ __forceinline__ void of_all_lanes_1() {
    bits = __float_as_uint(m);
    bits = max(bits, other<32>(bits));
    bits = max(bits, other<16>(bits));
  }
  __device__ __forceinline__ void of_all_lanes_2() {
    bits = (uint32_t)__builtin_amdgcn_readfirstlane((int)row_max(bits));
    e = clamp_exp(bits);
  }
  // The group's scale: the walk's, or where that does not fit its own, which the block's word then names.
  __device__ __forceinline__ void choose(int unit, bool flag) {
    const bool shared = bits == 0 || (!flag && e <= unit && e >= unit - kBelow);
    word = shared ? 0 : e | (flag ? kFlag : 0);
    up = pow2_of(141 - (shared ? unit : e));
  }
  // Whether the walk's scale surely fits, from each lane's own largest: all below the scale, and one not far below.
  __device__ __forceinline__ bool fits(int unit) {
    const float most = pow2_of(min(unit + 1, kMaxExp) - 127), least = pow2_of(max(unit - kBelow, 1) - 127);
    return __ballot(!(m < most)) == 0 && __ballot(m >= least) != 0;
  }
  // Whether the rows are of unlike sizes: kSpread binades between the largest and the least.
  __device__ __forceinline__ bool unlike() {
    uint32_t least = 255;
    if constexpr (!kValues) {
      uint32_t r = __float_as_uint(m);  // a row's lanes are 8 apart
      r = max(r, other<32>(r));
      r = max(r, other<16>(r));
      r = max(r, ror<8>(r));
      if (r != 0) least = r >> 23;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t r = __float_as_uint(amax3(amax3(0.0f, x[j].x, x[j].y), x[j].z, x[j].w));
        r = max(r, other<16>(r));
        r = row_max(r);
        if (r != 0) least = min(least, r >> 23);
      }
      least = min(least, other<32>(least));
    }
    return e - __builtin_amdgcn_readfirstlane((int)row_min(least)) > kSpread;
  }
  // Where the group's halves go; fragments j of hi and lo are 4 (keys) or 2 (values) j on, the lo one behind.
  __device__ __forceinline__ static _Float16* place(_Float16* lds, int i, int group, int lane) {
    if constexpr (kValues) {
      return lds + 2 * kKHalves + i % 3 * kVHalves + (group / 2) * 8 * kFrag + lane * 8 + (group & 1) * 4;
    } else {
      const int c8 = lane >> 3;
      return lds + (i & 1) * kKHalves + (c8 >> 2) * 2 * kFrag + ((c8 & 1) * 32 + 8 * group + (lane & 7)) * 8 +
             (c8 >> 1 & 1) * 4;
    }
  }
  __device__ __forceinline__ void convert(int j, _Float16* at) {
    f32x4 v;
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = (kValues ? x[u][j] : x[j][u]) * up;
    uint32_t l0, l1;
    const uint32_t h0 = split2(v.x, v.y, l0), h1 = split2(v.z, v.w, l1);
    constexpr int kStep = kValues ? 2 : 4;
    *(u32x2*)(at + kStep * j * kFrag) = u32x2{h0, h1};
    *(u32x2*)(at + (kStep * j + 1) * kFrag) = u32x2{l0, l1};
  }
  __device__ __forceinline__ static void wipe(_Float16* at) {
    constexpr int kStep = kValues ? 2 : 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      *(u32x2*)(at + kStep * j * kFrag) = u32x2{};
      *(u32x2*)(at + (kStep * j + 1) * kFrag) = u32x2{};
    }
  }
};

// What the waves of a workgroup share besides the operands.
struct Shared {
  int meta[4][8];  // a block's words: of its key groups, then of its value groups
  int apart[4];    // whether one of them is not 0
  uint32_t slow[kMaxSplitRows / kBlock / 32];  // blocks left to the slow path
};
// The walk's scales, from the largest of each group of its first block.
__device__ __forceinline__ int walk_scale(const int* e) {
  const int most = max(max(e[0], e[1]), max(e[2], e[3]));
  return __builtin_amdgcn_readfirstlane(min(max(most, kMinExp) + kAbove, kMaxExp));
}

// The rows of one request as a walk meets them, page by page.
struct RowWalk {
  const float* pool;  // of the layer, the head and k
  const uint32_t* lookup;
  int64_t page_stride, slot_stride;
  int P, last_page, end;
  const float* base;  // the block's first row
  const float* next;  // the next page's, looked up ahead of its use
  int left;           // rows from the block's first to its page's end
  __device__ __forceinline__ const float* at(int row) const {
    return pool + (int64_t)min(ldc(lookup + row / P), (uint32_t)last_page) * page_stride +
           (int64_t)(row % P) * slot_stride;
  }
  __device__ __forceinline__ void start(int row) {
    base = at(row);
    left = P - row % P;
    next = at(min(row + left, end - 1));
  }
  __device__ __forceinline__ void step(int row) {  // to the block that starts at `row`
    left -= kBlock;
    base += kBlock * slot_stride;
    if (left == 0) {
      base = next;
      left = P;
      next = at(min(row + P, end - 1));
    }
  }
};

// A converting wave: 8 key rows and 8 value rows of each block, loaded two blocks ahead.
__device__ __forceinline__ void convert_walk(RowWalk rows, int64_t kv_stride, int begin, int shown, int group,
                                             _Float16* lds, Shared& sh) {
  const int end = rows.end, blocks = (end - begin + kBlock - 1) / kBlock, lane = lane_id();
  __builtin_amdgcn_s_setprio(3);
  const uint32_t row_bytes = (uint32_t)rows.slot_stride * 4u;
  Stage<false> k[2];
  Stage<true> v[2];
  const auto load = [&](int i, int at) {  // block i into buffer `at`
    const int last = end - 1 - (begin + i * kBlock);
    k[at].load(rows.base, kv_stride, row_bytes, group, last, lane);
    v[at].load(rows.base, kv_stride, row_bytes, group, last, lane);
  };
  const auto measure = [&](auto& x, int i) {
    const int key0 = begin + i * kBlock, last = end - 1 - key0;
    if (8 * group + 7 > last) x.clear_past(group, last, lane);
    x.largest();
    x.of_all_lanes_1();
    x.of_all_lanes_2();
    // rows hidden from some query: what they hold must not cost the others their bits
    return x.bits >= 0x7f800000u || (key0 + 8 * group + 7 >= shown && x.unlike());
  };
  const auto convert = [&](auto& x, int which, int i, bool flag, int unit, _Float16* at) {
    x.choose(unit, flag);
    sh.meta[i & 3][which + group] = x.word;
    if (x.word != 0) atomicOr(&sh.apart[i & 3], 1);
    if (flag) {  // the block's weights will be zero, and so must be what they multiply
      x.wipe(at);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x.convert(j, at);
    }
  };
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    k[j].at = (uint32_t)(8 * group + k[j].row_in_group(lane)) * row_bytes + k[j].column(lane);
    v[j].at = (uint32_t)(8 * group + v[j].row_in_group(lane)) * row_bytes + v[j].column(lane);
  }
  rows.start(begin);
  load(0, 0);
  if (blocks > 1) {
    rows.step(begin + kBlock);
    load(1, 1);
  }
  const bool kflag = measure(k[0], 0), vflag = measure(v[0], 0);
  sh.meta[0][group] = k[0].bits == 0 || kflag ? 0 : k[0].e;
  sh.meta[0][4 + group] = v[0].bits == 0 || vflag ? 0 : v[0].e;
  if (group == 0 && lane < 4) sh.apart[lane] = 0;
  lds_barrier();
  const int kunit = walk_scale(sh.meta[0]), vunit = walk_scale(sh.meta[0] + 4);
  lds_barrier();
  _Float16* const k_at = Stage<false>::place(lds, 0, group, lane);
  _Float16* const v_at = Stage<true>::place(lds, 0, group, lane);
  convert(k[0], 0, 0, kflag, kunit, k_at);
  convert(v[0], 4, 0, vflag, vunit, v_at);
  if (blocks > 2) {
    rows.step(begin + 2 * kBlock);
    load(2, 0);
  }
  lds_barrier();
  const int plain = (min(end, shown) - begin) / kBlock;  // blocks whose rows every query sees
  int v_buf = 1;
  const auto step = [&](int i, int at) {  // block i + 1, from buffer `at`, in the interval of block i
    if (i + 1 < blocks) {
      _Float16* kp = k_at + (at & 1) * kKHalves;  // at is 1 where i + 1 is odd
      _Float16* vp = v_at + v_buf * kVHalves;
      if (group == 0) sh.apart[(i + 3) & 3] = 0;  // of block i - 1, which all have read, for block i + 3
      k[at].largest();
      v[at].largest();
      if (i + 1 < plain && k[at].fits(kunit) && v[at].fits(vunit)) {
        k[at].up = pow2_of(141 - kunit);
        v[at].up = pow2_of(141 - vunit);
        sh.meta[(i + 1) & 3][group] = 0;
        sh.meta[(i + 1) & 3][4 + group] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) k[at].convert(j, kp);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[at].convert(j, vp);
      } else {
        const bool kf = measure(k[at], i + 1);
        convert(k[at], 0, i + 1, kf, kunit, kp);
        const bool vf = measure(v[at], i + 1);
        convert(v[at], 4, i + 1, vf, vunit, vp);
      }
      v_buf = v_buf == 2 ? 0 : v_buf + 1;
      if (i + 3 < blocks) {
        rows.step(begin + (i + 3) * kBlock);
        load(i + 3, at);
      }
    }
    lds_barrier();
  };
#pragma unroll 1
  for (int i = 0; i <= blocks; i += 2) {
    step(i, 1);
    if (i + 1 <= blocks) step(i + 1, 0);
  }
}

// An attending wave.  The two of a SIMD (w and w + 4) take turns: between two barriers the first runs the
// products of block i (the values of i - 1, the scores of i) and then its weights, the second the weights of
// i - 1 first, so that the matrix pipe has one wave's products while the other's exponentials issue.
__device__ __forceinline__ void attend_walk(Queries& w, int begin, int end, bool idle, bool second, const _Float16* lds,
                                            const _Float16* qlo, Shared& sh) {
  const int blocks = (end - begin + kBlock - 1) / kBlock;
  lds_barrier();
  const int kunit = walk_scale(sh.meta[0]), vunit = walk_scale(sh.meta[0] + 4);
  const float c = scale_of(w, kunit);
  w.ev = w.most = vunit;
  lds_barrier();
  lds_barrier();
  bool have = false, moved = false;
  Weights p;
  f32x16 s = {};
  int v_at = 0;  // the buffer of block i - 1's values
#pragma unroll 1
  for (int i = 0; i <= blocks; ++i) {
    const int now = lane_now(), key0 = begin + i * kBlock;
    const _Float16* vb = lds + 2 * kKHalves + v_at * kVHalves + now * 8;
    const _Float16* kb = lds + (i & 1) * kKHalves + now * 8;
    const _Float16* qb = qlo + now * 8;
    const auto vf = [&](int t, int u, int part) { return *(const f16x8*)(vb + (8 * t + 2 * u + part) * kFrag); };
    const auto kf = [&](int t, int part) { return *(const f16x8*)(kb + (2 * t + part) * kFrag); };
    const auto ql = [&](int t) { return *(const f16x8*)(qb + t * kFrag); };
    const bool had = have;
    const int other_scales = sh.apart[i & 3];
    have = i < blocks && !idle && __ballot(w.limit > key0) != 0;
    if (had) add_values(w, p, vf);
    if (have) s = scores(w, kf, ql);
    v_at = i == 0 ? 0 : v_at == 2 ? 0 : v_at + 1;
    if (second) lds_barrier();
    if (have) {
      int live = w.limit - key0;
      const bool apart = moved || __builtin_amdgcn_readfirstlane(other_scales) != 0;
      if (apart) {
        if (apart_scores(w, s, sh.meta[i & 3], kunit, vunit, live > 0)) {
          if (now == 0) atomicOr(&sh.slow[i / 32], 1u << (i % 32));
          live = 0;
        }
        moved = __ballot(w.ev != vunit) != 0;
      }
      hide(s, live, now);
      const float lift = (float)kLift - move_max(w, largest_of(s) * c);
      if (apart) apart_weights(w, s, sh.meta[i & 3], vunit, c, lift);
      w.l += weigh(s, c, lift, p);
    }
    if (!second) lds_barrier();
  }
}

__global__ void __launch_bounds__(64 * (kTileWaves + kStageWaves), 3)
    k_chunk_tiles(ChunkArgs a, float* out, const float* q, int64_t q_stride, float scale, float* part, float* weights,
                  int slots, int split_rows, int splits) {
  __shared__ __align__(16) _Float16 lds[kLdsHalves];
  __shared__ __align__(16) Shared sh;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  // neighbours in `item` walk the same rows: they go to one XCD, whose L2 then serves all but the first
  const int per = (int)(gridDim.x / 8), item = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
  if (item >= slots * a.heads * splits) return;
  const int slot = slots - 1 - item % slots, head = item / slots % a.heads, split = item / slots / a.heads;
  QueryTile qt;
  if (!query_tile(a, kTileLog2, slot, qt)) return;
  const int t_last = min(qt.t0 + 32 * kTileWaves, qt.end) - 1;
  const int all_rows = rows_of(a, qt, t_last);
  const int begin = split * split_rows, end = min(begin + split_rows, all_rows);
  if (begin >= end) return;
  const int shown = rows_of(a, qt, qt.t0);  // rows past these are hidden from some query
  RowWalk rows{a.pool + a.layer_off + (int64_t)head * kD, a.lookup + (int64_t)qt.n * a.lookup_cols, a.page_stride,
               a.slot_stride, a.P, a.pages - 1, end, nullptr, nullptr, 0};
  if (wave >= kTileWaves) {
    convert_walk(rows, a.kv_stride, begin, shown, wave - kTileWaves, lds, sh);
    return;
  }
  for (int i = (int)threadIdx.x; i < kMaxSplitRows / kBlock / 32; i += 64 * kTileWaves) sh.slow[i] = 0;
  const int my_t = min(qt.t0 + 32 * wave + (lane & 31), t_last);
  const bool idle = qt.t0 + 32 * wave > t_last;  // a wave without queries
  Queries w;
  _Float16* qlo = lds + 2 * kKHalves + 3 * kVHalves + wave * kQHalves;
  load_queries(w, qlo, q + (int64_t)my_t * q_stride + (int64_t)head * kD, scale, min(rows_of(a, qt, my_t), end));
  attend_walk(w, begin, end, idle, wave >= kTileWaves / 2, lds, qlo, sh);
  if (idle) return;
  float* stash = (float*)lds + wave * 32 * kWave + lane;
#pragma unroll 1
  for (int i = 0; i < (end - begin + kBlock - 1) / kBlock; ++i) {
    const int k0 = begin + i * kBlock;
    if ((sh.slow[i / 32] >> (i % 32) & 1) == 0 || __ballot(w.limit > k0) == 0) continue;
    slow_block(w, q + (int64_t)my_t * q_stride + (int64_t)head * kD, scale, rows.at(k0), a.kv_stride, a.slot_stride,
               min(w.limit - k0, kBlock), stash);
  }
  const bool live = qt.t0 + 32 * wave + (lane & 31) <= t_last;
  store_queries(w, a, my_t, live, head, split, all_rows <= split_rows, out, part, weights);
}

// k_chunk_few: 32 queries a workgroup, whose 4 waves take the rows' blocks in turn, each straight from memory into
// the operands' lanes (keys: lane (row l % 32, columns 8 i + 4 (l / 32)); values: lane (columns 4 (l % 32) on, rows
// 16 t + 8 (j / 4) + 4 (l / 32) + j % 4)), and join their sums in LDS.
constexpr int kFewWaves = 4;
constexpr int kFewLog2 = 5;             // queries of a workgroup
constexpr int kFewSplitRows = kFewWaves * 64 * kBlock;  // a wave notes its slow blocks in 64 bits

// 32 rows of keys or values on their way from memory to the operands of one wave.
struct FewStage {
  f32x4 x[16];
  __device__ __forceinline__ float largest() const {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = amax3(amax3(m, x[i].x, x[i].y), x[i].z, x[i].w);
    return m;
  }
};
// The largest of 64 lanes, as bits (every lane has it).
__device__ __forceinline__ uint32_t wave_largest(float m) {
  uint32_t bits = __float_as_uint(m);
  bits = max(bits, other<32>(bits));
  bits = max(bits, other<16>(bits));
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)row_max(bits));
}
// The scale of a block whose lanes' largest are m: the walk's if that fits (unit 0: there is none yet, and the
// block sets it).
__device__ __forceinline__ int few_scale(float m, int& unit, bool& finite) {
  if (unit != 0) {
    const float most = pow2_of(min(unit + 1, kMaxExp) - 127), least = pow2_of(max(unit - kBelow, 1) - 127);
    if (__ballot(!(m < most)) == 0 && __ballot(m >= least) != 0) return unit;
  }
  const uint32_t bits = wave_largest(m);
  finite = finite && bits < 0x7f800000u;
  const int e = clamp_exp(bits);
  if (bits == 0) return unit != 0 ? unit : kMinExp;
  if (unit == 0 && bits < 0x7f800000u) return unit = min(e + kAbove, kMaxExp);
  return e;
}

__global__ void __launch_bounds__(64 * kFewWaves, 2)
    k_chunk_few(ChunkArgs a, float* out, const float* q, int64_t q_stride, float scale, float* part, float* weights,
                int slots, int split_rows, int splits) {
  __shared__ __align__(16) float sums[kFewWaves][32 * kD];  // a wave's sums, before that its slow path's stash,
  _Float16* const qs = (_Float16*)sums;  // and first the queries' operands, [part][step][lane][8]
  __shared__ float peak[kFewWaves][32], total[kFewWaves][32];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), h = lane >> 5;
  const int per = (int)(gridDim.x / 8), item = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
  if (item >= slots * a.heads * splits) return;
  const int slot = slots - 1 - item % slots, head = item / slots % a.heads, split = item / slots / a.heads;
  QueryTile qt;
  if (!query_tile(a, kFewLog2, slot, qt)) return;
  const int t_last = min(qt.t0 + 32, qt.end) - 1;
  const int all_rows = rows_of(a, qt, t_last);
  const int begin = split * split_rows, end = min(begin + split_rows, all_rows);
  if (begin >= end) return;
  const int shown = rows_of(a, qt, qt.t0);
  const int my_t = min(qt.t0 + (lane & 31), t_last);
  const float* my_q = q + (int64_t)my_t * q_stride + (int64_t)head * kD;
  Queries w;
  load_queries(w, qs + kQHalves, my_q, scale, min(rows_of(a, qt, my_t), end));  // every wave the same values
#pragma unroll
  for (int t = 0; t < 8; ++t) *(f16x8*)(qs + t * kFrag + lane * 8) = w.hi[t];
  __syncthreads();
  const float* pool = a.pool + a.layer_off + (int64_t)head * kD;
  const uint32_t* lookup = a.lookup + (int64_t)qt.n * a.lookup_cols;
  const uint32_t row_bytes = (uint32_t)a.slot_stride * 4u;
  const auto row_base = [&](int row) {
    return pool + (int64_t)min(ldc(lookup + row / a.P), (uint32_t)(a.pages - 1)) * a.page_stride +
           (int64_t)(row % a.P) * a.slot_stride;
  };
  int kunit = 0, vunit = 0;
  uint64_t slow = 0;
  FewStage k, v;
  const auto load_k = [&](int key0, int lane) {
    const int h = lane >> 5;
    const char* from = (const char*)row_base(key0);
    const uint32_t at = (uint32_t)min(lane & 31, end - 1 - key0) * row_bytes + 16u * h;
#pragma unroll
    for (int i = 0; i < 16; ++i) k.x[i] = *(const UOCR_GLOBAL f32x4*)(from + at + 32 * i);
  };
  const auto load_v = [&](int key0, int lane) {
    const int h = lane >> 5;
    const char* from = (const char*)(row_base(key0) + a.kv_stride);
    const int last = end - 1 - key0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = min(16 * (i / 8) + 8 * (i / 4 % 2) + 4 * h + i % 4, last);
      v.x[i] = *(const UOCR_GLOBAL f32x4*)(from + ((uint32_t)row * row_bytes + 16u * (lane & 31)));
    }
  };
  const int first = begin + wave * kBlock;
  if (first < end) {
    load_k(first, lane);
    load_v(first, lane);
  }
#pragma unroll 1
  for (int key0 = first, i = 0; key0 < end; key0 += kFewWaves * kBlock, ++i) {
    const int lane = lane_now(), h = lane >> 5;
    const int last = end - 1 - key0, next = key0 + kFewWaves * kBlock;
    int live = w.limit - key0;
    bool finite = true;
    if (last < kBlock - 1) {  // rows past the last were its copies
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if ((lane & 31) > last) k.x[j] = f32x4{};
        if (16 * (j / 8) + 8 * (j / 4 % 2) + 4 * h + j % 4 > last) v.x[j] = f32x4{};
      }
    }
    const float km = k.largest();
    const int ek = few_scale(km, kunit, finite);
    f32x16 s = {};
    const float kup = pow2_of(141 - ek);
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      u32x4 hi, lo;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const f32x4 y = k.x[2 * t + j] * kup;
        uint32_t l0, l1;
        hi[2 * j] = split2(y.x, y.y, l0);
        hi[2 * j + 1] = split2(y.z, y.w, l1);
        lo[2 * j] = l0;
        lo[2 * j + 1] = l1;
      }
      const f16x8 qh = *(const f16x8*)(qs + t * kFrag + lane * 8);
      s = mfma(halves(hi), *(const f16x8*)(qs + kQHalves + t * kFrag + lane * 8), s);
      s = mfma(halves(lo), qh, s);
      s = mfma(halves(hi), qh, s);
    }
    const float vm = v.largest();
    const int ev = few_scale(vm, vunit, finite);
    if (key0 + kBlock > shown) {
      // rows hidden from some query: what they hold must not cost the others their bits
      const auto apart = [](uint32_t least, int e) {
        least = min(least, other<32>(least));
        least = min(least, other<16>(least));
        return e - __builtin_amdgcn_readfirstlane((int)row_min(least)) > kSpread;
      };
      uint32_t r = max(__float_as_uint(km), other<32>(__float_as_uint(km)));
      bool unlike = apart(r != 0 ? r >> 23 : 255, min(ek, clamp_exp(wave_largest(km))));
      uint32_t least = 255;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        r = __float_as_uint(amax3(amax3(0.0f, v.x[j].x, v.x[j].y), v.x[j].z, v.x[j].w));
        r = max(r, other<16>(r));
        r = row_max(r);
        if (r != 0) least = min(least, r >> 23);
      }
      unlike = unlike || apart(least, min(ev, clamp_exp(wave_largest(vm))));
      finite = finite && !unlike;
    }
    if (!finite) {  // left to the slow path
      slow |= 1ull << i;
      live = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) v.x[j] = f32x4{};
    }
    if (next < end) load_k(next, lane);
    const float c = scale_of(w, ek);
    hide(s, live, lane);
    const float lift = (float)kLift - move_max(w, largest_of(s) * c);
    w.most = max(w.most, ev);
    if (__ballot(w.ev != ev) != 0) {
      // every lane to the block's unit, which a sum of larger values may leave no room for
      const int unit = max(ev, w.most - kRoom);
      const float f = __builtin_ldexpf(1.0f, w.ev - unit);
#pragma unroll
      for (int u = 0; u < 4; ++u) w.o[u] *= f;
      w.ev = unit;
    }
    Weights p;
    w.l += weigh(s, c, lift, p);
    const float vup = pow2_of(141 - max(ev, w.ev));
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        u32x4 hi, lo;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t rest;
          hi[j] = split2(v.x[8 * t + 2 * j][u] * vup, v.x[8 * t + 2 * j + 1][u] * vup, rest);
          lo[j] = rest;
        }
        w.o[u] = mfma(halves(hi), p.lo[t], w.o[u]);
        w.o[u] = mfma(halves(lo), p.hi[t], w.o[u]);
        w.o[u] = mfma(halves(hi), p.hi[t], w.o[u]);
      }
    if (next < end) load_v(next, lane);
  }
  __syncthreads();
  for (int i = 0; slow != 0; ++i, slow >>= 1) {
    const int key0 = first + i * kFewWaves * kBlock;
    if ((slow & 1) != 0)
      slow_block(w, my_q, scale, row_base(key0), a.kv_stride, a.slot_stride, min(w.limit - key0, kBlock),
                 sums[wave] + lane);
  }
  // the waves' sums at one maximum, in the values' own unit
  const float l = w.l + other32(w.l);
  if (h == 0) {
    peak[wave][lane] = w.m;
    total[wave][lane] = l;
  }
  __syncthreads();
  float m = peak[0][lane & 31];
#pragma unroll
  for (int j = 1; j < kFewWaves; ++j) m = fmaxf(m, peak[j][lane & 31]);
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < kFewWaves; ++j) {
    const float mj = peak[j][lane & 31], lj = total[j][lane & 31];
    sum += mj == -kInf ? lj : lj * __builtin_amdgcn_exp2f(mj - m);  // lj: 0, or NaN
  }
  const float f = (w.m == -kInf ? (l == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(w.m - m)) / sum;
  // column 4 r' + u of query l % 32, rows of 128 floats whose 16-byte pieces are rotated by the query
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int piece = 8 * (r / 4) + 4 * h + r % 4;
    f32x4 y;
#pragma unroll
    for (int u = 0; u < 4; ++u) y[u] = __builtin_ldexpf(w.o[u][r] * f, w.ev - 141);
    *(f32x4*)(sums[wave] + (lane & 31) * kD + 4 * ((piece + lane) & 31)) = y;
  }
  __syncthreads();
  const bool whole = all_rows <= split_rows;
  const int64_t stride = (int64_t)a.tokens * a.heads;
#pragma unroll
  for (int j = 0; j < 32 * 32 / (64 * kFewWaves); ++j) {
    const int i = j * 64 * kFewWaves + (int)threadIdx.x, query = i / 32, piece = i % 32;
    if (qt.t0 + query > t_last) continue;
    const int at = query * kD + 4 * ((piece + query) & 31);
    f32x4 y = *(const f32x4*)(sums[0] + at);
#pragma unroll
    for (int k2 = 1; k2 < kFewWaves; ++k2) y += *(const f32x4*)(sums[k2] + at);
    const int64_t th = (int64_t)(qt.t0 + query) * a.heads + head;
    *(UOCR_GLOBAL f32x4*)((whole ? out + th * kD : part + (split * stride + th) * kD) + 4 * piece) = y;
  }
  if (!whole && wave == 0 && h == 0 && qt.t0 + lane <= t_last)
    weights[split * stride + ((int64_t)(qt.t0 + lane) * a.heads + head)] =
        sum == 0.0f ? -kInf : m + __builtin_amdgcn_logf(sum);
}

// Joins the splits of a token's rows: one wave per (token, head), two columns a lane.  The splits
// hold normalised sums, so a split weighs what its weights sum to.
__global__ void __launch_bounds__(256) k_chunk_join(ChunkArgs a, float* out, const float* __restrict__ part,
                                                    const float* __restrict__ weights, int rows_log2, int split_rows) {
  const int64_t th = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
  if (th >= (int64_t)a.tokens * a.heads) return;
  const int t = (int)(th / a.heads), lane = lane_id();
  int n, first;
  int64_t row;
  if (!request_of(a, t, n, first, row)) return;
  const int end = min(ldg(a.offsets + n + 1), a.tokens);
  const int t_last = min(first + ((((t - first) >> rows_log2) + 1) << rows_log2), end) - 1;  // of its tile
  const int splits = ((int)min(row + (t_last - t) + 1, (int64_t)a.attend_max) + split_rows - 1) / split_rows;
  if (splits == 1) return;  // written by its tile
  const int64_t stride = (int64_t)a.tokens * a.heads;
  float m = -kInf;
  for (int s = 0; s < splits; ++s) m = fmaxf(m, ldg(weights + s * stride + th));
  float l = 0.0f, o0 = 0.0f, o1 = 0.0f;
  for (int s = 0; s < splits; ++s) {
    const float ws = ldg(weights + s * stride + th);
    if (ws == -kInf) continue;
    const float f = __builtin_amdgcn_exp2f(ws - m);
    const float* p = part + (s * stride + th) * kD + 2 * lane;
    l += f;
    o0 = __builtin_fmaf(f, ldg(p), o0);
    o1 = __builtin_fmaf(f, ldg(p + 1), o1);
  }
  out[th * kD + 2 * lane] = o0 / l;
  out[th * kD + 2 * lane + 1] = o1 / l;
}

}  // namespace

// How a call's rows are cut: tiles of 256 or of 32 queries, and splits of their rows where the tiles alone do not fill
// the device.
namespace {
constexpr int kCus = 256;
struct Cut {
  bool few;
  int rows_log2, slots, split_rows, splits;
};
Cut cut_of(int64_t tokens, int64_t requests, int heads, int attend_max) {
  Cut c{};
  c.few = requests > 0 && tokens / requests < 128;
  c.rows_log2 = c.few ? kFewLog2 : kTileLog2;
  c.slots = (int)((tokens >> c.rows_log2) + requests);
  const int64_t full = std::max<int64_t>(1, (tokens + (1 << c.rows_log2) - 1) >> c.rows_log2) * heads;
  const int most = c.few ? kFewSplitRows : kMaxSplitRows, least = c.few ? 2 * kFewWaves * kBlock : 1024;
  const int64_t wanted = std::max<int64_t>(1, (c.few ? 2 : 1) * kCus / full);
  const int64_t rows = (attend_max + wanted - 1) / wanted;
  c.split_rows = (int)std::min<int64_t>(most, std::max<int64_t>(least, (rows + 127) / 128 * 128));
  c.splits = (int)(((int64_t)attend_max + c.split_rows - 1) / c.split_rows);
  return c;
}
}  // namespace

size_t chunk_workspace_bytes(int64_t tokens, int64_t requests, int heads, int attend_max) {
  const Cut c = cut_of(tokens, requests, heads, attend_max);
  return c.splits > 1 ? (size_t)c.splits * tokens * heads * (kD + 4) * sizeof(float) : 0;
}

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
  const float* q = rotated ? p.out : p.q;
  const int64_t q_stride = rotated ? (int64_t)p.heads * kD : p.in_stride;
  const Cut c = cut_of(p.tokens, p.requests, p.heads, p.attend_max);
  float* part = (float*)p.workspace;
  float* weights = part + (int64_t)c.splits * p.tokens * p.heads * kD;
  const int64_t items = (int64_t)c.slots * p.heads * c.splits;
  const dim3 grid((unsigned)((items + 7) / 8 * 8));
  if (c.few)
    UOCR_LAUNCH("chunk_few", k_chunk_few, grid, dim3(64 * kFewWaves), 0, s, a, p.out, q, q_stride, p.scale, part, weights,
                c.slots, c.split_rows, c.splits);
  else
    UOCR_LAUNCH("chunk_tiles", k_chunk_tiles, grid, dim3(64 * (kTileWaves + kStageWaves)), 0, s, a, p.out, q, q_stride,
                p.scale, part, weights, c.slots, c.split_rows, c.splits);
  if (c.splits > 1)
    UOCR_LAUNCH("chunk_join", k_chunk_join, dim3((unsigned)((p.tokens * p.heads + 3) / 4)), dim3(256), 0, s, a, p.out,
                part, weights, c.rows_log2, c.split_rows);
  return hipGetLastError();
}

}  // namespace uocr
