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
// k_chunk_store writes the new rows into the pool, and rotated queries into out, before k_chunk_tiles, which reads
// every row from there.  (Queries rotated by the tiles as they are read: 10 us more for 8 prompts of up to 512.)  In
// k_chunk_few a new row is read from the inputs (rotated by whoever reads it, where it comes unrotated) and stored by
// the workgroup whose queries its token is among; nothing else in the launch reads that pool row.
//
// k_chunk_tiles (256 queries a workgroup) and k_chunk_few (32) run the two products on the fp16 matrix instruction,
// each operand as a pair of halves, and keep a running maximum and sum of every query (below).  A piece that the pairs
// cannot hold (values that are not finite, keys whose scores would lose bits beside larger ones, sums that came out too
// small for what the pairs leave out) is done again in fp32 by the same workgroup.
#include <algorithm>

#include "chunk_device.h"
#include "uocr_kernels.h"

namespace uocr {

namespace {

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

__device__ __forceinline__ float* row_ptr(const ChunkArgs& a, int n, int h, int r, int kv) {
  const uint32_t page = min(ldg(a.lookup + (int64_t)n * a.lookup_cols + r / a.P), (uint32_t)(a.pages - 1));
  return a.pool + (int64_t)page * a.page_stride + kv * a.kv_stride + a.layer_off +
         (int64_t)(r % a.P) * a.slot_stride + (int64_t)h * kD;
}

// The tensors whose rows are in_stride floats apart.
struct Inputs {
  const float* q;
  const float* k_new;
  const float* v_new;
};

// Lane d < 64 of a wave: the pair (d, d + 64) of token t's k and v of one head into the pool.
__device__ __forceinline__ void store_pair(const ChunkArgs& a, const Rope& rope, const Inputs& in, const Chunk& c, int t,
                                           int h, int d) {
  const int64_t src = (int64_t)t * a.in_stride + (int64_t)h * kD, row = (int64_t)c.cached + (t - c.first);
  if (row >= a.max_rows) return;  // past what the lookup row addresses: not stored
  const float* k = in.k_new + src;
  float* kp = row_ptr(a, c.n, h, (int)row, 0) + d;
  if (rope.positions != nullptr) {
    const int64_t at = (int64_t)min(max(ldg(rope.positions + t), 0), rope.table_rows - 1) * kD;
    kp[0] = rotated(k, rope.cos_t + at, rope.sin_t + at, d);
    kp[64] = rotated(k, rope.cos_t + at, rope.sin_t + at, d + 64);
  } else {
    kp[0] = ldg(k + d);
    kp[64] = ldg(k + d + 64);
  }
  kp[a.kv_stride] = ldg(in.v_new + src + d);
  kp[a.kv_stride + 64] = ldg(in.v_new + src + d + 64);
}

// One wave per (token, head).  Bound by memory: 8 prompts of up to 512 tokens, 100 MB read and written, 18 us.
__global__ void __launch_bounds__(256) k_chunk_store(ChunkArgs a, Rope rope, Inputs in, float* out) {
  const int64_t th = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  if (th >= (int64_t)a.tokens * a.heads) return;
  const int t = (int)(th / a.heads);
  Chunk c;
  if (!chunk_of(a, t, c)) return;
  const int h = (int)(th % a.heads), d = lane_id();
  if (rope.positions != nullptr) {
    const int64_t at = (int64_t)min(max(ldg(rope.positions + t), 0), rope.table_rows - 1) * kD;
    const float* q = in.q + (int64_t)t * a.in_stride + (int64_t)h * kD;
    out[th * kD + d] = rotated(q, rope.cos_t + at, rope.sin_t + at, d);
    out[th * kD + d + 64] = rotated(q, rope.cos_t + at, rope.sin_t + at, d + 64);
  }
  store_pair(a, rope, in, c, t, h, d);
}

// ------------------------------------------------------------------ fp32 products on the fp16 matrix instruction
//
// An operand x (times a power of two that brings its group's largest to [2^14, 2^15)) is held
// as hi = fp16(x), lo = fp16(x - hi): 22 bits, or 2^-39 of the group's largest where
// that is more.  hi hi + hi lo + lo hi leaves out lo lo, 2^-22 of the product at most.
// Where 2^-39 of the largest could count, kSharp (scores) and faint (sums) find it out.

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kInf = __builtin_huge_valf();
constexpr int kBlock = 32;    // rows (keys) a wave takes at a time: the rows of one matrix instruction
constexpr int kMinExp = 15;   // exponents of a group's scale: 2^(141 - e) is a normal fp32
constexpr int kMaxExp = 254;
// Weights are held as 2^kLift p, high above fp16's smallest, and a maximum may lag by 2^kSlack before the sums are rescaled:
// 2^15.9 is below fp16's largest.  (A lift of 15 and a slack of 0.9 rescale more often: eight chunks of 256 over 1000 rows
// 73.2 us for 72.1.)
constexpr int kLift = 13;
constexpr float kSlack = 2.9f;
constexpr int kNear = 6;      // binades by which a lane's unit may be above the values now added
constexpr int kGone = 64;     // binades below a lane's unit from which on values leave nothing in it
constexpr int kRoom = 60;     // binades that a sum may stand above the values now added to it
constexpr float kSharp = 0x1p-15f;  // the most of a score, in binades, that one step of the operands' products may be
constexpr int kAbove = 2;     // binades of the walk's scales above its first block's largest,
constexpr int kBelow = 10;    // and below the scale that a group's largest may be
constexpr int kFlag = 1 << 16;  // a group that the fp16 pairs cannot hold
constexpr int kFrag = 64 * 8;   // halves of an operand: 8 of each lane
constexpr int kMaxSplitRows = 1 << 16;  // rows of one workgroup

// Six instructions with the scaling before it.  (Four, where each half is one product rounded to fp16 in place: 474 us
// for 450 in k_chunk_tiles at 2048 tokens over 14001 rows, and nothing gained in k_chunk_few.)
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
// The largest of 64 lanes, as bits (every lane has it).
__device__ __forceinline__ uint32_t wave_largest(float m) {
  uint32_t bits = __float_as_uint(m);
  bits = max(bits, other<32>(bits));
  bits = max(bits, other<16>(bits));
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)row_max(bits));
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
  int most;    // the largest unit of the sum so far, less the binades by which its weights shrank since
  f32x16 o[4];
};

__device__ __forceinline__ void start_queries(Queries& w, float scale, int limit) {
  w.unit = __builtin_fabsf(scale) * 1.44269504f;
  w.limit = limit;
  w.m = -kInf;
  w.l = 0.0f;
  w.ev = w.most = kMinExp;  // (a sum of zeros)
#pragma unroll
  for (int u = 0; u < 4; ++u) w.o[u] = f32x16{};
}
// The exponent of a query's scale (one that is not finite has no scores, whatever it is scaled by).
__device__ __forceinline__ int query_exp(uint32_t bits) { return bits < 0x7f800000u ? clamp_exp(bits) : kMinExp; }
__device__ __forceinline__ void load_queries(Queries& w, _Float16* qlo, const float* row, float scale, int limit) {
  const int h = lane_id() >> 5;
  f32x4 x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = *(const UOCR_GLOBAL f32x4*)(row + 8 * i + 4 * h);
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = amax3(amax3(m, x[i].x, x[i].y), x[i].z, x[i].w);
  const uint32_t bits = max(__float_as_uint(m), other<32>(__float_as_uint(m)));
  w.exp = query_exp(bits);
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
  start_queries(w, scale, limit);
}

__device__ __forceinline__ void scale_sums(Queries& w, int by) {  // by 2^by, past fp32's exponents in two steps
  const int most = min(max(by, -126), 126);
#pragma unroll
  for (int u = 0; u < 4; ++u) w.o[u] *= pow2_of(most);
  if (__ballot(by != most) == 0) return;
#pragma unroll
  for (int u = 0; u < 4; ++u) w.o[u] *= __builtin_ldexpf(1.0f, by - most);
}
// Brings a lane's unit to where values of exponent eb can be added: at or above it, and not more
// than kNear below, as far as the sum of larger ones (2^kRoom at most) stays in range.
__device__ __forceinline__ void set_unit(Queries& w, int eb, bool attends) {
  const int need = max(eb, w.most - kRoom);
  const bool move = attends && (need > w.ev || need < w.ev - kNear);
  if (__ballot(move) != 0) {
    scale_sums(w, move ? w.ev - need : 0);
    w.ev = move ? need : w.ev;
  }
  w.most = attends ? max(w.most, w.ev) : w.most;
}

// Moves a lane's running maximum to mx, where that is more by kSlack; returns what to take off its scores.
__device__ __forceinline__ float move_max(Queries& w, float mx) {
  mx = fmaxf(mx, other32(mx));
  const bool up = mx > w.m + kSlack;
  if (__ballot(up) != 0) {
    const float alpha = up ? __builtin_amdgcn_exp2f(w.m - mx) : 1.0f;
    w.most = up ? max(w.most - (int)fminf(mx - w.m, 256.0f), kMinExp) : w.most;
    w.m = up ? mx : w.m;
    w.l *= alpha;
#pragma unroll
    for (int u = 0; u < 4; ++u) w.o[u] *= alpha;
  }
  return w.m == -kInf ? 0.0f : w.m;
}

// Whether a lane's sum is too small for what the pairs leave out of it; rows: how many, top: the largest of their values'
// exponents (0: none but zeros).  In the sum's units a row is off by 2^-25, of its weight, times a value of 2^15 at most,
// and by its weight times 2^-25, of its value (beside 2^-22 of the product): rows 2^-10 + l 2^-25 in all, of which the sum
// has to be 2^17 times as much.  Values of like sizes make it so by far; less it is where a row of large values has no
// weight, or a row of small ones nearly all of it.
__device__ __forceinline__ bool faint(const Queries& w, int rows, int top) {
  float m = 0.0f;
#pragma unroll
  for (int u = 0; u < 4; ++u)
#pragma unroll
    for (int r = 0; r < 16; r += 2) m = amax3(m, w.o[u][r], w.o[u][r + 1]);
  m = amax3(m, m, other32(m));
  const float l = w.l + other32(w.l), off = __builtin_ldexpf((float)rows, 7 + min(top - w.most, 0)) + 0x1p-8f * l;
  return top != 0 && l > 0.0f && m < __builtin_ldexpf(off, w.most - w.ev);
}

// What the fp32 form reads: a request's rows from the pool, and from old_rows on from the inputs.
struct SlowRows {
  const float* pool;  // of the layer, the head and k
  const uint32_t* lookup;
  const float* k_new;  // as if row 0 were new
  const float* v_new;
  int64_t page_stride, kv_stride, slot_stride, in_stride;
  int P, last_page, old_rows, end;
  Rope rope;
  int64_t token;  // row 0's
};
__device__ __forceinline__ void rotate_at(const Rope& rope, int64_t token, int col, f32x4& lo, f32x4& hi) {
  const int64_t at = (int64_t)min(max(ldg(rope.positions + token), 0), rope.table_rows - 1) * kD + col;
  const float *c = rope.cos_t + at, *s = rope.sin_t + at;
  rotate4(lo, hi, *(const UOCR_GLOBAL f32x4*)c, *(const UOCR_GLOBAL f32x4*)(c + 64), *(const UOCR_GLOBAL f32x4*)s,
          *(const UOCR_GLOBAL f32x4*)(s + 64));
}
// The binades of a weight above 1 (NaN: as the largest).
__device__ __forceinline__ int weight_exp(float p) {
  return p == 0.0f ? -kMaxExp : min((int)(__float_as_uint(p) >> 23) - 127, 16) - kLift;
}
// A block of rows in fp32, for inputs that the pairs cannot hold: the matrix instruction of that type, whose results have
// the same layout (step r of the second product is keys 8 (r / 4) + r % 4 of lanes 0 to 31 and 4 on of the others, whose
// weights the lanes hold).  Each value row is brought to its own largest and its weights take up the binades, and a
// lane's unit follows what the weighted rows come to: a row without weight costs the others nothing, whatever its size.
// Values that are not finite reach the queries that attend them only.  q: the lane's query, of token q_token.
// stash: 32 floats a lane.
__device__ __forceinline__ void slow_block(Queries& w, const SlowRows& rows, const float* q, int64_t q_token, int key0,
                                           float scale, float* stash) {
  const int lane = lane_id(), h = lane >> 5, last = min(rows.end - 1 - key0, kBlock - 1), live = w.limit - key0;
  const int old_rows = rows.old_rows - key0;  // of the block
  const uint32_t page = min(ldg(rows.lookup + key0 / rows.P), (uint32_t)rows.last_page);
  const float* base = rows.pool + (int64_t)page * rows.page_stride + (int64_t)(key0 % rows.P) * rows.slot_stride;
  f32x16 s = {};
  {
    const int key = min(lane & 31, last);
    const float* k = (key < old_rows ? base + key * rows.slot_stride : rows.k_new + (int64_t)(key0 + key) * rows.in_stride) +
                     4 * h;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      f32x4 kl = *(const UOCR_GLOBAL f32x4*)(k + 8 * i), kh = *(const UOCR_GLOBAL f32x4*)(k + 8 * i + 64);
      f32x4 ql = *(const UOCR_GLOBAL f32x4*)(q + 8 * i + 4 * h), qh = *(const UOCR_GLOBAL f32x4*)(q + 8 * i + 4 * h + 64);
      if (rows.rope.positions != nullptr) {
        rotate_at(rows.rope, q_token, 8 * i + 4 * h, ql, qh);
        if (key >= old_rows) rotate_at(rows.rope, rows.token + key0 + key, 8 * i + 4 * h, kl, kh);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s = __builtin_amdgcn_mfma_f32_32x32x2f32(kl[e], ql[e], s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_f32_32x32x2f32(kh[e], qh[e], s, 0, 0, 0);
      }
    }
  }
  float mx = -kInf;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    s[r] = 8 * (r / 4) + 4 * h + r % 4 < live ? s[r] * scale * 1.44269504f : -kInf;
    mx = fmaxf(mx, s[r]);
  }
  const float mu = move_max(w, mx);
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const float p = __builtin_amdgcn_exp2f(s[r] - mu + (float)kLift);
    w.l += p;
    stash[r * kWave] = p;
  }
  const auto key_of = [](int r, int h) { return 8 * (r / 4) + 4 * h + r % 4; };
  const auto finite = [](float x) { return (__float_as_uint(x) & 0x7fffffffu) < 0x7f800000u; };
  const auto only_finite = [&](f32x4 x) {
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = finite(x[u]) ? x[u] : 0.0f;
    return x;
  };
  const auto v_row = [&](int key) {
    return key < old_rows ? base + rows.kv_stride + key * rows.slot_stride
                          : rows.v_new + (int64_t)(key0 + key) * rows.in_stride;
  };
  const auto value = [&](int r) {  // columns 4 (l % 32) on of the lane's row
    return *(const UOCR_GLOBAL f32x4*)(v_row(min(key_of(r, h), last)) + 4 * (lane & 31));
  };
  int top = 0;  // of the weighted rows, as an exponent of values
#pragma unroll 1
  for (int r = 0; r < 16; ++r) {
    const f32x4 x = only_finite(value(r));
    uint32_t bits = __float_as_uint(amax3(amax3(0.0f, x.x, x.y), x.z, x.w));
    bits = row_max(max(bits, other<16>(bits)));
    const int e = clamp_exp(bits);
    stash[(16 + r) * kWave] = __int_as_float(e);
    if (bits != 0) top = max(top, e + weight_exp(stash[r * kWave]));
  }
  top = max(top, (int)other<32>((uint32_t)top));
  set_unit(w, max(top, kMinExp), live > 0);
  uint32_t odd = 0;  // rows with values that are not finite
#pragma unroll 1
  for (int r = 0; r < 16; ++r) {
    const int e = __float_as_int(stash[(16 + r) * kWave]);
    const f32x4 v = value(r), x = only_finite(v) * pow2_of(141 - e);
    const float p = __builtin_ldexpf(stash[r * kWave], e - w.ev);
#pragma unroll
    for (int u = 0; u < 4; ++u) w.o[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[u], p, w.o[u], 0, 0, 0);
    const uint64_t bad = __ballot(!finite(v.x) || !finite(v.y) || !finite(v.z) || !finite(v.w));
    if ((uint32_t)bad != 0) odd |= 1u << key_of(r, 0);
    if (bad >> 32 != 0) odd |= 1u << key_of(r, 1);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  for (; odd != 0; odd &= odd - 1) {
    const int key = __builtin_ctz(odd);
    if (key >= live) continue;
    // the weight is held by the lane of the key's half
    const float p = stash[(4 * (key / 8) + key % 4) * kWave + (lane & 31) + 8 * (key & 4) - lane];
    const float* v = v_row(key) + 16 * h;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const f32x4 x = *(const UOCR_GLOBAL f32x4*)(v + 32 * (i / 4) + 4 * (i % 4));
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (!finite(x[u])) w.o[u][i] = __builtin_fmaf(p, x[u], w.o[u][i]);
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the stash is read before the next block's is written
}
// The kernel's arguments read once more, so that a part that hardly ever runs keeps none of them in registers before it.
template <typename T>
__device__ __forceinline__ T arguments_again() {
  uint64_t at = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  static_assert(sizeof(T) % 4 == 0, "whole words");
  uint32_t words[sizeof(T) / 4];
#pragma unroll
  for (size_t i = 0; i < sizeof(T) / 4; ++i) words[i] = ((const UOCR_CONST uint32_t*)at)[i];
  T args;
  __builtin_memcpy(&args, words, sizeof(T));
  return args;
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
// What one of the products' sum counts as in a score's binades, where the keys' scale is ek.  (> 0: hidden rows stay at
// -inf.)  A small element of a key or a query is off by 2^-25 of such a unit, and meets 2^15 at most: with 128 of each, a
// score is off by a quarter of it.  Up to kSharp that is 2^-17, whatever the rows' sizes; beyond, scores of 2^15 and more
// are at hand, and the block is not for the pairs.
__device__ __forceinline__ float scale_of(const Queries& w, int ek) {
  return __builtin_amdgcn_fmed3f(__builtin_ldexpf(w.unit, w.exp + (ek - 282)), 1e-35f, 3.4e38f);
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
// weights: the scores at the walk's scale, and the units of the sums.  Returns whether the block is not for
// the pairs.
__device__ __forceinline__ bool apart_scores(Queries& w, f32x16& s, const int* meta, int kunit, int vunit, float c,
                                             bool attends) {
  int any = 0, most = 0, far = -kMaxExp;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int wk = meta[g], wv = meta[4 + g];
    const int ek = wk == 0 ? kunit : wk & (kFlag - 1), ev = wv == 0 ? vunit : wv & (kFlag - 1);
    any |= wk | wv;
    most = max(most, ev);
    far = max(far, ek - kunit);
#pragma unroll
    for (int r = 4 * g; r < 4 * g + 4; ++r) s[r] = __builtin_ldexpf(s[r], ek - kunit);
  }
  const bool blunt = attends && __builtin_ldexpf(c, far) > kSharp;
  const bool slow = __ballot(any >= kFlag || far > kRoom || blunt) != 0;
  set_unit(w, most, attends && !slow);
  return slow;
}
// Then the weights take up the binades from w.ev to their value group's scale: the scores are moved so that the
// weights come out so, and the sum of the weights has what they lack.
__device__ __forceinline__ void apart_weights(Queries& w, f32x16& s, const int* meta, int vunit, float c, float lift) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int wv = meta[4 + g], by = max(min((wv == 0 ? vunit : wv & (kFlag - 1)) - w.ev, 0), -kGone);
    const float lack = __builtin_ldexpf(1.0f, -by) - 1.0f, move = (float)by / c;
#pragma unroll
    for (int r = 4 * g; r < 4 * g + 4; ++r) {
      s[r] += move;
      w.l = __builtin_fmaf(lack, __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, lift)), w.l);
    }
  }
}

// ------------------------------------------------------------------ tiles of queries

// The pieces of a call: a tile of 2^rows_log2 queries of one request with one split of its rows and one head.  Of up to
// 64 requests they are dealt one after the other, the longest first (a lane per request counts its pieces); else by
// tile, where tile j of request n is slot floor(off[n] / rows) + n + j, which no other tile is, with slots and splits
// left out.  Workgroups go round the XCDs: neighbours walk the same rows, and stay on one XCD, whose L2 then serves all
// but the first.  Those without a piece are best dealt last: left between the others, 8 chunks of 256 over 1000 rows
// took 138 us for 78 (every other workgroup was empty, and the others met on half of the shader engines), and two of
// 1024 in splits of 256 took 84 us for 60 (some CUs had two pieces, others none).
struct QueryTile : Chunk {
  int t0;  // the tile's first token
};
// Rows that token t of the request attends.
__device__ __forceinline__ int rows_of(const ChunkArgs& a, const QueryTile& q, int t) {
  return (int)min((int64_t)q.cached + (t - q.first) + 1, (int64_t)a.attend_max);
}
struct Cuts {
  int rows_log2, slots, split_rows, splits;
  Divide by_split, by_slots, by_splits;
};
struct Piece : QueryTile {
  int head, split, t_last;  // t_last: the tile's last token
};
__device__ __forceinline__ bool find_piece(const ChunkArgs& a, const Cuts& c, Piece& q) {
  const int turn = (int)(blockIdx.x / 8), xcd = (int)(blockIdx.x % 8), rows = 1 << c.rows_log2;
  int j;
  if (a.requests <= 64) {
    const int i = min(lane_id(), a.requests - 1);
    const int off = ldg(a.offsets + i), next = min(ldg(a.offsets + i + 1), a.tokens);
    const int cached = (int)min(ldg(a.cache_lengths + i), (uint32_t)a.max_rows);
    const bool some = lane_id() < a.requests && off >= 0 && off < next;
    const int tiles = some ? ((next - off - 1) >> c.rows_log2) + 1 : 0;
    // splits of tile j: those of its last token's rows
    const auto cuts = [&](int cached, int length, int j) {
      const int64_t rows = (int64_t)cached + min((j + 1) << c.rows_log2, length);
      return c.by_split((int)min(rows, (int64_t)a.attend_max) - 1) + 1;
    };
    int pieces = tiles;
    if (c.splits > 1) {
      pieces = 0;
      for (int k = 0; __ballot(k < tiles) != 0; ++k)
        if (k < tiles) pieces += cuts(cached, next - off, k);
    }
    const int upto = wave_scan_i(pieces), total = __builtin_amdgcn_readlane(upto, 63);
    const int per = (total * a.heads + 7) / 8, item = xcd * per + turn;
    if (turn >= per || item >= total * a.heads) return false;
    q.head = item / total;
    int left = item - q.head * total;
    const int at = __popcll(__ballot(upto <= left));  // the request whose pieces reach past it
    left -= __builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(pieces, at);
    q.n = at;
    q.first = __builtin_amdgcn_readlane(off, at);
    q.end = __builtin_amdgcn_readlane(next, at);
    q.cached = (uint32_t)__builtin_amdgcn_readlane(cached, at);
    j = __builtin_amdgcn_readlane(tiles, at) - 1;
    if (c.splits > 1) {
      for (; j > 0; --j) {
        const int here = cuts((int)q.cached, q.end - q.first, j);
        if (left < here) break;
        left -= here;
      }
      q.split = left;
    } else {
      q.split = 0;
      j -= left;
    }
  } else {
    const int item = xcd * (int)(gridDim.x / 8) + turn;
    if (item >= c.slots * a.heads * c.splits) return false;
    const int by_tile = c.by_slots(item), slot = c.slots - 1 - (item - by_tile * c.slots);
    q.head = c.by_splits(by_tile);
    q.split = by_tile - q.head * c.splits;
    (Chunk&)q = find_chunk(a, c.rows_log2, true, slot);
    j = slot - ((q.first >> c.rows_log2) + q.n);
    if (q.first < 0 || j < 0 || (int64_t)j << c.rows_log2 >= q.end - q.first) return false;
  }
  q.t0 = q.first + (j << c.rows_log2);
  q.t_last = min(q.t0 + rows, q.end) - 1;
  return true;
}

// The arguments of the attending kernels.
struct Attend {
  ChunkArgs a;
  Rope rope;
  Inputs in;  // where no row is new to the kernel, q alone
  float scale;
  float* out;
  float* part;
  float* weights;
  Cuts cuts;
};
// What one piece of them is: rows [begin, stop) of its request's, of all_rows that the tile attends.
struct Work : Piece {
  int begin, stop, all_rows;
};
__device__ __forceinline__ bool find_work(const Attend& p, Work& w) {
  if (!find_piece(p.a, p.cuts, w)) return false;
  w.all_rows = rows_of(p.a, w, w.t_last);
  w.begin = w.split * p.cuts.split_rows;
  w.stop = min(w.begin + p.cuts.split_rows, w.all_rows);
  return true;
}
// A wave's queries, from the tile's token t0 on, over the blocks from row `first` on, `step` rows apart, in fp32.  Bound by
// that matrix instruction, an eighth of the pairs' rate with their three products, and by the loads before it; with the
// pairs' walk before, 2048 tokens over 14001 rows take 3894 us for 455, 8 requests of 7 over 1150 78 for 23.5.
__device__ __forceinline__ void attend_in_fp32(Queries& w, const Attend& p, const Work& work, int t0, int first, int step,
                                               bool news, float* stash) {
  const int my_t = min(t0 + (lane_id() & 31), work.t_last);
  const int64_t head = (int64_t)work.head * kD, token = work.first - work.cached;  // row 0's
  const SlowRows rows{p.a.pool + p.a.layer_off + head, p.a.lookup + (int64_t)work.n * p.a.lookup_cols,
                      news ? p.in.k_new + token * p.a.in_stride + head : nullptr,
                      news ? p.in.v_new + token * p.a.in_stride + head : nullptr, p.a.page_stride, p.a.kv_stride,
                      p.a.slot_stride, p.a.in_stride, p.a.P, p.a.pages - 1, news ? work.cached : work.stop, work.stop,
                      p.rope, token};
  start_queries(w, p.scale, min(rows_of(p.a, work, my_t), work.stop));
#pragma unroll 1
  for (int key0 = first; key0 >= work.begin && key0 < work.stop; key0 += step)
    if (__ballot(w.limit > key0) != 0)
      slow_block(w, rows, p.in.q + (int64_t)my_t * p.a.in_stride + head, my_t, key0, p.scale, stash);
}

// The logarithm of a sum of weights, of which the lift would leave fewer bits.
__device__ __forceinline__ float log2_weight(float l) { return __builtin_amdgcn_logf(l * pow2_of(-kLift)); }
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
    weights[(int64_t)split * a.tokens * a.heads + th] = l == 0.0f ? -kInf : w.m + log2_weight(l);
}

// k_chunk_tiles: 8 waves of 32 queries each walk the rows together, a block of 32 at a time.  4 more bring the
// rows, two blocks ahead, turn them into fp16 pairs and write them to LDS as the matrix operands they will
// be, an operand's 64 lanes side by side.
//
// Bound by the matrix instruction and the power it draws: 2048 tokens over 14001 rows, 10 heads, are 158 GFLOP, three
// times that as fp16 products, in 433 to 469 us (cards differ): 1.01 to 1.09 PFLOP/s, where a large fp16 matrix product
// reaches 1.13 (and an fp32 one 0.153, which would be 1031 us).  256 queries, since each row is converted once for all of
// them; the operands, 144 KB, take a CU's LDS.  Waves that convert for themselves, without the four: 538 us; blocks of 64
// rows: 716 (spills); conversions between the matrix instructions: 588; both waves of a SIMD in step: 527; the new rows
// stored and rotated here and not by k_chunk_store: 551, and 8 prompts 83 us for 68.
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

  __device__ __forceinline__ static int row_in_group(int lane) { return kValues ? 4 * (lane >> 5) : lane & 7; }
  __device__ __forceinline__ static uint32_t column(int lane) { return 16u * (kValues ? lane & 31 : lane >> 3); }
  // 32 rows are below 2^32 bytes: 32 bits of offset a lane, from a scalar base.  Rows past the last are its
  // copies, zeroed before they are converted.
  __device__ __forceinline__ void load(const float* from, uint32_t row_bytes, int group, int last, int lane) {
    const int row = 8 * group + row_in_group(lane);
    if (last >= kBlock - 1) {
      const uint32_t at = (uint32_t)row * row_bytes + column(lane);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[j] = kValues ? *(const UOCR_GLOBAL f32x4*)((const char*)from + (at + j * row_bytes))
                       : *(const UOCR_GLOBAL f32x4*)((const char*)from + at + 128 * j);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[j] = *(const UOCR_GLOBAL f32x4*)((const char*)from + ((uint32_t)min(row + (kValues ? j : 0), last) * row_bytes +
                                                                column(lane) + (kValues ? 0u : 128u * j)));
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
};

// What the waves of a workgroup share besides the operands.
struct Shared {
  int meta[4][8];  // a block's words: of its key groups, then of its value groups
  int apart[4];    // whether one of them is not 0
  int top;         // the largest of the values' exponents (0: none but zeros)
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
__device__ __forceinline__ void convert_walk(RowWalk rows, int64_t kv_stride, int begin, int group,
                                             _Float16* lds, Shared& sh) {
  const int end = rows.end, blocks = (end - begin + kBlock - 1) / kBlock, lane = lane_id();
  __builtin_amdgcn_s_setprio(3);
  const uint32_t row_bytes = (uint32_t)rows.slot_stride * 4u;
  Stage<false> k[2];
  Stage<true> v[2];
  const auto load = [&](int i, int at) {  // block i into buffer `at`
    const int last = end - 1 - (begin + i * kBlock);
    k[at].load(rows.base, row_bytes, group, last, lane);
    v[at].load(rows.base + kv_stride, row_bytes, group, last, lane);
  };
  const auto measure = [&](auto& x, int i) {
    const int last = end - 1 - (begin + i * kBlock);
    if (8 * group + 7 > last) x.clear_past(group, last, lane);
    x.largest();
    x.of_all_lanes_1();
    x.of_all_lanes_2();
    return x.bits >= 0x7f800000u;
  };
  const auto convert = [&](auto& x, int which, int i, bool flag, int unit, _Float16* at) {
    x.choose(unit, flag);
    sh.meta[i & 3][which + group] = x.word;
    if (x.word != 0) atomicOr(&sh.apart[i & 3], 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) x.convert(j, at);
  };
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
  if (group == 0 && lane == 0) sh.top = 0;
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
  float top = v[0].m;  // of the lane's values
  const auto give_top = [&] {
    const uint32_t bits = wave_largest(top);
    if (lane == 0 && bits != 0) atomicMax(&sh.top, clamp_exp(bits));
  };
  if (blocks == 1) give_top();
  lds_barrier();
  const int full = (end - begin) / kBlock;
  int v_buf = 1;
  const auto step = [&](int i, int at) {  // block i + 1, from buffer `at`, in the interval of block i
    if (i + 1 < blocks) {
      _Float16* kp = k_at + (at & 1) * kKHalves;  // at is 1 where i + 1 is odd
      _Float16* vp = v_at + v_buf * kVHalves;
      if (group == 0) sh.apart[(i + 3) & 3] = 0;  // of block i - 1, which all have read, for block i + 3
      k[at].largest();
      v[at].largest();
      top = fmaxf(top, v[at].m);
      if (i + 2 == blocks) give_top();
      if (i + 1 < full && k[at].fits(kunit) && v[at].fits(vunit)) {
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

// An attending wave; returns whether the pairs held all that it met.  The two of a SIMD (w and w + 4) take turns: between
// two barriers the first runs the products of block i (the values of i - 1, the scores of i) and then its weights, the
// second the weights of i - 1 first, so that the matrix pipe has one wave's products while the other's exponentials
// issue.
__device__ __forceinline__ bool attend_walk(Queries& w, int begin, int end, bool idle, bool second, const _Float16* lds,
                                            const _Float16* qlo, const Shared& sh) {
  const int blocks = (end - begin + kBlock - 1) / kBlock;
  lds_barrier();
  const int kunit = walk_scale(sh.meta[0]), vunit = walk_scale(sh.meta[0] + 4);
  const float c = scale_of(w, kunit);
  w.ev = vunit;
  lds_barrier();
  lds_barrier();
  const bool blunt = __ballot(c > kSharp) != 0;  // the walk's scale is not for these queries: each block's is looked at
  bool have = false, moved = blunt, ever = false;  // whether a block was apart
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
      const int live = w.limit - key0;
      const bool apart = moved || __builtin_amdgcn_readfirstlane(other_scales) != 0;
      if (apart) {
        ever = true;
        if (apart_scores(w, s, sh.meta[i & 3], kunit, vunit, c, live > 0)) idle = true;
        moved = blunt || __ballot(w.ev != vunit) != 0;
      }
      hide(s, live, now);
      const float lift = (float)kLift - move_max(w, largest_of(s) * c);
      if (apart) apart_weights(w, s, sh.meta[i & 3], vunit, c, lift);
      w.l += weigh(s, c, lift, p);
      if (live > 0) w.most = max(w.most, w.ev);
    }
    if (!second) lds_barrier();
  }
  // (weights that took up binades are off by as much beside small values as beside large ones)
  const int top = sh.top != 0 && ever ? kMaxExp : sh.top;
  return !idle && __ballot(faint(w, w.limit - begin, top)) == 0;
}

__global__ void __launch_bounds__(64 * (kTileWaves + kStageWaves), 3) k_chunk_tiles(Attend p) {
  __shared__ __align__(16) _Float16 lds[kLdsHalves];
  __shared__ __align__(16) Shared sh;
  const ChunkArgs& a = p.a;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  Work qt;
  if (!find_work(p, qt) || qt.begin >= qt.stop) return;
  if (wave >= kTileWaves) {
    const RowWalk rows{a.pool + a.layer_off + (int64_t)qt.head * kD, a.lookup + (int64_t)qt.n * a.lookup_cols, a.page_stride,
                       a.slot_stride, a.P, a.pages - 1, qt.stop, nullptr, nullptr, 0};
    convert_walk(rows, a.kv_stride, qt.begin, wave - kTileWaves, lds, sh);
    return;
  }
  const int t0 = qt.t0 + 32 * wave;
  const bool idle = t0 > qt.t_last;  // a wave without queries
  Queries w;
  _Float16* qlo = lds + 2 * kKHalves + 3 * kVHalves + wave * kQHalves;
  const int my_t = min(t0 + (lane & 31), qt.t_last);
  load_queries(w, qlo, p.in.q + (int64_t)my_t * a.in_stride + (int64_t)qt.head * kD, p.scale,
               min(rows_of(a, qt, my_t), qt.stop));
  const bool held = attend_walk(w, qt.begin, qt.stop, idle, wave >= kTileWaves / 2, lds, qlo, sh);
  if (idle) return;
  if (!held) {
    const Attend again = arguments_again<Attend>();
    find_work(again, qt);
    attend_in_fp32(w, again, qt, qt.t0 + 32 * wave, qt.begin, kBlock, false, (float*)lds + wave * 32 * kWave + lane_now());
  }
  const Attend to = arguments_again<Attend>();
  const int t = qt.t0 + 32 * wave + (lane_now() & 31);  // not kept through the walk
  store_queries(w, to.a, min(t, qt.t_last), t <= qt.t_last, qt.head, qt.split, qt.all_rows <= to.cuts.split_rows, to.out,
                to.part, to.weights);
}

// k_chunk_few: 32 queries a workgroup, whose 4 waves take the rows' blocks in turn, each straight from memory into the
// operands' lanes (keys: lane (row l % 32, columns 8 i + 4 (l / 32)); values: lane (columns 4 (l % 32) on, rows
// 16 t + 8 (j / 4) + 4 (l / 32) + j % 4)), and join their sums in LDS.
//
// Bound by the trips to memory where there are few rows (metadata; queries, page and positions; rows and tables: 11 us
// for 4 tokens over 300 rows) and by the rows' bytes where there are many: 8 requests of 7 over 1150 rows, 68 MB, in
// 21 us, 3.2 TB/s.  (The form in fp32 behind it costs 0.8 of them by being there, whichever way it is called.)  No row goes
// by way of LDS, so two workgroups share a CU, and one's loads are under way while the other multiplies.
constexpr int kFewWaves = 4;
constexpr int kFewLog2 = 5;  // queries of a workgroup
constexpr int kFewSplitRows = kFewWaves * 64 * kBlock;

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

// The last block of a wave, which begins with it.
__device__ __forceinline__ int few_first(const Work& w, int wave) {
  return w.begin + ((w.stop - w.begin + kBlock - 1) / kBlock - 1 - wave) * kBlock;
}

__global__ void __launch_bounds__(64 * kFewWaves, 2) k_chunk_few(Attend p) {
  const ChunkArgs& a = p.a;
  const Rope& rope = p.rope;
  const Inputs& in = p.in;
  const float scale = p.scale;
  __shared__ __align__(16) float sums[kFewWaves][32 * kD];  // the waves' sums, before that the fp32 form's stash,
  _Float16* const qs = (_Float16*)sums;             // and first the queries' operands, [part][step][lane][8]
  __shared__ float peak[kFewWaves][32], total[kFewWaves][32];
  __shared__ int q_exp[32], redo[kFewWaves];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  Work qt;
  if (!find_work(p, qt)) return;
  const int head = qt.head, t_last = qt.t_last, begin = qt.begin, end = qt.stop;
  if (qt.split == 0)  // new rows that none attends
    for (int t = qt.t0 + wave; t <= t_last; t += kFewWaves)
      if ((int64_t)qt.cached + (t - qt.first) >= a.attend_max) store_pair(a, rope, in, qt, t, head, lane);
  if (begin >= end) return;
  const float* pool = a.pool + a.layer_off + (int64_t)head * kD;
  const uint32_t* lookup = a.lookup + (int64_t)qt.n * a.lookup_cols;
  const uint32_t row_bytes = (uint32_t)a.slot_stride * 4u;
  const auto row_base = [&](int row) {
    return pool + (int64_t)min(ldc(lookup + row / a.P), (uint32_t)(a.pages - 1)) * a.page_stride +
           (int64_t)(row % a.P) * a.slot_stride;
  };
  // rows from old_rows on are the inputs', those from my_rows on this workgroup's to store
  const int old_rows = qt.cached, my_rows = qt.cached + (qt.t0 - qt.first);
  const auto token_of = [&](int row) { return (int64_t)(qt.first + (row - qt.cached)); };
  FewStage k, v;
  int row_pos = 0;  // the position of this lane's key row, where it is a new one
  const auto load_k = [&](const float* base, int key0, int lane) {
    const int row = min(lane & 31, end - 1 - key0), h = lane >> 5;
    const char* from = (const char*)base + ((uint32_t)row * row_bytes + 16u * h);
    if (key0 + kBlock > old_rows) {
      if (key0 + row >= old_rows)
        from = (const char*)(in.k_new + token_of(key0 + row) * a.in_stride + (int64_t)head * kD + 4 * h);
      if (rope.positions != nullptr) row_pos = ldg(rope.positions + max(token_of(key0 + row), (int64_t)0));
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) k.x[i] = *(const UOCR_GLOBAL f32x4*)(from + 32 * i);
  };
  const auto v_row = [](int j, int h) { return 16 * (j / 8) + 8 * (j / 4 % 2) + 4 * h + j % 4; };
  const auto load_v = [&](const float* base, int key0, int lane) {
    const char* from = (const char*)(base + a.kv_stride);
    const int last = end - 1 - key0;
    if (key0 + kBlock <= old_rows) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        v.x[j] = *(const UOCR_GLOBAL f32x4*)(from + ((uint32_t)min(v_row(j, lane >> 5), last) * row_bytes +
                                                     16u * (lane & 31)));
    } else {
      const float* news = in.v_new + token_of(key0) * a.in_stride + (int64_t)head * kD;
      const uint32_t new_bytes = (uint32_t)a.in_stride * 4u;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int row = min(v_row(j, lane >> 5), last);
        const bool old = key0 + row < old_rows;
        v.x[j] = *(const UOCR_GLOBAL f32x4*)((old ? from : (const char*)news) +
                                             ((uint64_t)((uint32_t)row * (uint64_t)(old ? row_bytes : new_bytes)) +
                                              16u * (lane & 31)));
      }
    }
  };
  // The new rows of a block: keys rotated, this tile's own rows stored.
  const auto take_new = [&](int key0, int lane) {
    const int h = lane >> 5, row = key0 + (lane & 31);
    float* to = const_cast<float*>(row_base(key0));
    if (rope.positions != nullptr && row >= old_rows && row < end) {
      const int pos = min(max(row_pos, 0), rope.table_rows - 1);
      const float* ct = rope.cos_t + (int64_t)pos * kD + 4 * h;
      const float* st = rope.sin_t + (int64_t)pos * kD + 4 * h;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        rotate4(k.x[i], k.x[i + 8], *(const UOCR_GLOBAL f32x4*)(ct + 8 * i), *(const UOCR_GLOBAL f32x4*)(ct + 8 * i + 64),
                *(const UOCR_GLOBAL f32x4*)(st + 8 * i), *(const UOCR_GLOBAL f32x4*)(st + 8 * i + 64));
    }
    if (row >= my_rows && row < end) {
      float* p = to + (int64_t)(lane & 31) * a.slot_stride + 4 * h;
#pragma unroll
      for (int i = 0; i < 16; ++i) *(UOCR_GLOBAL f32x4*)(p + 8 * i) = k.x[i];
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int r = v_row(j, h);
      if (key0 + r >= my_rows && key0 + r < end)
        *(UOCR_GLOBAL f32x4*)(to + a.kv_stride + (int64_t)r * a.slot_stride + 4 * (lane & 31)) = v.x[j];
    }
  };
  // The blocks are dealt from the last one, which has the new rows: their latencies begin first.  What does not wait
  // for one another is asked for together: the first block's page, the queries and their positions; then the rows
  // and the tables.
  const int first = few_first(qt, wave);
  {
    constexpr int R = 32 / kFewWaves, kPieces = 16 / kFewWaves, kStep = kD / kPieces;
    const float* base = first >= begin ? row_base(first) : pool;
    // the queries' operands: each wave 32 / kFewWaves of them, lane (query l % R, columns kStep i + 4 (l / R))
    const int row = wave * R + lane % R, col = 4 * (lane / R), t = min(qt.t0 + row, t_last);
    const float* src = in.q + (int64_t)t * a.in_stride + (int64_t)head * kD + col;
    int pos = 0;
    if (rope.positions != nullptr) pos = ldg(rope.positions + t);
    f32x4 x[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) x[i] = *(const UOCR_GLOBAL f32x4*)(src + kStep * i);
    __builtin_amdgcn_sched_barrier(0);
    if (first >= begin) {
      load_k(base, first, lane);
      load_v(base, first, lane);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (rope.positions != nullptr) {
      pos = min(max(pos, 0), rope.table_rows - 1);
      const float* ct = rope.cos_t + (int64_t)pos * kD + col;
      const float* st = rope.sin_t + (int64_t)pos * kD + col;
#pragma unroll
      for (int i = 0; i < kPieces / 2; ++i)
        rotate4(x[i], x[i + kPieces / 2], *(const UOCR_GLOBAL f32x4*)(ct + kStep * i),
                *(const UOCR_GLOBAL f32x4*)(ct + kStep * i + 64), *(const UOCR_GLOBAL f32x4*)(st + kStep * i),
                *(const UOCR_GLOBAL f32x4*)(st + kStep * i + 64));
    }
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) m = amax3(amax3(m, x[i].x, x[i].y), x[i].z, x[i].w);
    uint32_t bits = __float_as_uint(m);  // a query's lanes are R apart
    bits = max(bits, other<32>(bits));
    bits = max(bits, other<16>(bits));
    bits = max(bits, ror<8>(bits));
    const int e = query_exp(bits);
    q_exp[row] = e;
    const float up = __builtin_copysignf(pow2_of(141 - e), scale);  // the scale's sign goes into the query
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int d = kStep * i + col;
      const f32x4 y = x[i] * up;
      uint32_t l0, l1;
      const uint32_t h0 = split2(y.x, y.y, l0), h1 = split2(y.z, y.w, l1);
      _Float16* at = qs + (d / 16) * kFrag + ((d / 4 % 2) * 32 + row) * 8 + (d / 8 % 2) * 4;
      *(u32x2*)at = u32x2{h0, h1};
      *(u32x2*)(at + kQHalves) = u32x2{l0, l1};
    }
  }
  __syncthreads();
  Queries w;
  w.exp = q_exp[lane & 31];
  const int my_t = min(qt.t0 + (lane & 31), t_last);
  start_queries(w, scale, min(rows_of(a, qt, my_t), end));
  int kunit = 0, vunit = 0;
  bool held = true;  // whether the pairs hold all so far
  float top = 0.0f;  // the largest of the lane's values
#pragma unroll 1
  for (int key0 = first; key0 >= begin; key0 -= kFewWaves * kBlock) {
    const int lane = lane_now(), h = lane >> 5;
    const int last = end - 1 - key0, next = key0 - kFewWaves * kBlock;
    const int live = w.limit - key0;
    bool finite = true;
    if (key0 + kBlock > old_rows) take_new(key0, lane);
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
    top = fmaxf(top, vm);
    const float c = scale_of(w, ek);
    const bool attends = live > 0;
    // (a sum of larger values may leave no room for the block's unit)
    held = held && finite && __ballot(attends && (c > kSharp || w.most - ev > kRoom)) == 0;
    const float* next_base = next >= begin ? row_base(next) : pool;
    if (next >= begin) load_k(next_base, next, lane);
    hide(s, live, lane);
    const float lift = (float)kLift - move_max(w, largest_of(s) * c);
    // the queries that attend it to the block's unit; to the others nothing is added
    w.most = attends ? max(w.most, ev) : w.most;
    const int by = attends ? w.ev - ev : 0;
    if (__ballot(by != 0) != 0) {
      scale_sums(w, by);
      w.ev -= by;
    }
    Weights p;
    w.l += weigh(s, c, lift, p);
    const float vup = pow2_of(141 - ev);
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
    if (next >= begin) load_v(next_base, next, lane);
  }
  const uint32_t bits = wave_largest(top);
  held = held && __ballot(faint(w, min(w.limit - begin, first - begin + kBlock), bits == 0 ? 0 : clamp_exp(bits))) == 0;
  const int h = lane_now() >> 5;  // not kept through the walk
  const auto publish = [&] {
    const int lane = lane_now();
    const float l = w.l + other32(w.l);
    if (lane < 32) {
      peak[wave][lane] = w.m;
      total[wave][lane] = l;
    }
    if (lane == 0) redo[wave] = !held;
    __syncthreads();
  };
  publish();
  if (__builtin_amdgcn_readfirstlane(redo[0] | redo[1] | redo[2] | redo[3]) != 0) {
    const Attend again = arguments_again<Attend>();
    find_work(again, qt);
    __syncthreads();
    attend_in_fp32(w, again, qt, qt.t0, few_first(qt, wave), -kFewWaves * kBlock, true, sums[wave] + lane_now());
    publish();
  }
  // the waves' sums at one maximum, in the values' own unit
  const float l = total[wave][lane & 31];
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
  // query l % 32, a row of 128 floats whose 16-byte pieces are rotated by the query
  const auto at = [&](int r) { return (lane & 31) * kD + 4 * ((8 * (r / 4) + 4 * h + r % 4 + lane) & 31); };
  const auto mine = [&](int r) {
    f32x4 y;
#pragma unroll
    for (int u = 0; u < 4; ++u) y[u] = __builtin_ldexpf(w.o[u][r] * f, w.ev - 141);
    return y;
  };
#pragma unroll
  for (int r = 0; r < 16; ++r) *(f32x4*)(sums[wave] + at(r)) = mine(r);
  __syncthreads();
  const Attend to = arguments_again<Attend>();
  const bool whole = qt.all_rows <= to.cuts.split_rows;
  const int64_t stride = (int64_t)to.a.tokens * to.a.heads;
#pragma unroll
  for (int j = 0; j < 32 * 32 / (64 * kFewWaves); ++j) {
    const int i = j * 64 * kFewWaves + (int)threadIdx.x, query = i / 32, piece = i % 32;
    if (qt.t0 + query > qt.t_last) continue;
    const int from = query * kD + 4 * ((piece + query) & 31);
    f32x4 y = *(const f32x4*)(sums[0] + from);
#pragma unroll
    for (int k2 = 1; k2 < kFewWaves; ++k2) y += *(const f32x4*)(sums[k2] + from);
    const int64_t th = (int64_t)(qt.t0 + query) * to.a.heads + qt.head;
    *(UOCR_GLOBAL f32x4*)((whole ? to.out + th * kD : to.part + (qt.split * stride + th) * kD) + 4 * piece) = y;
  }
  if (!whole && wave == 0 && h == 0 && qt.t0 + lane <= qt.t_last)
    to.weights[qt.split * stride + ((int64_t)(qt.t0 + lane) * to.a.heads + qt.head)] =
        sum == 0.0f ? -kInf : m + log2_weight(sum);
}

// Joins the splits of a token's rows: a wave takes four heads of a token, four columns a lane, half a wave a head.  The
// splits hold normalised sums, so a split weighs what its weights sum to.  Bound by the trips to memory (metadata, then
// the splits): 3 us for 4 tokens, 6.0 us for 8 prompts of up to 512, 8.9 us for 2048 tokens of 3 splits (31 MB).  A wave
// to each head looked the metadata up ten times as often: 10.3 and 15 us.
constexpr int kJoinHeads = 4;
__global__ void __launch_bounds__(256) k_chunk_join(ChunkArgs a, float* out, const float* __restrict__ part,
                                                    const float* __restrict__ weights, int rows_log2, Divide by_split) {
  const int groups = (a.heads + kJoinHeads - 1) / kJoinHeads;
  const int64_t w = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  const int64_t t = w / groups;
  if (t >= a.tokens) return;
  QueryTile q;
  if (!chunk_of(a, (int)t, q)) return;
  const int t_last = min(q.first + (((((int)t - q.first) >> rows_log2) + 1) << rows_log2), q.end) - 1;  // of its tile
  const int splits = by_split(rows_of(a, q, t_last) - 1) + 1;
  if (splits == 1) return;  // written by its tile
  const int lane = lane_id(), h0 = (int)(w - t * groups) * kJoinHeads + lane / 32;
  const int64_t stride = (int64_t)a.tokens * a.heads;
  constexpr int kTwo = kJoinHeads / 2, kAtOnce = 4;  // heads of a lane, splits read together
  float m[kTwo], l[kTwo];
  f32x4 o[kTwo];
#pragma unroll
  for (int u = 0; u < kTwo; ++u) {
    m[u] = -kInf;
    l[u] = 0.0f;
    o[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  for (int s0 = 0; s0 < splits; s0 += kAtOnce) {
    float ws[kTwo][kAtOnce];
    f32x4 p[kTwo][kAtOnce];
#pragma unroll
    for (int u = 0; u < kTwo; ++u)
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int64_t at = min(s0 + j, splits - 1) * stride + t * a.heads + min(h0 + 2 * u, a.heads - 1);
        ws[u][j] = ldg(weights + at);
        p[u][j] = *(const UOCR_GLOBAL f32x4*)(part + at * kD + 4 * (lane & 31));
      }
#pragma unroll
    for (int u = 0; u < kTwo; ++u) {
      float mn = m[u];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) mn = fmaxf(mn, ws[u][j]);
      if (mn == -kInf) mn = 0.0f;
      const float keep = __builtin_amdgcn_exp2f(m[u] - mn);
      l[u] *= keep;
      o[u] *= keep;
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        if (s0 + j >= splits || ws[u][j] == -kInf) continue;  // a split without a weight has no sum
        const float f = __builtin_amdgcn_exp2f(ws[u][j] - mn);
        l[u] += f;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[u][e] = __builtin_fmaf(f, p[u][j][e], o[u][e]);
      }
      m[u] = mn;
    }
  }
#pragma unroll
  for (int u = 0; u < kTwo; ++u)
    if (h0 + 2 * u < a.heads)
      *(UOCR_GLOBAL f32x4*)(out + (t * a.heads + h0 + 2 * u) * kD + 4 * (lane & 31)) = o[u] / l[u];
}

}  // namespace

// How a call's rows are cut: tiles of 256 or of 32 queries, and splits of their rows where the tiles alone do not fill
// the device.  A tile of 256 has a CU to itself and converts each row once for all its queries, but a short chunk
// leaves most of it empty, and it has more to set up; tiles of 32 convert and read each row eight times as often.
// Measured, 10 heads, tiles of 256 / tiles of 32, in us: one request of 256 tokens 32 / 18, of 512 39 / 23, of 1024
// 46 / 58; of 256 tokens over 2000 cached rows 43 / 38, of 512 49 / 72, of 32 over 14000 50 / 46, of 64 53 / 58, of 128
// 59 / 95, of 512 202 / 348; four of 128 tokens 22 / 18, of 512 50 / 43; eight of 32 over 1000 rows 34 / 25, of 64
// 37 / 42, of 128 45 / 61; 64 of 33 over 300 73 / 57, of 64 95 / 73; 100 of 7 over 500 118 / 87.  The rule goes by two
// numbers and takes the slower near its border: one of 64 over 14000, eight of 64 over 1000, four of 512, by up to a
// sixth.  It was measured at 10 heads, and takes every request for an average one: a chunk of 2048 over 14001 rows, 456
// us alone, takes 1081 beside 31 of one token, and 4 tokens over 14001 rows 44 us alone and 110 beside seven empty chunks.
//
// More splits than fill the device once make some CUs take two pieces while others wait: two requests of 1024 in
// splits of 256 rows 55 us, of 1024 rows 86.  Tiles of 32 go two to a CU, and share it: 256, 384 and 512 pieces, eight
// requests of 7 over 1150 rows 27 / 24 / 27 us, of 32 over 1000 32 / 25 / 25, one of 8 over 14000 39 / 44 / 44.
namespace {
constexpr int kCus = 256;
struct Cut : Cuts {
  bool few;
};
Cut cut_of(int64_t tokens, int64_t requests, int heads, int attend_max) {
  Cut c{};
  c.few = requests > 0 && (tokens / requests <= 64 || tokens * attend_max < 1 << 19);
  c.rows_log2 = c.few ? kFewLog2 : kTileLog2;
  const int64_t rows = (int64_t)1 << c.rows_log2;
  c.slots = (int)(requests > 64 ? tokens / rows + requests
                                : tokens < requests ? tokens : (tokens - requests) / rows + requests);
  // Of about so many tiles (half of a request's last one is queries) each attends on average the part f of attend_max,
  // and has one split at least: tiles (1 - f + f splits) pieces.
  const double tiles = (double)std::max(requests, (tokens + rows - 1) / rows + (requests - 1) / 2) * heads;
  const double f = 1.0 - 0.5 * std::min(1.0, (double)tokens / ((double)std::max<int64_t>(1, requests) * attend_max));
  const int64_t splits = std::max(1, (int)(((c.few ? kCus * 3 / 2 : kCus) / std::max(1.0, tiles) - (1.0 - f)) / f));
  const int64_t least = c.few ? 4 * kBlock : 256, most = c.few ? kFewSplitRows : kMaxSplitRows;
  c.split_rows = (int)std::min(most, std::max(least, ((attend_max + splits - 1) / splits + 127) / 128 * 128));
  // two splits of 128 rows and their join take the time of one of 256, and a launch more
  if (c.few && attend_max <= 2 * least) c.split_rows = (int)(2 * least);
  c.splits = (int)(((int64_t)attend_max + c.split_rows - 1) / c.split_rows);
  c.by_split = divide_by(c.split_rows);
  c.by_slots = divide_by(std::max(1, c.slots));
  c.by_splits = divide_by(c.splits);
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
  const Rope rope{p.positions, p.cos_table, p.sin_table, p.table_rows};
  const Cut c = cut_of(p.tokens, p.requests, p.heads, p.attend_max);
  const int64_t pairs = p.tokens * p.heads, items = (int64_t)c.slots * p.heads * c.splits;
  const int64_t joins = p.tokens * ((p.heads + kJoinHeads - 1) / kJoinHeads);
  const dim3 by_pair((unsigned)((pairs + 3) / 4)), grid((unsigned)((items + 7) / 8 * 8));
  // (where a wave counts the pieces, offsets that do not ascend may give each request all of them)
  if (items > (p.requests <= 64 ? INT32_MAX / p.requests : INT32_MAX) - 8) return hipErrorInvalidValue;
  const Inputs in{p.q, p.k_new, p.v_new};
  float* part = (float*)p.workspace;
  float* weights = part + (int64_t)c.splits * pairs * kD;
  if (!c.few) {
    UOCR_LAUNCH("chunk_store", k_chunk_store, by_pair, dim3(256), 0, s, a, rope, in, p.out);
    const bool rotated_q = p.positions != nullptr;  // they wait in out
    if (rotated_q) a.in_stride = (int64_t)p.heads * kD;
    const Attend tiles{a, Rope{}, Inputs{rotated_q ? p.out : p.q, nullptr, nullptr}, p.scale, p.out, part, weights, c};
    UOCR_LAUNCH("chunk_tiles", k_chunk_tiles, grid, dim3(64 * (kTileWaves + kStageWaves)), 0, s, tiles);
  } else {
    const Attend few{a, rope, in, p.scale, p.out, part, weights, c};
    UOCR_LAUNCH("chunk_few", k_chunk_few, grid, dim3(64 * kFewWaves), 0, s, few);
  }
  if (c.splits > 1)
    UOCR_LAUNCH("chunk_join", k_chunk_join, dim3((unsigned)((joins + 3) / 4)), dim3(256), 0, s, a, p.out, part, weights,
                c.rows_log2, c.by_split);
  return hipGetLastError();
}

}  // namespace uocr
