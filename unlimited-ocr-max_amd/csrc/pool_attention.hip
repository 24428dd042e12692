// Attention over a KV page pool that holds int8, and of trees of drafted tokens over either pool: the decode op and its
// form for a chunk (unlimited_ocr_max/decoder.py:425-437, store_k/v_cache_ragged then flash_attention_ragged; the
// pages and their rows of unlimited_ocr_max/kv_cache.py:1-36).
//
//   fp32 pool  [pages][2 (k, v)][layers][P][heads][D] floats, D = 128
//   int8 pool  [pages][2 (k, v)][layers][P][slot] bytes; a slot is a row: its heads' 128 values each, then a float
//              scale of each head, padded to a multiple of 128 bytes.  A value stands for itself times the scale.
//
// Token t of request n has a new row (its k and v), which is stored first, and attends a set of its request's rows:
//   out = sum_r softmax_r(scale * q.k_r) v_r, 0 where the set is empty;
//   decode  rows [0, attend_length + 1), the new row at write_index (a ring's may be anywhere),
//   chunk   rows [0, cached + i], i the token's place in its chunk, the new row the last of them,
//   tree    rows [0, cached) and row cached + j for every bit j < 64 of the token's mask.
// What is attended is what the pool holds: an int8 pool's new rows count as they were rounded, so that a prompt's
// results do not depend on how it was cut.
//
// Products: the matrix instruction of bf16, fp32 sums.  An fp32 operand is held as three bf16 numbers whose sum it is
// (24 bits, of its own exponent: no scale is shared, and nothing is too large); an int8 one is a bf16 number.  So a
// product with an int8 operand is exact in three, and six of the nine of two fp32 operands leave out 2^-21 of the product
// where the lower bits of both are ones, some 2^-24 on average, always towards zero as the terms are cut off: what the sums
// round is about as much (outputs are within 1e-6 of 64 bits' either way), and two products more would be a third more of
// the matrix instructions.  bf16 ends at 2^-133: of values below 2^-100 the lower bits are lost.
// The scores are S^T = K Q^T and the results O^T = V^T P^T: a lane owns a query, and its 16 scores of a block of 32 rows
// come in the order in which the second product wants the weights.
#include <algorithm>
#include <type_traits>

#include "chunk_device.h"
#include "int8_rows.h"
#include "uocr_kernels.h"

namespace uocr {

namespace {

constexpr int kBlock = 32;     // rows a wave takes at a time: the rows of one matrix instruction
constexpr int kQueries = 32;   // of a workgroup
constexpr int kQueriesLog2 = 5;
constexpr int kWaves = 4, kRound = kWaves * kBlock;
constexpr int kThreads = kWaves * kWave;
constexpr float kInf = __builtin_huge_valf();
// A maximum may lag by so many binades before the sums are rescaled (the weights are floats: nothing is lost).
constexpr float kSlack = 8.0f;

enum Mode { kOne, kCausal, kTree };
constexpr PoolForm form_of(Mode m) { return m == kOne ? kPoolDecode : m == kCausal ? kPoolChunk : kPoolTree; }

struct PoolArgs {
  char* pool;
  int64_t page_bytes, kv_bytes, layer_bytes;  // of a page, of its k half, from its start to the layer
  int slot_bytes;
  int P, heads, pages;
  int max_rows;  // lookup_cols * P: rows a lookup row can address
  const uint32_t* lookup;
  int lookup_cols;
  int requests, tokens;
  const uint32_t* cache_lengths;  // decode: attend lengths
  const int32_t* offsets;         // [requests + 1]; decode: none, request i is token i
  const uint32_t* write_index;    // decode
  const int64_t* visible;         // tree
  int attend_max;
  int64_t in_stride;  // floats between rows of q / k_new / v_new
  const float* q;
  const float* k_new;
  const float* v_new;
  float* out;
  float scale;
  Rope rope;
  bool stores;  // whether the attending kernel stores the new rows, else k_pool_store has
};

// Where row r of request n is, and head h's values in it.
__device__ __forceinline__ char* slot_of(const PoolArgs& a, int n, int r) {
  const uint32_t page = min(ldg(a.lookup + (int64_t)n * a.lookup_cols + r / a.P), (uint32_t)(a.pages - 1));
  return a.pool + (int64_t)page * a.page_bytes + a.layer_bytes + (int64_t)(r % a.P) * a.slot_bytes;
}

// Stores k and v of kItems (token, head) pairs as rows of request n, whose loads are under way together: token t's heads from h0
// on as row `row` (kOf == kHeads), or head h0 of the tokens t, t + kWaves, ... below `end` as the rows row, row + kWaves, ...
// Half of the wave has the key, half the value, a lane 4 columns.
enum Items { kHeads, kTokens };
template <bool kInt8, Items kOf, int kItems>
__device__ __forceinline__ void store_rows(const PoolArgs& a, int n, int row, int t, int end, int h0) {
#pragma clang fp contract(off)
  const int lane = lane_id(), c = lane & 31;
  const bool key = lane < 32, turn = a.rope.positions != nullptr;
  const float* x = (key ? a.k_new : a.v_new) + 4 * c;
  f32x4 y[kItems], pair[kItems];  // the pair of column d is d +- 64
  int pos[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int ti = kOf == kHeads ? t : min(t + i * kWaves, end - 1), h = kOf == kHeads ? min(h0 + i, a.heads - 1) : h0;
    const int64_t at = (int64_t)ti * a.in_stride + (int64_t)h * kD;
    y[i] = *(const UOCR_GLOBAL f32x4*)(x + at);
    if (turn) {
      pair[i] = *(const UOCR_GLOBAL f32x4*)(x + at + (c < 16 ? 64 : -64));
      pos[i] = kOf == kTokens || i == 0 ? min(max(ldg(a.rope.positions + ti), 0), a.rope.table_rows - 1) : pos[0];
    }
  }
  char* slot[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i)
    slot[i] = kOf == kHeads && i > 0 ? slot[0]
                                     : slot_of(a, n, kOf == kHeads ? row : min(row + i * kWaves, row + (end - 1 - t))) + (key ? 0 : a.kv_bytes);
  if (turn) {
    f32x4 cs[kItems], sn[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int64_t at = (int64_t)pos[i] * kD + 4 * c;
      cs[i] = kOf == kHeads && i > 0 ? cs[0] : *(const UOCR_GLOBAL f32x4*)(a.rope.cos_t + at);
      sn[i] = kOf == kHeads && i > 0 ? sn[0] : *(const UOCR_GLOBAL f32x4*)(a.rope.sin_t + at);
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float turned = y[i][e] * cs[i][e] + (c < 16 ? -pair[i][e] : pair[i][e]) * sn[i][e];
        y[i][e] = key ? turned : y[i][e];
      }
  }
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int h = kOf == kHeads ? h0 + i : h0;
    if (kOf == kHeads ? h >= a.heads : t + i * kWaves >= end) break;
    if constexpr (kInt8) {
      uint32_t most = max(max(abs_bits(y[i].x), abs_bits(y[i].y)), max(abs_bits(y[i].z), abs_bits(y[i].w)));
#pragma unroll
      for (int off = 1; off <= 8; off *= 2) most = max(most, (uint32_t)__shfl_xor((int)most, off, kWave));
      const float scale = row_scale(max(most, other<16>(most)));
      const uint32_t q = to_int8x4(y[i].x, y[i].y, y[i].z, y[i].w, scale);
      stg((uint32_t*)(slot[i] + h * kD) + c, q);
      if (c == 0) stg((float*)(slot[i] + a.heads * kD) + h, scale);
    } else {
      *(UOCR_GLOBAL f32x4*)((float*)slot[i] + h * kD + 4 * c) = y[i];
    }
  }
}

// One wave per (token, 4 heads), which waits for the request's words once.  Bound by memory: 2900 tokens of ten heads in 11 us,
// 3.4 TB/s.  Queries that come before RoPE are rotated where they are read.
constexpr int kStoreHeads = 4;
template <bool kInt8>
__global__ void __launch_bounds__(256) k_pool_store(PoolArgs a) {
  const int groups = (a.heads + kStoreHeads - 1) / kStoreHeads;
  const int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  if (item >= (int64_t)a.tokens * groups) return;
  const int t = (int)(item / groups), h0 = (int)(item % groups) * kStoreHeads;
  Chunk c;
  if (!chunk_of(a, t, c)) return;
  const int64_t row = (int64_t)c.cached + (t - c.first);
  if (row < a.max_rows) store_rows<kInt8, kHeads, kStoreHeads>(a, c.n, (int)row, t, t + 1, h0);  // else past what the lookup row addresses
}

// ------------------------------------------------------------------ which piece of the work a workgroup takes

// A call's rows are cut into splits where the tiles of queries alone do not fill the device.
struct PoolCuts {
  int split_rows, splits, slots;  // rows of a split at least; splits of a tile and tiles of queries at most
  int fill;                       // up to 64 requests: pieces of a head that fill the device (0: splits have split_rows)
  int groups;                     // a request's pieces side by side: its heads, or pairs of them
  bool few;                       // decode: fewer (request, head) pairs than half the CUs
  bool tiles;                     // k_pool_tiles takes the queries
  bool round;                     // pieces go round the XCDs
  Divide by_split, by_heads;
};
// A tile of a request's tokens [t0, t_last], a head, and rows [begin, stop) of those that the tile attends.
struct Piece : Chunk {
  int t0, t_last, head, split, begin, stop;
  bool whole;  // no other piece of the tile
};
// Rows that a tile attends whose last token is t_last.
template <Mode kMode>
__device__ __forceinline__ int tile_rows(const PoolArgs& a, int cached, int length, int last) {
  const int64_t rows = (int64_t)cached + (kMode == kCausal ? last + 1 : min(length, 64));
  return (int)min(rows, (int64_t)a.attend_max);
}
// Rows of each of a request's splits, where one has at most `most`: of a size, to a round of the waves.  (None is empty: with
// n splits of at most `most` rows there are more than (n - 1) * most.)
__device__ __forceinline__ int rows_of_split(int rows, int most) {
  const int n = (rows - 1) / most + 1;
  return n == 1 ? rows : ((rows - 1) / n / kRound + 1) * kRound;
}
__device__ __forceinline__ Chunk request_at(const PoolArgs& a, int i) {
  Chunk c;
  c.n = i;
  c.first = ldg(a.offsets + i);
  c.end = min(ldg(a.offsets + i + 1), a.tokens);
  c.cached = (int)min(ldg(a.cache_lengths + i), (uint32_t)a.max_rows);
  return c;
}
// Items go to the XCDs in stretches, the tiles that read the same rows of a head side by side and the heads next: their XCD
// reads the rows once, and the heads of an int8 row share the line of their scales.  (Pieces that go round the XCDs: eight
// trees of 61 over 4000 rows 130 us for 110.)  Up to 64 requests every wave counts the pieces
// that there are, and cuts them so that the device is filled by them once: the host does not know the lengths (with splits
// from the longest, eight trees over 1667 to 4000 rows 92 us for 81).  Of more requests, a piece is a slot, whose tile and
// split may not exist.  most_rows: where the join finds the rows of a split.
template <Mode kMode, int kLog2>
__device__ __forceinline__ bool find_piece(const PoolArgs& a, const PoolCuts& c, int* most_rows, Piece& p) {
  const int turn = (int)(blockIdx.x / 8), xcd = (int)(blockIdx.x % 8);
  uint32_t most = (uint32_t)c.split_rows;
  int j, rows;  // the tile; rows of a split
  if (a.requests <= 64) {
    const Chunk mine = request_at(a, min(lane_id(), a.requests - 1));
    const bool some = lane_id() < a.requests && mine.first >= 0 && mine.first < mine.end;
    const int length = some ? mine.end - mine.first : 0;
    const int tiles = (length + (1 << kLog2) - 1) >> kLog2;
    const int all = some ? tile_rows<kMode>(a, mine.cached, length, length - 1) : 1;
    if (c.fill > 0) {
      // (a tile's last split leaves half of one empty)
      float sum = (float)tiles * (float)all;
      sum += from_up<32>(sum), sum += from_up<16>(sum), sum += from_up<8>(sum);
      sum += from_up<4>(sum), sum += from_up<2>(sum), sum += from_up<1>(sum);
      sum = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(sum)));
      const float guess = sum / (float)max(1, c.fill - wave_sum_i(tiles) / 2);
      most = max(most, ((uint32_t)fminf(guess, (float)a.attend_max) / kRound + 1) * kRound);
      while (most < (uint32_t)a.attend_max && wave_sum_i(tiles * (int)((uint32_t)(all - 1) / most + 1)) > c.fill)
        most += max(most / 8 / kRound, 1u) * kRound;
    }
    const int my_rows = rows_of_split(all, (int)most);
    // tiles whose last query comes before the row
    const auto before = [&](uint32_t row, int cached) {
      return kMode == kCausal && (int)row > cached ? ((int)row - cached) >> kLog2 : 0;
    };
    int pieces = tiles;
    for (uint32_t row = my_rows; __ballot(row < (uint32_t)all) != 0;)
      if (row < (uint32_t)all) pieces += tiles - before(row, mine.cached), row += my_rows;
    const int upto = wave_scan_i(pieces), total = __builtin_amdgcn_readlane(upto, 63);
    if (c.splits > 1 && blockIdx.x == 0) stg(most_rows, (int)most);
    const int per = (total * a.heads + 7) / 8;
    const int turns = c.by_heads(turn), item = c.round ? turn + (7 * turns + xcd) * a.heads : xcd * per + turn;
    if (item >= total * a.heads || (!c.round && turn >= per)) return false;
    const int at = __popcll(__ballot(upto <= c.by_heads(item)));  // the request whose pieces reach past it
    int left = item - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(pieces, at)) * a.heads;
    p.n = at;
    p.first = __builtin_amdgcn_readlane(mine.first, at);
    p.end = __builtin_amdgcn_readlane(mine.end, at);
    p.cached = __builtin_amdgcn_readlane(mine.cached, at);
    rows = __builtin_amdgcn_readlane(my_rows, at);
    j = __builtin_amdgcn_readlane(tiles, at) - 1;
    p.split = 0;
    int here;  // tiles that have the split
    for (uint32_t row = 0;; row += rows, ++p.split) {
      here = j + 1 - before(row, p.cached);
      if (left < here * a.heads) break;
      left -= here * a.heads;
    }
    p.head = left / here;
    j -= left - p.head * here;
  } else {
    const int item = xcd * (int)(gridDim.x / 8) + turn;
    const int cell = c.by_heads(item), slot = cell / c.splits;  // the splits of a tile one after the other
    if (c.splits > 1 && blockIdx.x == 0) stg(most_rows, (int)most);
    if (slot >= c.slots) return false;
    p.head = item - cell * a.heads;
    p.split = cell - slot * c.splits;
    (Chunk&)p = find_chunk(a, kLog2, true, slot);
    j = slot - ((p.first >> kLog2) + p.n);
    if (p.first < 0 || j < 0 || (int64_t)j << kLog2 >= p.end - p.first) return false;
    rows = rows_of_split(tile_rows<kMode>(a, p.cached, p.end - p.first, p.end - p.first - 1), c.split_rows);
  }
  p.t0 = p.first + (j << kLog2);
  p.t_last = min(p.t0 + (1 << kLog2), p.end) - 1;
  const int all = tile_rows<kMode>(a, p.cached, p.end - p.first, p.t_last - p.first);
  p.whole = all <= rows;
  if ((int64_t)p.split * rows >= all) return false;
  p.begin = p.split * rows;
  p.stop = p.begin + min(rows, all - p.begin);
  return true;
}

// ------------------------------------------------------------------ operands

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ bf16x8 bf(u32x4 v) { return __builtin_bit_cast(bf16x8, v); }
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
// The upper halves of a and b, a's in the lower half.
__device__ __forceinline__ uint32_t uppers(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ float upper(float a) { return __uint_as_float(__float_as_uint(a) & 0xffff0000u); }
// a and b as sums of three bf16 numbers each, the bits of a float from the first on: exact.
__device__ __forceinline__ uint32_t split3(float a, float b, uint32_t& mid, uint32_t& lo) {
  const float ra = a - upper(a), rb = b - upper(b);
  mid = uppers(ra, rb);
  lo = uppers(ra - upper(ra), rb - upper(rb));
  return uppers(a, b);
}
// Signed bytes B and C of v as a bf16 pair.
template <int B, int C>
__device__ __forceinline__ uint32_t bytes_bf16(uint32_t v, uint32_t w) {
  return uppers(i8_to_f32<B>((int)v), i8_to_f32<C>((int)w));
}

constexpr int kFrag = 64 * 8;                 // numbers of an operand: 8 of each lane
constexpr int kQTerm = 8 * kFrag;             // of a term of the queries, [step][lane][8]

// 32 rows of keys or of values on their way from memory to the operands of one wave.
template <bool kInt8>
struct Stage;
template <>
struct Stage<false> {
  f32x4 x[16];
};
template <>
struct Stage<true> {
  uint32_t x[16];
  float scale;  // of row l % 32
};

// Slot (lane half h, j) of step t of the first product is column 32 (t / 2) + 16 h + 8 (t % 2) + j;
// slot (h, j) of step t of the second one is row 16 t + 8 (j / 4) + 4 h + j % 4 of the block.
__device__ __forceinline__ int value_row(int j, int h) { return 16 * (j / 8) + 8 * (j / 4 % 2) + 4 * h + j % 4; }

// `from`: the block's first slot; last: its last row that is read.
template <bool kInt8>
__device__ __forceinline__ void load_keys(Stage<kInt8>& k, const PoolArgs& a, const char* from, int head, int last, int lane) {
  const int h = lane >> 5;
  const uint32_t row = (uint32_t)(min(lane & 31, last) * a.slot_bytes), at = (uint32_t)head * kD;
  if constexpr (kInt8) {
    k.scale = *(const UOCR_GLOBAL float*)(from + (row + (uint32_t)(a.heads * kD + 4 * head)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x4 v = *(const UOCR_GLOBAL u32x4*)(from + (row + at + 16u * h) + 32 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) k.x[4 * i + e] = v[e];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      k.x[i] = *(const UOCR_GLOBAL f32x4*)(from + (row + 4 * at + 64u * h) + 128 * (i / 4) + 16 * (i % 4));
  }
}
template <bool kInt8>
__device__ __forceinline__ void load_values(Stage<kInt8>& v, const PoolArgs& a, const char* from, int head, int last,
                                            int lane) {
  from += a.kv_bytes;
  const int h = lane >> 5, c = lane & 31;
  if constexpr (kInt8)
    v.scale = *(const UOCR_GLOBAL float*)(from + (uint32_t)(min(c, last) * a.slot_bytes + a.heads * kD + 4 * head));
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const uint32_t row = (uint32_t)(min(value_row(j, h), last) * a.slot_bytes + head * (kInt8 ? kD : 4 * kD));
    if constexpr (kInt8)
      v.x[j] = *(const UOCR_GLOBAL uint32_t*)(from + (row + 4u * c));
    else
      v.x[j] = *(const UOCR_GLOBAL f32x4*)(from + (row + 16u * c));
  }
}

// S^T of a block: 32 rows by 32 queries.  q: the queries' terms in LDS.
template <bool kInt8>
__device__ __forceinline__ f32x16 scores(const Stage<kInt8>& k, const uint16_t* q, int lane) {
  f32x16 s = {};
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const bf16x8 qh = *(const bf16x8*)(q + t * kFrag + lane * 8);
    const bf16x8 qm = *(const bf16x8*)(q + kQTerm + t * kFrag + lane * 8);
    const bf16x8 ql = *(const bf16x8*)(q + 2 * kQTerm + t * kFrag + lane * 8);
    if constexpr (kInt8) {
      u32x4 kk;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t x = k.x[4 * (t / 2) + 2 * (t % 2) + e];
        kk[2 * e] = bytes_bf16<0, 1>(x, x);
        kk[2 * e + 1] = bytes_bf16<2, 3>(x, x);
      }
      s = mfma(bf(kk), ql, s);
      s = mfma(bf(kk), qm, s);
      s = mfma(bf(kk), qh, s);
    } else {
      u32x4 hi, mid, lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x4 x = k.x[2 * t + e / 2];
        uint32_t m, l;
        hi[e] = split3(x[2 * (e % 2)], x[2 * (e % 2) + 1], m, l);
        mid[e] = m;
        lo[e] = l;
      }
      s = mfma(bf(lo), qh, s);
      s = mfma(bf(hi), ql, s);
      s = mfma(bf(mid), qm, s);
      s = mfma(bf(mid), qh, s);
      s = mfma(bf(hi), qm, s);
      s = mfma(bf(hi), qh, s);
      __builtin_amdgcn_sched_barrier(0);  // no steps' terms ahead: they would take the registers of the rows under way
    }
  }
  return s;
}


struct Attend {
  PoolArgs a;
  PoolCuts cuts;
  float* part;  // [split][token][head][D], where a tile has several splits
  float* tops;  // [split][token][head][2]: the maximum (log2) and the sum of the weights
  int* most_rows;  // [1]: rows of a split at most
};

// A lane's query: running maximum (log2), the sum of the weights of the lane's rows, the weighted values.
struct Running {
  float m, l;
  f32x16 o[4];  // register r of o[u]: column 4 (8 (r / 4) + 4 h + r % 4) + u
};

__device__ __forceinline__ void start(Running& w) {
  w.m = -kInf;
  w.l = 0.0f;
#pragma unroll
  for (int u = 0; u < 4; ++u) w.o[u] = f32x16{};
}

// Which of a block's rows a lane's query attends: those below `live`, or, for a tree, the bits of a word.
__device__ __forceinline__ uint32_t tree_rows(uint64_t visible, int off, int live) {
  uint32_t set;
  if (off >= 0)
    set = off < 64 ? (uint32_t)(visible >> off) : 0u;
  else
    set = off > -32 ? (uint32_t)(visible << -off) | ((1u << -off) - 1u) : ~0u;
  return live >= 32 ? set : set & ((1u << max(live, 0)) - 1u);
}

// Scores (times log2 e) to weights: the maximum moves where it lags by more than kSlack, and what was summed follows.
__device__ __forceinline__ void weigh(Running& w, f32x16& s) {
  float mx = s[0];
#pragma unroll
  for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
  mx = fmaxf(mx, other32(mx));
  const bool up = mx > w.m + kSlack;
  if (__ballot(up) != 0) {
    const float alpha = up ? __builtin_amdgcn_exp2f(w.m - mx) : 1.0f;
    w.m = up ? mx : w.m;
    w.l *= alpha;
#pragma unroll
    for (int u = 0; u < 4; ++u) w.o[u] *= alpha;
  }
  const float off = w.m == -kInf ? 0.0f : w.m;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    s[r] = __builtin_amdgcn_exp2f(s[r] - off);
    w.l += s[r];
  }
}

// Step t of the second product: the weights of 8 rows as three terms, and the values' columns in turn.
template <int T>
__device__ __forceinline__ void split_weights(const f32x16& p, u32x4& hi, u32x4& mid, u32x4& lo) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t m, l;
    hi[e] = split3(p[8 * T + 2 * e], p[8 * T + 2 * e + 1], m, l);
    mid[e] = m;
    lo[e] = l;
  }
}
template <int T, int U>
__device__ __forceinline__ void add_column(Running& w, const Stage<true>& v, u32x4 ph, u32x4 pm, u32x4 pl) {
  u32x4 x;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = bytes_bf16<U, U>(v.x[8 * T + 2 * e], v.x[8 * T + 2 * e + 1]);
  w.o[U] = mfma(bf(x), bf(pl), w.o[U]);
  w.o[U] = mfma(bf(x), bf(pm), w.o[U]);
  w.o[U] = mfma(bf(x), bf(ph), w.o[U]);
}
template <int T, int U>
__device__ __forceinline__ void add_column(Running& w, const Stage<false>& v, u32x4 ph, u32x4 pm, u32x4 pl) {
  u32x4 hi, mid, lo;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t m, l;
    hi[e] = split3(v.x[8 * T + 2 * e][U], v.x[8 * T + 2 * e + 1][U], m, l);
    mid[e] = m;
    lo[e] = l;
  }
  w.o[U] = mfma(bf(lo), bf(ph), w.o[U]);
  w.o[U] = mfma(bf(hi), bf(pl), w.o[U]);
  w.o[U] = mfma(bf(mid), bf(pm), w.o[U]);
  w.o[U] = mfma(bf(mid), bf(ph), w.o[U]);
  w.o[U] = mfma(bf(hi), bf(pm), w.o[U]);
  w.o[U] = mfma(bf(hi), bf(ph), w.o[U]);
  __builtin_amdgcn_sched_barrier(0);
}
template <int T, bool kInt8>
__device__ __forceinline__ void add_values(Running& w, const Stage<kInt8>& v, const f32x16& p) {
  u32x4 hi, mid, lo;
  split_weights<T>(p, hi, mid, lo);
  add_column<T, 0>(w, v, hi, mid, lo);
  add_column<T, 1>(w, v, hi, mid, lo);
  add_column<T, 2>(w, v, hi, mid, lo);
  add_column<T, 3>(w, v, hi, mid, lo);
}

// The rows (bits of the block's) with a value that is not finite, whose values become 0: a row that a query does not
// attend must leave nothing in its sum, and one that it attends makes it NaN.
__device__ __forceinline__ uint32_t take_infinite(Stage<true>&) { return 0; }  // int8 is finite
__device__ __forceinline__ uint32_t take_infinite(Stage<false>& v) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, abs_bits(v.x[j][e]));
  if (__ballot(top >= 0x7f800000u) == 0) return 0;
  uint32_t bad = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) most = max(most, abs_bits(v.x[j][e]));
    const uint64_t who = __ballot(most >= 0x7f800000u);
    if ((uint32_t)who != 0) bad |= 1u << value_row(j, 0);
    if ((who >> 32) != 0) bad |= 1u << value_row(j, 1);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t none = abs_bits(v.x[j][e]) >= 0x7f800000u ? 0u : ~0u;
      v.x[j][e] = __uint_as_float(__float_as_uint(v.x[j][e]) & none);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  return bad;
}

// 32 queries of a head, whose rows' blocks the workgroup's waves take in turn and whose sums they join in LDS.  Every wave
// converts its own rows, from registers to registers: what it waits for is the next block's loads, and two workgroups on a CU
// wait in turn.  Of few rows bound by the trips to memory before the first block (15 tokens over 300 int8 rows 15 us); of
// many by the conversions and products, which take about as long as one another (eight trees of 26 to 61 over 1667 to 4000
// rows: int8 35 us, 1.7 TB/s; fp32, with twice the products and three times the conversions, 80 us, 2.9 TB/s).
template <bool kInt8, Mode kMode>
__global__ void __launch_bounds__(kThreads, 2) k_pool_attend(Attend p) {
  const PoolArgs& a = p.a;
  __shared__ __align__(16) float sums[kWaves][kQueries * kD];  // first the queries' terms, [term][step][lane][8]
  uint16_t* const qs = (uint16_t*)sums;
  __shared__ __align__(16) float row_scales[kWaves][2][kBlock];  // of a block's keys and values
  __shared__ float peak[kWaves][kQueries], total[kWaves][kQueries];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), h = lane >> 5;
  Piece w;
  if (!find_piece<kMode, kQueriesLog2>(a, p.cuts, p.most_rows, w)) return;
  const int stop = w.stop, head = w.head;
  // the first row of the request that no token attends
  const int unread = tile_rows<kMode>(a, w.cached, w.end - w.first, w.end - w.first - 1);
  const uint32_t* lookup = a.lookup + (int64_t)w.n * a.lookup_cols;
  const auto block_at = [&](int row) {
    return a.pool + (int64_t)min(ldc(lookup + row / a.P), (uint32_t)(a.pages - 1)) * a.page_bytes + a.layer_bytes +
           (int64_t)(row % a.P) * a.slot_bytes;
  };
  const int first = w.begin + kBlock * wave;
  Stage<kInt8> k, v;
  {
    // the queries' terms: thread (query tid / 8, octets tid % 8 and 8 on)
    const int query = (int)threadIdx.x / 8, d = 8 * ((int)threadIdx.x % 8), t = min(w.t0 + query, w.t_last);
    const float* src = a.q + (int64_t)t * a.in_stride + (int64_t)head * kD + d;
    f32x4 x[4] = {*(const UOCR_GLOBAL f32x4*)src, *(const UOCR_GLOBAL f32x4*)(src + 4),
                  *(const UOCR_GLOBAL f32x4*)(src + 64), *(const UOCR_GLOBAL f32x4*)(src + 68)};
    int pos = 0;
    if (a.rope.positions != nullptr) pos = min(max(ldg(a.rope.positions + t), 0), a.rope.table_rows - 1);
    const char* from = block_at(first);
    const bool early = !a.stores || first + kBlock <= w.cached;  // no row among them that this workgroup has yet to store
    if (first < stop && early) {
      load_keys(k, a, from, head, stop - 1 - first, lane);
      load_values(v, a, from, head, stop - 1 - first, lane);
    }
    if (a.stores) {
      // The new rows that this workgroup reads, and of its tile's tokens those that none does.  (Workgroups that read the
      // same rows store the same bits.)
      constexpr int kAtOnce = kInt8 ? 4 : 2;
      const int behind = w.first - w.cached;  // of a row, its token
      for (int r = max(w.begin, w.cached) + wave; r < stop; r += kAtOnce * kWaves)
        store_rows<kInt8, kTokens, kAtOnce>(a, w.n, r, behind + r, behind + stop, head);
      if (w.split == 0) {
        // tokens of the tile whose rows no token attends
        const int t0 = max(w.t0, behind + unread), end = (int)min((int64_t)w.t_last + 1, (int64_t)behind + a.max_rows);
        for (int t = t0 + wave; t < end; t += kAtOnce * kWaves)
          store_rows<kInt8, kTokens, kAtOnce>(a, w.n, t - behind, t, end, head);
      }
      __syncthreads();
      if (first < stop && !early) {
        load_keys(k, a, from, head, stop - 1 - first, lane);
        load_values(v, a, from, head, stop - 1 - first, lane);
      }
    }
    if (a.rope.positions != nullptr) {
      const float *ct = a.rope.cos_t + (int64_t)pos * kD + d, *st = a.rope.sin_t + (int64_t)pos * kD + d;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        rotate4(x[i], x[i + 2], *(const UOCR_GLOBAL f32x4*)(ct + 4 * i), *(const UOCR_GLOBAL f32x4*)(ct + 4 * i + 64),
                *(const UOCR_GLOBAL f32x4*)(st + 4 * i), *(const UOCR_GLOBAL f32x4*)(st + 4 * i + 64));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int col = d + 64 * i, step = 2 * (col / 32) + col / 8 % 2, half = col / 16 % 2;
      u32x4 hi, mid, lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t m, l;
        hi[e] = split3(x[2 * i + e / 2][2 * (e % 2)], x[2 * i + e / 2][2 * (e % 2) + 1], m, l);
        mid[e] = m;
        lo[e] = l;
      }
      uint16_t* at = qs + step * kFrag + (half * 32 + query) * 8;
      *(u32x4*)at = hi;
      *(u32x4*)(at + kQTerm) = mid;
      *(u32x4*)(at + 2 * kQTerm) = lo;
    }
  }
  const float c = a.scale * 1.44269504f;
  const int my_t = min(w.t0 + (lane & 31), w.t_last);
  // rows below `all` are attended by every query of the tile
  const int all = min(stop, kMode == kCausal ? w.cached + (w.t0 - w.first) + 1 : w.cached);
  const int limit = kMode == kCausal ? min(w.cached + (my_t - w.first) + 1, stop) : stop;
  uint64_t visible = 0;
  if constexpr (kMode == kTree) visible = (uint64_t)ldg(a.visible + my_t);
  Running run;
  start(run);
  __syncthreads();
  const auto walk = [&](auto careful) {
#pragma unroll 1
    for (int key0 = first; key0 < stop; key0 += kWaves * kBlock) {
      const int next = key0 + kWaves * kBlock;
      const char* next_base = next < stop ? block_at(next) : a.pool;
      f32x16 s = scores(k, qs, lane);
      f32x4 vs[4];
      if constexpr (kInt8) {
        row_scales[wave][h][lane & 31] = h == 0 ? k.scale * c : v.scale;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 ks = *(const f32x4*)&row_scales[wave][0][8 * g + 4 * h];
          vs[g] = *(const f32x4*)&row_scales[wave][1][8 * g + 4 * h];
#pragma unroll
          for (int e = 0; e < 4; ++e) s[4 * g + e] *= ks[e];
        }
        __builtin_amdgcn_wave_barrier();
      } else {
        s *= c;
      }
      __builtin_amdgcn_sched_barrier(0);
      if (next < stop) load_keys(k, a, next_base, head, stop - 1 - next, lane);
      const bool masked = key0 + kBlock > all;
      if (masked) {
        asm volatile("");  // a branch: as selects the masks would be a sixth of a block's instructions
        uint32_t set = 0;
        if constexpr (kMode == kTree) set = tree_rows(visible, key0 - w.cached, stop - key0);
        const int live = limit - key0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = 8 * (r / 4) + 4 * h + r % 4;
          const bool seen = kMode == kTree ? (set >> row & 1u) != 0 : row < live;
          s[r] = seen ? s[r] : -kInf;
        }
      }
      if constexpr (decltype(careful)::value) {
        const uint32_t bad = take_infinite(v);
        if (bad != 0) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (bad >> (8 * (r / 4) + 4 * h + r % 4) & 1u && s[r] != -kInf) run.l = __uint_as_float(0x7fc00000u);
        }
      }
      weigh(run, s);
      if constexpr (kInt8) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= vs[r / 4][r % 4];
        if (masked) {  // the scales of rows that are not attended may be anything
          asm volatile("");
          uint32_t set = 0;
          if constexpr (kMode == kTree) set = tree_rows(visible, key0 - w.cached, stop - key0);
          const int live = limit - key0;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int row = 8 * (r / 4) + 4 * h + r % 4;
            const bool seen = kMode == kTree ? (set >> row & 1u) != 0 : row < live;
            s[r] = seen ? s[r] : 0.0f;
          }
        }
      }
      add_values<0>(run, v, s);
      add_values<1>(run, v, s);
      if (next < stop) load_values(v, a, next_base, head, stop - 1 - next, lane);
    }
  };
  walk(std::false_type{});
  if constexpr (!kInt8) {
    // A value that is not finite leaves NaN in every sum, of queries that do not attend its row too: then once more, such
    // values apart.  (Looked for in every block, they would take the registers of the rows under way.)
    float none = 0.0f * run.l;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) none = __builtin_fmaf(run.o[u][r], 0.0f, none);
    if (__ballot(none != none) != 0) {
      start(run);
      if (first < stop) {
        load_keys(k, a, block_at(first), head, stop - 1 - first, lane);
        load_values(v, a, block_at(first), head, stop - 1 - first, lane);
      }
      walk(std::true_type{});
    }
  }
  const float mine = run.l + other32(run.l);
  if (h == 0) {
    peak[wave][lane] = run.m;
    total[wave][lane] = mine;
  }
  __syncthreads();
  // the waves' sums at one maximum (a wave without rows has a sum of 0; NaN stays NaN)
  float m = peak[0][lane & 31];
#pragma unroll
  for (int j = 1; j < kWaves; ++j) m = fmaxf(m, peak[j][lane & 31]);
  const auto weight = [&](float mj) { return mj == -kInf ? (m == -kInf ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(mj - m); };
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < kWaves; ++j) {
    const float lj = total[j][lane & 31];
    sum += lj == 0.0f || lj != lj ? lj : lj * weight(peak[j][lane & 31]);
  }
  const bool whole = w.whole;
  float f = weight(run.m);
  if (whole) f = sum == 0.0f ? 0.0f : sum != sum ? sum : f / sum;
  // query l % 32, a row of 128 floats whose 16-byte pieces are rotated by the query
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    f32x4 y;
#pragma unroll
    for (int u = 0; u < 4; ++u) y[u] = run.o[u][r] * f;
    *(f32x4*)(sums[wave] + (lane & 31) * kD + 4 * ((8 * (r / 4) + 4 * h + r % 4 + lane) & 31)) = y;
  }
  const int64_t stride = (int64_t)a.tokens * a.heads;
  if (!whole && wave == 0 && h == 0 && w.t0 + lane <= w.t_last) {
    float* to = p.tops + 2 * (w.split * stride + (int64_t)(w.t0 + lane) * a.heads + head);
    stg(to, m);
    stg(to + 1, sum);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kQueries * 32 / kThreads; ++j) {
    const int i = j * kThreads + (int)threadIdx.x, query = i / 32, piece = i % 32;
    if (w.t0 + query > w.t_last) continue;
    const int at = query * kD + 4 * ((piece + query) & 31);
    f32x4 y = *(const f32x4*)(sums[0] + at);
#pragma unroll
    for (int u = 1; u < kWaves; ++u) y += *(const f32x4*)(sums[u] + at);
    const int64_t th = (int64_t)(w.t0 + query) * a.heads + head;
    *(UOCR_GLOBAL f32x4*)((whole ? a.out + th * kD : p.part + (w.split * stride + th) * kD) + 4 * piece) = y;
  }
}

// ------------------------------------------------------------------ many tokens a request, over an int8 pool
//
// 256 queries of a head, 32 a wave.  Bound by the matrix instruction: a block of 32 rows is 48 of them a wave, beside some
// 200 other instructions for the scores, and with one row's conversion shared by 8 waves those fit under them (two waves a
// SIMD, the one's products under the other's exponentials): 2048 queries over 14001 rows 430 to 470 us as the card's clock
// goes, 1.0 to 1.1 PFLOP/s of bf16 products beside 1.24 of a large matrix product.  64 rows are in LDS as operands, the next
// 64 on their way:
//   keys    [block 2][step 8][slot 64][8], slot (32 half + row) ^ step: the columns 16 step + 8 half on.  (The exchange
//           spreads a row's steps, which 8 lanes write at once, over the banks.)
//   values  [block 2][step 2][u 4][lane 64][8]: as value_row has them, column 4 (lane % 32) + u.
constexpr int kTileWaves = 8, kTileThreads = kTileWaves * kWave, kTileLog2 = 8;
constexpr int kTileRows = 2 * kBlock;
constexpr int kTileHalves = kTileRows * kD;  // numbers of a tile's keys, or values

struct TileRaw {  // a thread's part of 64 rows: 16 bytes of a key, 4 of 4 values, and a scale
  u32x4 k;
  uint32_t v[4];
  float scale;
};

__global__ void __launch_bounds__(kTileThreads, 2) k_pool_tiles(Attend p) {
  const PoolArgs& a = p.a;
  __shared__ __align__(16) uint16_t keys[2][kTileHalves], values[2][kTileHalves];
  __shared__ __align__(16) uint16_t q_lo[kTileWaves][kQTerm];
  __shared__ __align__(16) float scales[2][2][kTileRows];
  const int tid = (int)threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid / kWave), h = lane >> 5;
  Piece w;
  if (!find_piece<kCausal, kTileLog2>(a, p.cuts, p.most_rows, w)) return;
  const int stop = w.stop, head = w.head;
  const uint32_t* lookup = a.lookup + (int64_t)w.n * a.lookup_cols;
  const auto slots_at = [&](int row) {  // of 32 rows, which lie in one page
    return a.pool + (int64_t)min(ldc(lookup + row / a.P), (uint32_t)(a.pages - 1)) * a.page_bytes + a.layer_bytes +
           (int64_t)(row % a.P) * a.slot_bytes;
  };
  // ---- a tile's rows: memory to registers, registers to LDS
  const int key = tid / 8, chunk = tid % 8;                                // the thread's key and columns 16 chunk on
  const int v_block = wave / 4, v_first = 16 * (wave / 2 % 2) + 4 * (wave % 2) + 8 * h;  // its values' rows, v_first on
  const auto load = [&](TileRaw& r, int row0) {
    const int last = a.max_rows - kBlock;  // (rows past the table's are asked for nowhere)
    const char* lower = slots_at(min(row0, last));
    const char* upper = slots_at(min(row0 + kBlock, last));
    const char* mine = key < kBlock ? lower : upper;
    r.k = *(const UOCR_GLOBAL u32x4*)(mine + (uint32_t)((key % kBlock) * a.slot_bytes + head * kD + 16 * chunk));
    const char* from = (v_block == 0 ? lower : upper) + a.kv_bytes;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r.v[i] = *(const UOCR_GLOBAL uint32_t*)(from + (uint32_t)((v_first + i) * a.slot_bytes + head * kD + 4 * (lane & 31)));
    if (wave < 2) {  // the first wave the keys' scales, the second the values'
      const char* at = (lane < kBlock ? lower : upper) + (wave == 0 ? 0 : a.kv_bytes);
      r.scale = *(const UOCR_GLOBAL float*)(at + (uint32_t)((lane & 31) * a.slot_bytes + a.heads * kD + 4 * head));
    }
  };
  const float c = a.scale * 1.44269504f;
  const auto convert = [&](const TileRaw& r, int buf) {
    u32x4 lo, hi;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      lo[2 * e] = bytes_bf16<0, 1>(r.k[e], r.k[e]);
      lo[2 * e + 1] = bytes_bf16<2, 3>(r.k[e], r.k[e]);
      hi[2 * e] = bytes_bf16<0, 1>(r.k[2 + e], r.k[2 + e]);
      hi[2 * e + 1] = bytes_bf16<2, 3>(r.k[2 + e], r.k[2 + e]);
    }
    uint16_t* kt = keys[buf] + ((key / kBlock) * 8 + chunk) * kFrag;
    *(u32x4*)(kt + ((key % kBlock) ^ chunk) * 8) = lo;
    *(u32x4*)(kt + ((32 + key % kBlock) ^ chunk) * 8) = hi;
    uint16_t* vt = values[buf] + wave / 2 * 4 * kFrag + (32 * (wave % 2) + (lane & 31)) * 8 + 4 * h;
    const auto column = [&](auto u) {
      constexpr int U = decltype(u)::value;
      *(u32x2*)(vt + U * kFrag) = u32x2{bytes_bf16<U, U>(r.v[0], r.v[1]), bytes_bf16<U, U>(r.v[2], r.v[3])};
    };
    column(std::integral_constant<int, 0>{});
    column(std::integral_constant<int, 1>{});
    column(std::integral_constant<int, 2>{});
    column(std::integral_constant<int, 3>{});
    if (wave < 2) scales[buf][wave][lane] = wave == 0 ? r.scale * c : r.scale;
  };
  TileRaw raw;
  load(raw, w.begin);
  // ---- the wave's queries: columns 16 t + 8 h on of step t; the last terms in LDS
  const int t0 = w.t0 + 32 * wave, my_t = min(t0 + (lane & 31), w.t_last);
  const bool idle = t0 > w.t_last;  // a wave without queries converts
  u32x4 q_hi[8], q_mid[8];
  {
    const float* row = a.q + (int64_t)my_t * a.in_stride + (int64_t)head * kD + 8 * h;
    const float *ct = nullptr, *st = nullptr;
    if (a.rope.positions != nullptr) {
      const int64_t at = (int64_t)min(max(ldg(a.rope.positions + my_t), 0), a.rope.table_rows - 1) * kD + 8 * h;
      ct = a.rope.cos_t + at;
      st = a.rope.sin_t + at;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {  // with step t + 4, 64 columns on
      f32x4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = *(const UOCR_GLOBAL f32x4*)(row + 16 * t + 4 * (i % 2) + 64 * (i / 2));
      if (ct != nullptr)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int at = 16 * t + 4 * i;
          rotate4(x[i], x[i + 2], *(const UOCR_GLOBAL f32x4*)(ct + at), *(const UOCR_GLOBAL f32x4*)(ct + at + 64),
                  *(const UOCR_GLOBAL f32x4*)(st + at), *(const UOCR_GLOBAL f32x4*)(st + at + 64));
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        u32x4 lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t mid, last;
          q_hi[t + 4 * i][e] = split3(x[2 * i + e / 2][2 * (e % 2)], x[2 * i + e / 2][2 * (e % 2) + 1], mid, last);
          q_mid[t + 4 * i][e] = mid;
          lo[e] = last;
        }
        *(u32x4*)(q_lo[wave] + (t + 4 * i) * kFrag + lane * 8) = lo;
      }
    }
  }
  const int most = idle ? 0 : min(w.cached + (min(t0 + 31, w.t_last) - w.first) + 1, stop);  // rows that the wave attends
  const int all = min(w.cached + (t0 - w.first) + 1, stop);                                 // that all of its queries do
  const int limit = min(w.cached + (my_t - w.first) + 1, stop);
  Running run;
  start(run);
  convert(raw, 0);
  if (w.begin + kTileRows < stop) load(raw, w.begin + kTileRows);
  lds_barrier();
  const auto attend = [&](int key0, int buf, int block) {
    const uint16_t* kt = keys[buf] + block * 8 * kFrag;
    f32x16 s = {};
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const bf16x8 k = *(const bf16x8*)(kt + t * kFrag + (lane ^ t) * 8);
      s = mfma(k, *(const bf16x8*)(q_lo[wave] + t * kFrag + lane * 8), s);
      s = mfma(k, bf(q_mid[t]), s);
      s = mfma(k, bf(q_hi[t]), s);
    }
    f32x4 vs[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 ks = *(const f32x4*)&scales[buf][0][32 * block + 8 * g + 4 * h];
      vs[g] = *(const f32x4*)&scales[buf][1][32 * block + 8 * g + 4 * h];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[4 * g + e] *= ks[e];
    }
    const bool masked = key0 + kBlock > all;
    if (masked) {
      asm volatile("");  // a branch: as selects the masks would be a quarter of a block's instructions
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 8 * (r / 4) + 4 * h + r % 4 < limit - key0 ? s[r] : -kInf;
    }
    weigh(run, s);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] *= vs[r / 4][r % 4];
    if (masked) {  // the scales of rows that are not attended may be anything
      asm volatile("");
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 8 * (r / 4) + 4 * h + r % 4 < limit - key0 ? s[r] : 0.0f;
    }
    const uint16_t* vt = values[buf] + block * 8 * kFrag + lane * 8;
    const auto step = [&](auto t) {
      constexpr int T = decltype(t)::value;
      u32x4 hi, mid, lo;
      split_weights<T>(s, hi, mid, lo);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bf16x8 v = *(const bf16x8*)(vt + (4 * T + u) * kFrag);
        run.o[u] = mfma(v, bf(lo), run.o[u]);
        run.o[u] = mfma(v, bf(mid), run.o[u]);
        run.o[u] = mfma(v, bf(hi), run.o[u]);
      }
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
  };
  int buf = 0;
#pragma unroll 1
  for (int key0 = w.begin; key0 < stop; key0 += kTileRows, buf ^= 1) {
    if (key0 < most) attend(key0, buf, 0);
    if (key0 + kTileRows < stop) {
      convert(raw, buf ^ 1);
      if (key0 + 2 * kTileRows < stop) load(raw, key0 + 2 * kTileRows);
    }
    if (key0 + kBlock < most) attend(key0 + kBlock, buf, 1);
    lds_barrier();
  }
  if (idle || t0 + (lane & 31) > w.t_last) return;
  const float sum = run.l + other32(run.l);
  const bool whole = w.whole;
  const float f = !whole ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
  const int64_t th = (int64_t)my_t * a.heads + head, part = w.split * (int64_t)a.tokens * a.heads + th;
  float* to = (whole ? a.out + th * kD : p.part + part * kD) + 16 * h;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    f32x4 y;
#pragma unroll
    for (int u = 0; u < 4; ++u) y[u] = run.o[u][r] * f;
    *(UOCR_GLOBAL f32x4*)(to + 32 * (r / 4) + 4 * (r % 4)) = y;
  }
  if (!whole && h == 0) {
    stg(p.tops + 2 * part, run.m);
    stg(p.tops + 2 * part + 1, sum);
  }
}

// ------------------------------------------------------------------ one token a request, over an int8 pool
//
// A single query leaves 31 of 32 columns of the matrix instruction empty, and one head's rows are its alone: the products
// are fp32 multiply-adds on converted bytes, two instructions a byte, which at 64 lanes a clock is 32 bytes a clock of a
// CU, three times what memory brings.  8 lanes have a row, 16 columns each, of the keys as of the values, so a row's weight
// is where its values are: every group of 8 lanes has a softmax of its own, and nothing crosses lanes in the loop but a
// score's three sums.  Bound by the trips to memory where rows are few (one request of 640 rows: 11 us, where the fp32
// pool's kernel, which cuts at 128 rows, takes 7).  Where they are many (24 of 1445 to 4000: 45 us, 3.8 TB/s) nothing is near
// its limit all the time: 240 workgroups of unlike lengths, one a CU, are there for 69 % of it, the L1s wait for misses for
// 46 %, the vector units are busy for 24 %.  A row's scale is 4 bytes of a line of its own, a third of the requests to L2: with
// one head a wave the lines cost a fifth of the time, so two heads share them where workgroups are many.
constexpr int kOneWaves = 12;  // as many as have their registers on a CU
constexpr int kOneParts = 16;  // columns of a lane

// Rows that request n's token attends.
__device__ __forceinline__ int one_rows(const PoolArgs& a, int n) {
  return (int)min((int64_t)min(ldc(a.cache_lengths + n), (uint32_t)(a.max_rows - 1)) + 1, (int64_t)a.attend_max);
}

// The sum over the 8 lanes of a group; the largest.
template <typename F>
__device__ __forceinline__ uint32_t of_group(uint32_t v, F f) {
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, false));   // lane ^ 1
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, false));   // lane ^ 2
  return f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false));  // 7 - lane
}
__device__ __forceinline__ float group_sum(float v) {
  return __uint_as_float(of_group(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  return of_group(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
// Over the groups of a head, 8, 16 and, where the wave has one head, 32 lanes apart.
template <int kHeads, typename F>
__device__ __forceinline__ float of_head(float v, F f) {
  v = f(v, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x128, 0xf, 0xf, false)));
  v = f(v, __uint_as_float(other<16>(__float_as_uint(v))));
  return kHeads == 1 ? f(v, other32(v)) : v;
}

// What a lane reads of a wave's heads: 64 / kHeads lanes have a head, whose group g has rows (8 / kHeads) i + g of a block,
// columns 16 part on.
template <int kHeads>
struct OneLane {
  static constexpr int kRows = 32 / kHeads;  // of a block
  int part, group, sub, head;
  __device__ __forceinline__ int row(int i) const { return 8 / kHeads * i + group; }
};
template <int kHeads>
struct OneRows {
  u32x4 k[4], v[4];
  float ks, vs;  // of row sub % kRows
};
template <int kHeads>
__device__ __forceinline__ void one_load(u32x4 (&x)[4], float& scale, const PoolArgs& a, const char* from,
                                         const OneLane<kHeads>& l) {
  const uint32_t at = (uint32_t)(l.group * a.slot_bytes + l.head * kD + 16 * l.part);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = *(const UOCR_GLOBAL u32x4*)(from + 8 / kHeads * i * a.slot_bytes + at);
  scale = *(const UOCR_GLOBAL float*)(from + (uint32_t)(l.sub % OneLane<kHeads>::kRows * a.slot_bytes + a.heads * kD + 4 * l.head));
}

// A lane's 16 columns of a row, rotated where `ct` is not null (its tables' row): the pair of column d is d +- 64.
__device__ __forceinline__ void load_columns(float (&x)[kOneParts], const float* row, const float* ct, const float* st, int part) {
#pragma clang fp contract(off)
#pragma unroll
  for (int i = 0; i < kOneParts / 4; ++i) {
    const f32x4 y = *(const UOCR_GLOBAL f32x4*)(row + 16 * part + 4 * i);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * i + e] = y[e];
  }
  if (ct == nullptr) return;
#pragma unroll
  for (int i = 0; i < kOneParts / 4; ++i) {
    const f32x4 y = *(const UOCR_GLOBAL f32x4*)(row + 16 * (part ^ 4) + 4 * i);
    const f32x4 c = *(const UOCR_GLOBAL f32x4*)(ct + 16 * part + 4 * i), s = *(const UOCR_GLOBAL f32x4*)(st + 16 * part + 4 * i);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * i + e] = x[4 * i + e] * c[e] + (part < 4 ? -y[e] : y[e]) * s[e];
  }
}
// A group's row as its lanes' bytes, and its scale.
__device__ __forceinline__ u32x4 quantize_columns(const float (&x)[kOneParts], float& scale) {
  uint32_t most = 0;
#pragma unroll
  for (int e = 0; e < kOneParts; ++e) most = max(most, abs_bits(x[e]));
  scale = row_scale(group_max(most));
  u32x4 q;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    q[i] = to_int8x4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3], scale);
  return q;
}

// What is computed from x after this is computed after this: conversions ahead of their use would take the registers of the
// rows under way.
__device__ __forceinline__ uint32_t held_back(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}
// A group's score: the lane's 16 products in four sums, then the lanes'.
__device__ __forceinline__ float dot16(const float (&q)[kOneParts], u32x4 x) {
  float s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s[i] = q[4 * i] * i8_to_f32<0>((int)x[i]);
    s[i] = __builtin_fmaf(q[4 * i + 1], i8_to_f32<1>((int)x[i]), s[i]);
    s[i] = __builtin_fmaf(q[4 * i + 2], i8_to_f32<2>((int)x[i]), s[i]);
    s[i] = __builtin_fmaf(q[4 * i + 3], i8_to_f32<3>((int)x[i]), s[i]);
  }
  return group_sum((s[0] + s[1]) + (s[2] + s[3]));
}
__device__ __forceinline__ void add16(float (&o)[kOneParts], float w, u32x4 x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int y = (int)held_back(x[i]);
    o[4 * i] = __builtin_fmaf(w, i8_to_f32<0>(y), o[4 * i]);
    o[4 * i + 1] = __builtin_fmaf(w, i8_to_f32<1>(y), o[4 * i + 1]);
    o[4 * i + 2] = __builtin_fmaf(w, i8_to_f32<2>(y), o[4 * i + 2]);
    o[4 * i + 3] = __builtin_fmaf(w, i8_to_f32<3>(y), o[4 * i + 3]);
  }
}
// The weight of a sum at maximum mj beside one at m; of sums without rows (0) and NaN.
__device__ __forceinline__ float weight_at(float mj, float l, float m) {
  if (l == 0.0f || l != l) return l;
  return mj == -kInf ? (m == -kInf ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(mj - m);
}

template <int kHeads>
__global__ void __launch_bounds__(kOneWaves * kWave) k_pool_one(Attend p) {
  const PoolArgs& a = p.a;
  __shared__ __align__(16) float sums[kOneWaves][kHeads][kD];
  __shared__ float peak[kOneWaves][kHeads], total[kOneWaves][kHeads];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  // Every request has a piece for each split and its heads, whose place follows from the workgroup's number: what does not
  // depend on one another is asked for together.
  const int turn = (int)(blockIdx.x / 8), round = p.cuts.by_heads(turn), cell = 8 * round + (int)(blockIdx.x % 8);
  const int head0 = kHeads * (turn - round * ((a.heads + kHeads - 1) / kHeads));
  const int n = cell / p.cuts.splits, split = cell - n * p.cuts.splits;
  if (n >= a.requests) return;
  OneLane<kHeads> me;
  me.sub = lane_id() % (kWave / kHeads);
  me.part = me.sub % 8;
  me.group = me.sub / 8;
  const int side = lane_id() / (kWave / kHeads);
  me.head = min(head0 + side, a.heads - 1);
  constexpr int kRows = OneLane<kHeads>::kRows, kStep = (kOneWaves - 1) * kRows;  // the last wave has the new row
  const int begin = split * p.cuts.split_rows, first = begin + kRows * wave;
  const uint32_t* lookup = a.lookup + (int64_t)n * a.lookup_cols;
  const auto block_at = [&](int row) {  // (rows past the table's are asked for nowhere)
    const int at = min(row, a.max_rows - kRows);
    return a.pool + (int64_t)min(ldc(lookup + at / a.P), (uint32_t)(a.pages - 1)) * a.page_bytes + a.layer_bytes +
           (int64_t)(at % a.P) * a.slot_bytes;
  };
  const char* first_at = block_at(first);
  const int all_rows = one_rows(a, n);
  const uint32_t write = ldc(a.write_index + n);
  const int64_t src = (int64_t)n * a.in_stride + (int64_t)me.head * kD;
  const float *ct = nullptr, *st = nullptr;
  if (a.rope.positions != nullptr) {
    const int64_t pos = (int64_t)min(max(ldc(a.rope.positions + n), 0), a.rope.table_rows - 1) * kD;
    ct = a.rope.cos_t + pos;
    st = a.rope.sin_t + pos;
  }
  const int stop = min(begin + p.cuts.split_rows, all_rows);
  if (begin >= stop) return;
  const float c = a.scale * 1.44269504f;
  const int new_row = write < (uint32_t)all_rows ? (int)write : -1;
  float q[kOneParts], m = -kInf, l = 0.0f, o[kOneParts] = {};
  if (wave < kOneWaves - 1) {
    // A block's rows lie in one page, so that all of them can be read, whether attended or not.
    OneRows<kHeads> r;
    if (first < stop) {
      one_load(r.k, r.ks, a, first_at, me);
      one_load(r.v, r.vs, a, first_at + a.kv_bytes, me);
    }
    load_columns(q, a.q + src, ct, st, me.part);
    // the next rows are asked for as these are used up
#pragma unroll 1
    for (int key0 = first; key0 < stop; key0 += kStep) {
      const int next = key0 + kStep;
      const float ks = r.ks * c;
      float s[4], vs[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int from = side * (kWave / kHeads) + me.row(i);
        s[i] = dot16(q, r.k[i]) * __shfl(ks, from, kWave);
        vs[i] = __shfl(r.vs, from, kWave);
        __builtin_amdgcn_sched_barrier(0);
      }
      const char* next_at = next < stop ? block_at(next) : nullptr;
      __builtin_amdgcn_sched_barrier(0);
      if (next < stop) one_load(r.k, r.ks, a, next_at, me);
      __builtin_amdgcn_sched_barrier(0);
      if (key0 + kRows > stop || (uint32_t)(new_row - key0) < (uint32_t)kRows)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = key0 + me.row(i);
          if (row >= stop || row == new_row) {  // what is there may be anything
            s[i] = -kInf;
            vs[i] = 0.0f;
          }
        }
      const float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
      const bool up = mx > m + kSlack;
      if (__ballot(up) != 0) {
        const float alpha = up ? __builtin_amdgcn_exp2f(m - mx) : 1.0f;
        m = up ? mx : m;
        l *= alpha;
#pragma unroll
        for (int e = 0; e < kOneParts; ++e) o[e] *= alpha;
      }
      const float off = m == -kInf ? 0.0f : m;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = __builtin_amdgcn_exp2f(s[i] - off);
        l += e;
        add16(o, e * vs[i], r.v[i]);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (next < stop) one_load(r.v, r.vs, a, next_at + a.kv_bytes, me);
      __builtin_amdgcn_sched_barrier(0);
    }
  } else if (write < (uint32_t)a.max_rows && (new_row < 0 ? split == 0 : new_row >= begin && new_row < stop)) {
    // The new row, while the others wait for memory: stored, and attended as it was rounded.  Every group of a head has all
    // of it; the first's weight counts.
    float x[kOneParts], ks, vs;
    load_columns(x, a.k_new + src, ct, st, me.part);
    const u32x4 k = quantize_columns(x, ks);
    load_columns(x, a.v_new + src, nullptr, nullptr, me.part);
    const u32x4 v = quantize_columns(x, vs);
    if (head0 + side < a.heads) {
      char* slot = slot_of(a, n, (int)write);
      if (me.group == 0) *(UOCR_GLOBAL u32x4*)(slot + me.head * kD + 16 * me.part) = k;
      if (me.group == 1) *(UOCR_GLOBAL u32x4*)(slot + a.kv_bytes + me.head * kD + 16 * me.part) = v;
      if (me.sub == 0) {
        stg((float*)(slot + a.heads * kD) + me.head, ks);
        stg((float*)(slot + a.kv_bytes + a.heads * kD) + me.head, vs);
      }
    }
    if (new_row >= 0 && me.group == 0) {
      load_columns(q, a.q + src, ct, st, me.part);
      const float s = dot16(q, k) * (ks * c);
      m = s == s ? s : -kInf;
      l = s == s ? 1.0f : s;
      add16(o, l * vs, v);
    }
  }
  // the groups' sums at one maximum, then the waves'
  const auto most = [](float x, float y) { return fmaxf(x, y); };
  const auto plus = [](float x, float y) { return x + y; };
  const float top = of_head<kHeads>(m, most), f = weight_at(m, l, top);
  l = of_head<kHeads>(l * f, plus);
#pragma unroll
  for (int e = 0; e < kOneParts; ++e) o[e] = of_head<kHeads>(o[e] * f, plus);
  if (me.group == 0) {
#pragma unroll
    for (int e = 0; e < kOneParts; e += 4)
      *(f32x4*)&sums[wave][side][16 * me.part + e] = f32x4{o[e], o[e + 1], o[e + 2], o[e + 3]};
  }
  if (me.sub == 0) {
    peak[wave][side] = top;
    total[wave][side] = l;
  }
  __syncthreads();
  const int at = (int)threadIdx.x / kD, d = (int)threadIdx.x % kD;
  if (at >= kHeads || head0 + at >= a.heads) return;
  float all = -kInf;
#pragma unroll
  for (int j = 0; j < kOneWaves; ++j) all = fmaxf(all, peak[j][at]);
  float sum = 0.0f, y = 0.0f;
#pragma unroll
  for (int j = 0; j < kOneWaves; ++j) {
    const float fj = weight_at(peak[j][at], total[j][at], all);
    sum = __builtin_fmaf(total[j][at], fj, sum);
    y = __builtin_fmaf(sums[j][at][d], fj, y);
  }
  const int64_t th = (int64_t)n * a.heads + head0 + at;
  if (all_rows <= p.cuts.split_rows) {
    stg(a.out + th * kD + d, y / sum);
  } else {
    const int64_t stride = (int64_t)a.tokens * a.heads;
    stg(p.part + (split * stride + th) * kD + d, y);
    if (d == 0) {
      stg(p.tops + 2 * (split * stride + th), all);
      stg(p.tops + 2 * (split * stride + th) + 1, sum);
    }
  }
}

// Joins the splits of a token's rows: half a wave a (token, head), four columns a lane.  Of many splits (`ways`) the four waves
// of a workgroup take every fourth: one wave would wait for the memory every few of them (8 tokens over 14000 rows, 37 splits:
// 21 us, 7 by four waves).
constexpr int kJoinAtOnce = 4;
template <Mode kMode, int kQueriesLog2>
__global__ void __launch_bounds__(256) k_pool_join(Attend p, bool ways) {
  __shared__ __align__(16) float sums[4][4 * kWave];
  const PoolArgs& a = p.a;
  const int groups = (a.heads + 1) / 2, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  const int64_t item = ways ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  const int64_t t = item / groups;
  if (t >= a.tokens) return;
  int splits;  // of its tile
  if constexpr (kMode == kOne) {
    splits = p.cuts.by_split(one_rows(a, (int)t) - 1) + 1;
  } else {
    Chunk c;
    if (!chunk_of(a, (int)t, c)) return;
    const int i = (int)t - c.first, length = c.end - c.first;
    const int t_last = min(((i >> kQueriesLog2) + 1) << kQueriesLog2, length) - 1;
    const int rows = rows_of_split(tile_rows<kMode>(a, c.cached, length, length - 1), ldg(p.most_rows));
    splits = (tile_rows<kMode>(a, c.cached, length, t_last) - 1) / rows + 1;
  }
  if (splits == 1) return;  // written by its tile
  const int lane = lane_id(), piece = lane & 31, head = (int)(item - t * groups) * 2 + lane / 32;
  const int64_t stride = (int64_t)a.tokens * a.heads, th = t * a.heads + min(head, a.heads - 1);
  float m = -kInf, l = 0.0f;
  for (int s = piece; s < splits; s += 32) m = fmaxf(m, ldg(p.tops + 2 * (s * stride + th)));
#pragma unroll
  for (int off = 1; off < 32; off *= 2) m = fmaxf(m, __shfl_xor(m, off, kWave));
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int base = 0; base < splits; base += 32) {
    float f = 0.0f;  // of split base + piece
    if (base + piece < splits) {
      const float* top = p.tops + 2 * ((base + piece) * stride + th);
      const float ms = ldg(top), ls = ldg(top + 1);
      f = ls == 0.0f ? 0.0f : ms == -kInf ? 1.0f : __builtin_amdgcn_exp2f(ms - m);
      l = __builtin_fmaf(f, ls, l);
    }
    const int upto = min(32, splits - base), step = ways ? 4 : 1;
    for (int s0 = ways ? wave : 0; s0 < upto; s0 += kJoinAtOnce * step) {
      f32x4 y[kJoinAtOnce];
#pragma unroll
      for (int i = 0; i < kJoinAtOnce; ++i)
        y[i] = *(const UOCR_GLOBAL f32x4*)(p.part + ((base + min(s0 + i * step, upto - 1)) * stride + th) * kD + 4 * piece);
#pragma unroll
      for (int i = 0; i < kJoinAtOnce; ++i) {
        if (s0 + i * step >= upto) break;
        const float fs = __shfl(f, s0 + i * step + (lane & 32), kWave);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(fs, y[i][e], o[e]);
      }
    }
  }
#pragma unroll
  for (int off = 1; off < 32; off *= 2) l += __shfl_xor(l, off, kWave);
  if (ways) {
    *(f32x4*)&sums[wave][4 * lane] = o;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < 4; ++w) o += *(const f32x4*)&sums[w][4 * lane];
  }
  if (head < a.heads) *(UOCR_GLOBAL f32x4*)(a.out + th * kD + 4 * piece) = l == 0.0f ? f32x4{} : o / l;
}

}  // namespace

// How a call's rows are cut.
namespace {
constexpr int kCus = 256;
// Rows of a decode's split at least: two rounds of a wave's 32 rows, four of 16 (one request over 4000 rows 14.5 us in splits
// of 704, 18.4 of 1408, 26 of 2816, on the device with the join; but 24 over 1000 19 in two and 16 whole).  Equal shares of
// all requests' rows instead, whose workgroups go from one request to the next: no faster (24 over 1445 to 4000 46 us both
// ways), as the rows are bound by their loads and not by the longest request.
constexpr int kOneLeast = 704;
PoolCuts cuts_of(int64_t tokens, int64_t requests, int heads, int attend_max, PoolForm form) {
  PoolCuts c{};
  const bool one = form == kPoolDecode;
  // Tiles of 256 queries share a row's conversion, and fill the device where there are many of them or their rows are many
  // (one chunk of 2048 over no rows 76 us against 87, over 14001 450 against 604; 512 over 14000 123 and 138; but 256 over
  // 14000 82 and 79, eight of 512 over none 46 and 37).
  c.tiles = form == kPoolChunk && requests > 0 && tokens / requests >= 256 && tokens * attend_max >= 3 << 20;
  const int queries = c.tiles ? 1 << kTileLog2 : kQueries;
  const int64_t tiles = one || requests <= 64 ? (tokens < requests ? tokens : (tokens - requests) / queries + requests)
                                              : tokens / queries + requests;
  c.slots = (int)tiles;
  c.few = one && requests * heads <= kCus / 2;
  c.groups = one && !c.few ? (heads + 1) / 2 : heads;
  c.split_rows = attend_max;
  if (one) {
    // As many splits as fill the device once, one workgroup a CU; with two heads a wave a few more rounds take less than a join.
    const int64_t fill = kCus / std::max<int64_t>(1, requests * c.groups);
    const int64_t splits = !c.few && attend_max <= 2 * kOneLeast ? 1 : std::max<int64_t>(1, fill);
    c.split_rows = (int)std::max<int64_t>(kOneLeast, ((attend_max + splits - 1) / splits + kOneLeast - 1) / kOneLeast * kOneLeast);
  } else if (attend_max <= 512) {
    // two splits of 256 rows and their join take the time of one of 512, and a launch more
    c.split_rows = 512;
  } else {
    // With up to half as many workgroups as the device holds (two on a CU, one of tiles' 8 waves) the rows are cut for it to
    // be full once, with up to as many twice; of more, the next takes the place of one that ends.  As to the lengths, none may
    // be shorter than the others: splits for all of them to be half as long are what the workspace has to hold.
    const int64_t mean = requests == 0 ? 1 : (tokens / requests + queries - 1) / queries * requests;
    const int64_t work = std::max<int64_t>(1, std::min(tiles, mean)) * heads, fits = c.tiles ? kCus : 2 * kCus;
    const int64_t full = work <= fits / 2 ? fits : work <= fits ? 2 * fits : 0;
    if (full > 0) {
      const int64_t longest = (attend_max + full / work - 1) / (full / work);
      const bool counts = requests > 1 && requests <= 64;
      c.fill = requests <= 64 ? (int)(full / heads) : 0;
      c.split_rows = (int)std::max<int64_t>(2 * kRound, ((counts ? longest / 2 : longest) + kRound - 1) / kRound * kRound);
    }
  }
  // Pieces that are not cut are as long as their requests: stretches of them would leave XCDs without work (64 chunks of 64
  // over 333 to 1000 rows 90 us, 71 round the XCDs; 32 over 1333 to 4000 168 and 120).
  c.round = form == kPoolChunk && requests <= 64 && c.fill == 0;
  c.splits = (int)(((int64_t)attend_max + c.split_rows - 1) / c.split_rows);
  c.by_split = divide_by(c.split_rows);
  c.by_heads = divide_by(c.groups);
  return c;
}

template <bool kInt8, Mode kMode>
hipError_t launch(const PoolAttention& p, const PoolArgs& a, hipStream_t s) {
  const PoolCuts c = cuts_of(p.tokens, p.requests, p.heads, p.attend_max, form_of(kMode));
  const int64_t pairs = p.tokens * p.heads;
  const int64_t pieces = c.fill > 0 ? std::max(c.fill, c.slots) : (int64_t)c.slots * c.splits;
  const int64_t items = (pieces + 7) / 8 * 8 * c.groups;
  const int64_t joins = p.tokens * ((p.heads + 1) / 2);
  // (where a wave counts the pieces, offsets that do not ascend may give each request all of them)
  const int64_t most = (int64_t)c.slots * c.splits * c.groups;
  if (pieces > INT32_MAX / c.groups - 8 || most > INT32_MAX / std::min<int64_t>(p.requests, 64) - 8) return hipErrorInvalidValue;
  const Attend at{a, c, (float*)p.workspace, (float*)p.workspace + (int64_t)c.splits * pairs * kD,
                  (int*)((float*)p.workspace + (int64_t)c.splits * pairs * (kD + 2))};
  const dim3 grid((unsigned)items);
  if constexpr (kMode == kOne) {
    if (c.few)
      UOCR_LAUNCH("pool_one", k_pool_one<1>, grid, dim3(kOneWaves * kWave), 0, s, at);
    else
      UOCR_LAUNCH("pool_one", k_pool_one<2>, grid, dim3(kOneWaves * kWave), 0, s, at);
  } else {
    if (!a.stores) {
      auto store = k_pool_store<kInt8>;
      const int64_t stores = p.tokens * ((p.heads + kStoreHeads - 1) / kStoreHeads);
      UOCR_LAUNCH("pool_store", store, dim3((unsigned)((stores + 3) / 4)), dim3(256), 0, s, a);
    }
    if (kMode == kCausal && c.tiles) {
      UOCR_LAUNCH("pool_tiles", k_pool_tiles, grid, dim3(kTileThreads), 0, s, at);
    } else {
      auto attend = k_pool_attend<kInt8, kMode>;
      UOCR_LAUNCH("pool_attend", attend, grid, dim3(kThreads), 0, s, at);
    }
  }
  if (c.splits > 1) {
    auto join = k_pool_join<kMode, kQueriesLog2>;
    if constexpr (kMode == kCausal)
      if (c.tiles) join = k_pool_join<kMode, kTileLog2>;
    const bool ways = c.splits > 8;
    UOCR_LAUNCH("pool_join", join, dim3((unsigned)(ways ? joins : (joins + 3) / 4)), dim3(256), 0, s, at, ways);
  }
  return hipGetLastError();
}
}  // namespace

size_t pool_workspace_bytes(int64_t tokens, int64_t requests, int heads, int attend_max, PoolForm form) {
  const PoolCuts c = cuts_of(tokens, requests, heads, attend_max, form);
  return c.splits > 1 && tokens > 0 ? (size_t)c.splits * tokens * heads * (kD + 2) * sizeof(float) + sizeof(int) : 0;
}

hipError_t launch_pool_attention(const PoolAttention& p, hipStream_t s) {
  if (p.tokens == 0 || p.requests == 0) return hipSuccess;
  PoolArgs a{};
  a.pool = (char*)p.kv_blocks;
  a.slot_bytes = p.slot_bytes;
  a.kv_bytes = (int64_t)p.layers * p.page_size * p.slot_bytes;
  a.page_bytes = 2 * a.kv_bytes;
  a.layer_bytes = (int64_t)p.layer * p.page_size * p.slot_bytes;
  a.P = p.page_size;
  a.heads = p.heads;
  a.pages = p.pages;
  a.max_rows = p.lookup_cols * p.page_size;
  a.lookup = p.lookup;
  a.lookup_cols = p.lookup_cols;
  a.requests = (int)p.requests;
  a.tokens = (int)p.tokens;
  a.cache_lengths = p.cache_lengths;
  a.offsets = p.chunk_offsets;
  a.write_index = p.write_index;
  a.visible = p.visible;
  a.attend_max = p.attend_max;
  a.in_stride = p.in_stride;
  a.q = p.q;
  a.k_new = p.k_new;
  a.v_new = p.v_new;
  a.out = p.out;
  a.scale = p.scale;
  a.rope = Rope{p.positions, p.cos_table, p.sin_table, p.table_rows};
  // Few new rows are stored by those that read them, which saves a launch; many would take a workgroup longer than that: 16
  // a step (chunks of 8 over none, 16 of them, 8.1 us for 10.5; of 4 over 300 rows, 40, 16.2 for 18.5; but one of 100 over none
  // 18.8 for 11.3).  Not each request's are known here, only all of them and their mean.
  a.stores = p.tokens <= 128 && p.tokens <= 32 * p.requests;  // (tiles have more tokens)
  if (p.write_index != nullptr) return launch<true, kOne>(p, a, s);
  if (p.visible == nullptr) return launch<true, kCausal>(p, a, s);
  return p.int8 ? launch<true, kTree>(p, a, s) : launch<false, kTree>(p, a, s);
}

}  // namespace uocr
