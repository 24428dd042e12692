// What the attention of several new tokens over a page pool shares, whatever the pool holds: which request a token
// belongs to, RoPE, exchanges between lanes.
#pragma once

#include "uocr_device.h"

namespace uocr {

namespace {

constexpr int kD = 128;  // head dim

// A request's chunk: its token rows [first, end) and its cached rows.
struct Chunk {
  int n, first, end, cached;
};
// The last request n with floor(off[n] / 2^log2) + (n if `numbered`) <= key, found by the whole wave: 64 probes at a
// time, whose last round brings the request's metadata along.  Offsets are device data: whatever they hold, the
// request is one of them.
template <typename Args>
__device__ __forceinline__ Chunk find_chunk(const Args& a, int log2, bool numbered, int64_t key) {
  const int lane = lane_id();
  const auto below = [&](int off, int i) { return (int64_t)(off >> log2) + (numbered ? i : 0) <= key; };
  int lo = 0, hi = a.requests;
  while (hi - lo > 64) {
    const int step = (hi - lo + 63) / 64, i = lo + lane * step;
    const bool b = i < hi && below(ldg(a.offsets + min(i, hi - 1)), i);
    lo = min(lo + (max(1, __popcll(__ballot(b))) - 1) * step, hi - 1);
    hi = min(hi, lo + step);
  }
  const int i = min(lo + lane, hi - 1);
  const int off = ldg(a.offsets + i), next = ldg(a.offsets + i + 1);
  const uint32_t cached = min(ldg(a.cache_lengths + i), (uint32_t)a.max_rows);
  const int at = __builtin_amdgcn_readfirstlane(max(1, __popcll(__ballot(lo + lane < hi && below(off, i)))) - 1);
  Chunk c;
  c.n = __builtin_amdgcn_readfirstlane(lo) + at;
  c.first = __builtin_amdgcn_readlane(off, at);
  c.end = min(__builtin_amdgcn_readlane(next, at), a.tokens);
  c.cached = __builtin_amdgcn_readlane((int)cached, at);
  return c;
}
// The chunk that holds token t (wave-uniform); false where none does.
template <typename Args>
__device__ __forceinline__ bool chunk_of(const Args& a, int t, Chunk& c) {
  c = find_chunk(a, 0, false, t);
  return c.first >= 0 && c.first <= t && t < c.end;
}

// RoPE's tables (positions null: q and k come rotated).
struct Rope {
  const int32_t* positions;
  const float* cos_t;
  const float* sin_t;
  int table_rows;
};

// Element d of the rotated row x, and four pairs of such: k_rope's arithmetic.
__device__ __forceinline__ float rotated(const float* x, const float* c, const float* s, int d) {
#pragma clang fp contract(off)
  return d < 64 ? ldg(x + d) * ldg(c + d) + (-ldg(x + d + 64)) * ldg(s + d)
                : ldg(x + d) * ldg(c + d) + ldg(x + d - 64) * ldg(s + d);
}
__device__ __forceinline__ void rotate4(f32x4& lo, f32x4& hi, f32x4 cl, f32x4 ch, f32x4 sl, f32x4 sh) {
#pragma clang fp contract(off)
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float l = lo[e], u = hi[e];
    lo[e] = l * cl[e] + (-u) * sl[e];
    hi[e] = u * ch[e] + l * sh[e];
  }
}

// Reductions in which every lane gets the result: over lanes 16 or 32 apart.
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
// The lane's number as the compiler cannot know it: what is computed from it inside a loop is computed there,
// and takes no register around the loop.
__device__ __forceinline__ int lane_now() {
  int l = lane_id();
  asm volatile("" : "+v"(l));
  return l;
}

}  // namespace

}  // namespace uocr
