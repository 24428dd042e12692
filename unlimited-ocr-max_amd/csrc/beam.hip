// A step of beam search: of every request's beams and their next tokens the best, and the beams' states in their order.
// The reference decodes one beam; what feeds this (logits after the n-gram guard, unlimited_ocr_max/ngram.py:33-53, and
// the guard's history) and what follows (the pages' forks) is this library's.
//
//   key(b, v) = score_b + (logit[b, v] - log sum_v exp logit[b, v])          a live beam
//   key(b, eos) = score_b, no other token                                    an ended one
//   rank = key / length^alpha, the length with the new token                 (given lengths; else rank = key)
//
// The K best of a request's K beams by rank, ties to the lower beam, of a beam to the larger logit, then to the lower token
// (beside a score of some size 64 bits do not tell the keys of a beam's tokens apart, and their logits do).  Keys and ranks
// are in 64 bits, the exponentials and their sum too (a sum's logarithm is off by 2e-12 at most): which of two near candidates
// wins decides what a request says.  A candidate whose rank is not finite (a token at -inf, a beam whose score or sum is not
// finite) comes after all others, as -inf; of a beam without a finite sum it is the first tokens that do.
#include "uocr_device.h"
#include "uocr_kernels.h"

namespace uocr {

namespace {

typedef float f32x4_at_float __attribute__((ext_vector_type(4), aligned(4)));

constexpr float kInf = __builtin_huge_valf();
constexpr int kList = 1024;  // candidates that are ranked against one another in LDS

// A float's bits in the order of the floats, which has -0.0 and 0.0 as one.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (int)b < 0 ? ~b : b | 0x80000000u;
}
// The float whose bits come there; of what lies below all of them, -inf.
__device__ __forceinline__ float of_ordered(uint32_t u) {
  return u <= 0x007fffffu ? -kInf : __uint_as_float((int)u < 0 ? u ^ 0x80000000u : ~u);
}
// A border that at least `most` lanes of a wave reach with `mine`, and few more: the most-th largest, its last 12 bits cut.
__device__ __forceinline__ uint32_t border_of(uint32_t mine, int most) {
  uint32_t t = 0;
#pragma unroll
  for (int bit = 31; bit >= 12; --bit) {
    const uint32_t up = t | 1u << bit;
    if (__popcll(__ballot(mine >= up)) >= most) t = up;
  }
  return t;
}

// Of the candidates that the threads of a workgroup hold, the first `most` (at most 32) by value (descending) and id
// (ascending).  `mine` is the thread's largest value (-inf: it has none); each(least, f) calls f(value, id) for its candidates
// that are no smaller than the float `least`, put(rank, value, id) takes a chosen one; returns their number.
//
// At least `most` candidates are no smaller than the most-th largest of a wave's lanes' largest ones (as floats, whose
// rounding keeps the order), and few are as large: those of the highest such border are listed, and ranked by counting.
// Where equal values fill the list, each next one is looked for among all.
template <typename V, typename Id, int kThreads>
struct Best {
  V value[kList];
  Id id[kList];
  uint32_t border[kThreads / kWave];
  int listed;
};
template <typename V, typename Id, int kThreads, typename Each, typename Put>
__device__ __forceinline__ int choose(Best<V, Id, kThreads>& b, int most, V mine, Each each, Put put) {
  const int tid = (int)threadIdx.x;
  static_assert(kThreads <= kList, "a thread has a place in the list");
  const V none = -(V)__builtin_huge_val();
  const uint32_t own_border = border_of(ordered((float)mine), most);
  if (lane_id() == 0) b.border[tid / kWave] = own_border;
  if (tid == 0) b.listed = 0;
  __syncthreads();
  uint32_t border = 0;
#pragma unroll
  for (int i = 0; i < kThreads / kWave; ++i) border = max(border, b.border[i]);
  const float least = of_ordered(border);
  if ((float)mine >= least)
    each(least, [&](V v, Id id) {
      const int at = atomicAdd(&b.listed, 1);
      if (at < kList) {
        b.value[at] = v;
        b.id[at] = id;
      }
    });
  __syncthreads();
  const int n = b.listed;
  if (n <= kList) {
    for (int i = tid; i < n; i += kThreads) {
      const V v = b.value[i];
      const Id id = b.id[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) rank += b.value[j] > v || (b.value[j] == v && b.id[j] < id);
      if (rank < most) put(rank, v, id);
    }
    return min(n, most);
  }
  V last = -none;  // the one chosen before: the next ones come after it
  Id last_id = -1;
  for (int k = 0; k < most; ++k) {
    V v = none;
    Id at = -1;
    each(-kInf, [&](V x, Id id) {
      const bool after = k == 0 || x < last || (x == last && id > last_id);
      if (after && (at < 0 || x > v || (x == v && id < at))) {
        v = x;
        at = id;
      }
    });
    __syncthreads();
    b.value[tid] = v;
    b.id[tid] = at;
    __syncthreads();
    for (int i = 0; i < kThreads; ++i) {
      const V x = b.value[i];
      const Id id = b.id[i];
      if (id >= 0 && (at < 0 || x > v || (x == v && id < at))) {
        v = x;
        at = id;
      }
    }
    if (at < 0) return k;
    if (tid == 0) put(k, v, at);
    last = v;
    last_id = at;
  }
  return most;
}

constexpr int kRowThreads = 256, kJoinThreads = 512;

struct BeamWork {  // of each row's pieces: the sum and the largest logit, the best tokens
  int pieces;
  Divide by_beam;  // candidates of a beam
  double* sums;
  float* tops;
  float* values;
  int* ids;
};

// max(a, b, c), NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_maximum3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// The sum of e^x of four -700 <= x <= 0, each off by 1.1e-12 of itself: 2^(x log2 e), whose whole part is what stays of it
// beside 1.5 2^52, in the sum's lower word, and the rest, a half at most, a polynomial (2^f by its values at nine Chebyshev
// nodes; eleven would be 3e-16 off and take 3 us more).  Four side by side: a step of one waits for the step before.
__device__ __forceinline__ double exp_sum4(const double (&x)[4]) {
  constexpr double kLog2E = 0x1.71547652b82fep+0, kWhole = 0x1.8p+52;
  constexpr double kPoly[] = {0x1.00dc4a532fb8ep-16, 0x1.4308ac85aa947p-13, 0x1.5d8745a728441p-10, 0x1.3b2ab7181b755p-7,
                              0x1.c6b08dd6fd234p-5, 0x1.ebfbdff823cedp-3, 0x1.62e42fef84cf0p-1, 0x1.0000000000000p+0};
  double u[4], f[4], y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) u[e] = __builtin_fma(x[e], kLog2E, kWhole);
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = u[e] - kWhole;
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = __builtin_fma(x[e], kLog2E, -f[e]), y[e] = 0x1.63d136366db24p-20;
#pragma unroll
  for (double c : kPoly) {
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = __builtin_fma(y[e], f[e], c);
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = __builtin_ldexp(y[e], __double2loint(u[e]));
  return (y[0] + y[1]) + (y[2] + y[3]);
}

// A workgroup has a piece of a row: its largest logit, its sum of exponentials, and its best K tokens.  Rows begin at any
// float (a load of 16 bytes wants 4-byte boundaries only), and a row's results do not depend on where.  Where rows are many
// (512 of 129280, a fifth of them ended: 51 us, 4.2 TB/s) bound by the vector units (busy 83 % of the time), most of whose
// work is the exponentials; few rows (4: 5.1 us) wait for their trip to memory.  (Exponentials and sums in 32 bits took 44, at
// memory's rate, and candidates of different beams nearer than 1e-6 could change places.)
template <int kPer>
__global__ void __launch_bounds__(kRowThreads, 7) k_beam_rows(BeamSelect p, BeamWork w) {
  __shared__ Best<float, int, kRowThreads> best;
  __shared__ float parts[kRowThreads / kWave];
  __shared__ double part_sums[kRowThreads / kWave];
  const int row = (int)blockIdx.y, piece = (int)blockIdx.x, tid = (int)threadIdx.x;
  if (p.ended != nullptr && ldg(p.ended + row) != 0) return;
  const int begin = piece * kRowThreads * kPer;
  const float* x = p.logits + (int64_t)row * p.vocab;
  float v[kPer];
  const auto token = [&](int i) { return begin + (i / 4 * kRowThreads + tid) * 4 + i % 4; };
  // Loads go before what other waves compute, and what is read once does not take the caches (512 rows 59 us without either, 56
  // with the latter, 55 with both; whole pieces then without their ends in mind 52, and seven waves a SIMD 51).
  __builtin_amdgcn_s_setprio(3);
  const auto put = [&](int i, f32x4 y) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[i + e] = y[e];
  };
  if (begin + kRowThreads * kPer <= p.vocab) {
    const float* from = x + begin;
#pragma unroll
    for (int i = 0; i < kPer; i += 4)
      put(i, __builtin_nontemporal_load((const UOCR_GLOBAL f32x4_at_float*)(from + i * kRowThreads + (uint32_t)tid * 4)));
  } else {
#pragma unroll
    for (int i = 0; i < kPer; i += 4) {
      const int at = token(i);
      f32x4 y = {-kInf, -kInf, -kInf, -kInf};
      if (at + 3 < p.vocab) {
        y = __builtin_nontemporal_load((const UOCR_GLOBAL f32x4_at_float*)(x + at));
      } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (at + e < p.vocab) y[e] = ldg(x + at + e);
      }
      put(i, y);
    }
  }
  __builtin_amdgcn_s_setprio(0);
  __builtin_amdgcn_sched_barrier(0);
  constexpr int kGroup = 8;  // tokens that are looked at together
  float largest[kPer / kGroup], mine = -kInf;
#pragma unroll
  for (int g = 0; g < kPer / kGroup; ++g) {
    const float* x = v + g * kGroup;
    largest[g] = max3(max3(max3(x[0], x[1], x[2]), x[3], x[4]), max3(x[5], x[6], x[7]), x[7]);
    mine = max3(mine, largest[g], largest[g]);
  }
  float m = tree_max(mine);  // (of the lanes without a NaN)
  if (lane_id() == 0) parts[tid / kWave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(parts[0], parts[1]), fmaxf(parts[2], parts[3]));
  // Terms and sum are in 64 bits: the sums of two rows decide between their candidates.  What is further below the largest than
  // 700 (e^-700 = 1e-304) counts as that far.
  double l = 0.0;
  const double off = m == -kInf ? 0.0 : (double)m;
#pragma unroll
  for (int i = 0; i < kPer; i += 4) {
    double x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __builtin_fmax((double)v[i + e] - off, -700.0);
    l += exp_sum4(x);
  }
  if (m == -kInf) l = 0.0;
  if (m == kInf || mine != mine) l = __builtin_nan("");
  for (int j = 32; j >= 1; j /= 2) l += __shfl_xor(l, j, kWave);
  if (lane_id() == 0) part_sums[tid / kWave] = l;
  __syncthreads();
  const int64_t at = (int64_t)row * w.pieces + piece;
  if (tid == 0) {
    w.tops[at] = m;
    w.sums[at] = (part_sums[0] + part_sums[1]) + (part_sums[2] + part_sums[3]);
  }
  float* values = w.values + at * p.beams;
  int* ids = w.ids + at * p.beams;
  // (of a row with a NaN nothing counts)
  const int found = choose(best, p.beams, mine,
                           [&](float least, auto f) {
#pragma unroll
                             for (int g = 0; g < kPer / kGroup; ++g)
                               if (largest[g] >= least) {
#pragma unroll
                                 for (int i = g * kGroup; i < (g + 1) * kGroup; ++i)
                                   if (v[i] >= least && v[i] > -kInf) f(v[i], token(i));
                               }
                           },
                           [&](int rank, float value, int id) {
                             values[rank] = value;
                             ids[rank] = id;
                           });
  for (int i = found + tid; i < p.beams; i += kRowThreads) ids[i] = -1;
}

__device__ __attribute__((noinline)) double full_exp(double x) { return exp(x); }

// A workgroup has a request: its beams' sums, their candidates, and the states of the chosen ones.  Bound by its dependent steps
// (sums, candidates, chosen, states): 7 us for one request of 4 beams, 10.5 for 64 of 8.
__global__ void __launch_bounds__(kJoinThreads) k_beam_join(BeamSelect p, BeamWork w) {
  __shared__ Best<double, int64_t, kJoinThreads> best;
  __shared__ double sums[kBeamsMost], scores[kBeamsMost], by[kBeamsMost];
  __shared__ int lengths[kBeamsMost], state[kBeamsMost];  // 0: live, 1: ended, 2: no finite sum
  __shared__ int tokens[kBeamsMost], parents[kBeamsMost];
  __shared__ float logits[kBeamsMost];
  const int K = p.beams, tid = (int)threadIdx.x, wave = tid / kWave, lane = lane_id();
  const bool penalised = p.lengths != nullptr && p.alpha != 0.0;
  const int64_t row0 = (int64_t)blockIdx.x * K;
  // The first candidates are asked for before the sums, which they wait for: of a request they lie one after another.
  constexpr int kHeld = 4;
  const int per = w.pieces * K, candidates = K * per;
  const int64_t first = row0 * per;
  int held_id[kHeld];
  float held[kHeld];
#pragma unroll
  for (int u = 0; u < kHeld; ++u) {
    const int i = tid + u * kJoinThreads;
    held_id[u] = i < candidates ? ldg(w.ids + first + i) : -1;
    held[u] = i < candidates ? ldg(w.values + first + i) : 0.0f;
  }
  for (int b = wave; b < K; b += kJoinThreads / kWave) {
    const int64_t row = row0 + b;
    const float* tops = w.tops + row * w.pieces;  // (an ended beam's are nobody's)
    const double* part_sums = w.sums + row * w.pieces;
    const bool ended = p.ended != nullptr && ldg(p.ended + row) != 0;
    const double score = ldg(p.scores + row);
    const int length = p.lengths != nullptr ? ldg(p.lengths + row) + (ended ? 0 : 1) : 0;
    const bool some = lane < w.pieces;
    const float m0 = some ? ldg(tops + lane) : -kInf;
    const double l0 = some ? ldg(part_sums + lane) : 0.0;
    float m = m0;
    for (int i = lane + kWave; i < w.pieces; i += kWave) m = fmaxf(m, ldg(tops + i));
    m = tree_max(m);
    const auto at_most = [&](float mi, double li) { return li == 0.0 ? 0.0 : li * full_exp((double)mi - (double)m); };
    double l = at_most(m0, l0);
    for (int i = lane + kWave; i < w.pieces; i += kWave) l += at_most(ldg(tops + i), ldg(part_sums + i));
    for (int off = 32; off >= 1; off /= 2) l += __shfl_xor(l, off, kWave);
    // (pow's code alone takes as long to fetch as all else here: length^|alpha| by the logarithm, in the lane next to the sum's.
    // Off by 2^-46 of itself at most, so that powers that near to a whole number count as that: beams of different lengths may
    // have equal ranks where their powers are whole.)
    const double logs = log(lane == 1 ? (double)length : l);
    const double lse = (double)m + __shfl(logs, 0, kWave);
    double power = penalised ? full_exp(__builtin_fabs(p.alpha) * __shfl(logs, 1, kWave)) : 1.0;
    const double whole = __builtin_rint(power);
    power = __builtin_fabs(power - whole) <= 0x1p-46 * power ? whole : power;
    if (lane == 0) {
      sums[b] = lse;
      scores[b] = score;
      by[b] = power;
      lengths[b] = length;
      state[b] = ended ? 1 : score - score == 0.0 && lse - lse == 0.0 ? 0 : 2;
    }
  }
  __syncthreads();
  const auto key_of = [&](int b, float logit) { return state[b] == 1 ? scores[b] : scores[b] + ((double)logit - sums[b]); };
  // A candidate's id is in the order of ties: 5 bits of its beam, 32 of its logit (the larger first), 26 of its place among the
  // beam's (a row's pieces and what each has found are in the order of their tokens where logits are equal).
  constexpr int kPlaceBits = 26, kBeamAt = kPlaceBits + 32;
  const auto offer = [&](auto f, int b, double key, float logit, int place) {
    const double rank = !penalised ? key : p.alpha < 0.0 ? key * by[b] : key / by[b];
    if (rank - rank == 0.0) f(rank, (int64_t)b << kBeamAt | (int64_t)~ordered(logit) << kPlaceBits | place);
  };
  const auto one = [&](auto f, int i, float logit, int id) {
    const int b = w.by_beam(i);
    if (state[b] == 0) {
      if (id >= 0) offer(f, b, key_of(b, logit), logit, i - b * per);
    } else if (state[b] == 1 && i == b * per) {
      offer(f, b, scores[b], 0.0f, 0);
    }
  };
  const auto each = [&](float least, auto f) {
    const auto some = [&](double rank, int64_t id) {
      if ((float)rank >= least) f(rank, id);
    };
#pragma unroll
    for (int u = 0; u < kHeld; ++u)
      if (tid + u * kJoinThreads < candidates) one(some, tid + u * kJoinThreads, held[u], held_id[u]);
    for (int i = tid + kHeld * kJoinThreads; i < candidates; i += kJoinThreads)
      one(some, i, ldg(w.values + first + i), ldg(w.ids + first + i));
  };
  double mine = -__builtin_huge_val();
  each(-kInf, [&](double rank, int64_t) { mine = rank > mine ? rank : mine; });
  const int found = choose(best, K, mine, each, [&](int rank, double, int64_t id) {
    const int b = (int)(id >> kBeamAt), place = (int)id & ((1 << kPlaceBits) - 1);
    parents[rank] = b;
    tokens[rank] = state[b] == 1 ? p.eos : ldg(w.ids + first + (b * per + place));
    logits[rank] = of_ordered(~(uint32_t)(id >> kPlaceBits));
  });
  __syncthreads();
  if (tid == 0)  // fewer with a finite rank than beams: the others in order
    for (int k = found, b = 0, t = 0; k < K;) {
      const int token = state[b] == 1 ? p.eos : t;
      bool taken = false;
      for (int i = 0; i < found; ++i) taken = taken || (parents[i] == b && tokens[i] == token);
      if (!taken) {
        parents[k] = b;
        tokens[k++] = token;
      }
      if (state[b] == 1 || ++t == p.vocab) {
        ++b;
        t = 0;
      }
    }
  __syncthreads();
  if (tid < K) {
    const int b = parents[tid], token = tokens[tid];
    const int64_t row = row0 + tid;
    const bool counts = tid < found;  // others come after all, as -inf
    const bool ended = p.ended != nullptr && ldg(p.ended + row0 + b) != 0;
    stg(p.tokens_out + row, token);
    stg(p.parents_out + row, (int)(row0 + b));
    stg(p.scores_out + row, counts ? (float)key_of(b, logits[tid]) : -kInf);
    stg(p.ended_out + row, (int)(ended || token == p.eos));
    if (p.lengths != nullptr) stg(p.lengths_out + row, lengths[b]);
  }
  if (p.history == nullptr) return;
  for (int k = wave; k < K; k += kJoinThreads / kWave) {
    const int64_t from = (row0 + parents[k]) * p.width, to = (row0 + k) * p.width;
    const int shift = p.ended != nullptr && ldg(p.ended + row0 + parents[k]) != 0 ? 0 : 1;
    for (int64_t i = lane; i < p.width; i += kWave)
      stg(p.history_out + to + i, i + shift < p.width ? ldg(p.history + from + i + shift) : tokens[k]);
  }
}

// Tokens of a thread: 8 where the rows are few, so that their pieces fill the device, else 32.
int per_thread(int64_t rows, int vocab) { return rows * ((vocab + 32 * kRowThreads - 1) / (32 * kRowThreads)) < 512 ? 8 : 32; }
int pieces_of(int64_t rows, int vocab) {
  const int size = per_thread(rows, vocab) * kRowThreads;
  return (int)(((int64_t)vocab + size - 1) / size);
}

}  // namespace

size_t beam_workspace_bytes(int64_t rows, int beams, int vocab) {
  return (size_t)rows * pieces_of(rows, vocab) * (3 + 2 * (size_t)beams) * 4;
}

hipError_t launch_beam_select(const BeamSelect& p, int64_t rows, void* workspace, hipStream_t s) {
  if (rows == 0) return hipSuccess;
  BeamWork w{};
  w.pieces = pieces_of(rows, p.vocab);
  w.by_beam = divide_by(w.pieces * p.beams);
  const int64_t n = rows * w.pieces;
  w.sums = (double*)workspace;
  w.tops = (float*)(w.sums + n);
  w.values = w.tops + n;
  w.ids = (int*)(w.values + n * p.beams);
  const dim3 grid((unsigned)w.pieces, (unsigned)rows), block(kRowThreads);
  const auto kernel = per_thread(rows, p.vocab) == 8 ? k_beam_rows<8> : k_beam_rows<32>;
  UOCR_LAUNCH("beam_rows", kernel, grid, block, 0, s, p, w);
  UOCR_LAUNCH("beam_join", k_beam_join, dim3((unsigned)(rows / p.beams)), dim3(kJoinThreads), 0, s, p, w);
  return hipGetLastError();
}

}  // namespace uocr
