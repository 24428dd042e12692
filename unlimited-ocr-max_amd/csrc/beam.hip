// A step of beam search: of every request's beams and their next tokens the best, and the beams' states in their order.
// The reference decodes one beam; what feeds this (logits after the n-gram guard, unlimited_ocr_max/ngram.py:33-53, and
// the guard's history) and what follows (the pages' forks) is this library's.
//
//   key(b, v) = score_b + (logit[b, v] - log sum_v exp logit[b, v])          a live beam
//   key(b, eos) = score_b, no other token                                    an ended one
//   rank = key / length^alpha, the length with the new token                 (given lengths; else rank = key)
//
// The K best of a request's K beams by rank, ties to the lower (beam, token).  Keys and ranks are in 64 bits: which
// of two near candidates wins decides what a request says.  A candidate whose rank is not finite (a token at -inf, a beam
// whose score or sum is not finite) comes after all others, as -inf; of a beam without a finite sum it is the first
// tokens that do.
#include "uocr_device.h"
#include "uocr_kernels.h"

namespace uocr {

namespace {

typedef float f32x4_at_float __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kThreads = 256;
constexpr float kInf = __builtin_huge_valf();
constexpr int kList = 1024;  // candidates that are ranked against one another in LDS

// Of the candidates that the threads of a workgroup hold, the first `most` by value (descending) and id (ascending).
// each(f) calls f(value, id) for a thread's candidates, put(rank, value, id) takes a chosen one; returns their number.
//
// At least `most` candidates are no smaller than the most-th largest of the threads' largest ones, and few are as large:
// those are listed, and ranked by counting.  Where equal values fill the list, each next one is looked for among all.
template <typename V, typename Id>
struct Best {
  V largest[kThreads];
  V value[kList];
  Id id[kList];
  V border;
  int listed;
};
template <typename V, typename Id, typename Each, typename Put>
__device__ __forceinline__ int choose(Best<V, Id>& b, int most, Each each, Put put) {
  const int tid = (int)threadIdx.x;
  const V none = -(V)__builtin_huge_val();
  V mine = none;
  each([&](V v, Id) { mine = v > mine ? v : mine; });
  b.largest[tid] = mine;
  if (tid == 0) b.listed = 0;
  __syncthreads();
  int before = 0;
  for (int i = 0; i < kThreads; ++i) {
    const V o = b.largest[i];
    before += o > mine || (o == mine && i < tid);
  }
  if (before == most - 1) b.border = mine;
  __syncthreads();
  const V border = b.border;
  if (mine >= border)
    each([&](V v, Id id) {
      if (v >= border) {
        const int at = atomicAdd(&b.listed, 1);
        if (at < kList) {
          b.value[at] = v;
          b.id[at] = id;
        }
      }
    });
  __syncthreads();
  const int n = b.listed;
  if (n <= kList) {
    for (int i = tid; i < n; i += kThreads) {
      const V v = b.value[i];
      const Id id = b.id[i];
      int rank = 0;
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
    each([&](V x, Id id) {
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

// A workgroup has a piece of a row: its largest logit, its sum of exponentials, and its best K tokens.  Rows begin at any
// float (a load of 16 bytes wants 4-byte boundaries only), and a row's results do not depend on where.
template <int kPer>
__global__ void __launch_bounds__(kThreads) k_beam_rows(BeamSelect p, BeamWork w) {
  __shared__ Best<float, int> best;
  __shared__ float parts[kThreads / kWave];
  const int row = (int)blockIdx.y, piece = (int)blockIdx.x, tid = (int)threadIdx.x;
  if (p.ended != nullptr && ldg(p.ended + row) != 0) return;
  const int begin = piece * kThreads * kPer;
  const float* x = p.logits + (int64_t)row * p.vocab;
  float v[kPer];
  const auto token = [&](int i) { return begin + (i / 4 * kThreads + tid) * 4 + i % 4; };
#pragma unroll
  for (int i = 0; i < kPer; i += 4) {
    const int at = token(i);
    f32x4 y = {-kInf, -kInf, -kInf, -kInf};
    if (at + 3 < p.vocab) {
      y = *(const UOCR_GLOBAL f32x4_at_float*)(x + at);
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (at + e < p.vocab) y[e] = ldg(x + at + e);
    }
    v[i] = y.x;
    v[i + 1] = y.y;
    v[i + 2] = y.z;
    v[i + 3] = y.w;
  }
  float m = v[0];
#pragma unroll
  for (int i = 1; i < kPer; ++i) m = fmaxf(m, v[i]);
  m = tree_max(m);
  if (lane_id() == 0) parts[tid / kWave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(parts[0], parts[1]), fmaxf(parts[2], parts[3]));
  __syncthreads();
  float l = 0.0f;
  const float off = m == -kInf ? 0.0f : m;
#pragma unroll
  for (int i = 0; i < kPer; ++i) l += __builtin_amdgcn_exp2f((v[i] - off) * 1.44269504f);
  l = tree_sum(l);
  if (lane_id() == 0) parts[tid / kWave] = l;
  __syncthreads();
  const int64_t at = (int64_t)row * w.pieces + piece;
  if (tid == 0) {
    w.tops[2 * at] = m;
    w.tops[2 * at + 1] = (parts[0] + parts[1]) + (parts[2] + parts[3]);
  }
  float* values = w.values + at * p.beams;
  int* ids = w.ids + at * p.beams;
  const int found = choose(best, p.beams,
                           [&](auto f) {
#pragma unroll
                             for (int i = 0; i < kPer; ++i)
                               if (v[i] > -kInf) f(v[i], token(i));
                           },
                           [&](int rank, float value, int id) {
                             values[rank] = value;
                             ids[rank] = id;
                           });
  for (int i = found + tid; i < p.beams; i += kThreads) ids[i] = -1;
}

// A workgroup has a request: its beams' sums, their candidates, and the states of the chosen ones.
__global__ void __launch_bounds__(kThreads) k_beam_join(BeamSelect p, BeamWork w) {
  __shared__ Best<double, int64_t> best;
  __shared__ double sums[kBeamsMost], scores[kBeamsMost], by[kBeamsMost];
  __shared__ int lengths[kBeamsMost], state[kBeamsMost];  // 0: live, 1: ended, 2: no finite sum
  __shared__ int tokens[kBeamsMost], parents[kBeamsMost];
  const int K = p.beams, tid = (int)threadIdx.x, wave = tid / kWave, lane = lane_id();
  const int64_t row0 = (int64_t)blockIdx.x * K;
  for (int b = wave; b < K; b += kThreads / kWave) {
    const int64_t row = row0 + b;
    const bool ended = p.ended != nullptr && ldg(p.ended + row) != 0;
    const double score = ldg(p.scores + row);
    double lse = 0.0;
    if (!ended) {
      const float* tops = w.tops + 2 * row * w.pieces;
      float m = -kInf;
      for (int i = lane; i < w.pieces; i += kWave) m = fmaxf(m, ldg(tops + 2 * i));
      m = tree_max(m);
      double l = 0.0;
      for (int i = lane; i < w.pieces; i += kWave) {
        const float mi = ldg(tops + 2 * i);
        const double li = ldg(tops + 2 * i + 1);
        l += li == 0.0 ? 0.0 : li * exp((double)mi - (double)m);
      }
      for (int off = 32; off >= 1; off /= 2) l += __shfl_xor(l, off, kWave);
      lse = (double)m + log(l);
    }
    if (lane == 0) {
      const int length = p.lengths != nullptr ? ldg(p.lengths + row) + (ended ? 0 : 1) : 0;
      const bool finite = score - score == 0.0 && lse - lse == 0.0;
      sums[b] = lse;
      scores[b] = score;
      by[b] = p.lengths != nullptr ? pow((double)length, p.alpha) : 1.0;
      lengths[b] = length;
      state[b] = ended ? 1 : finite ? 0 : 2;
    }
  }
  __syncthreads();
  const int per = w.pieces * K;
  const auto key_of = [&](int b, float logit) { return state[b] == 1 ? scores[b] : scores[b] + ((double)logit - sums[b]); };
  const auto offer = [&](auto f, int b, double key, int token) {
    const double rank = key / by[b];
    if (rank - rank == 0.0) f(rank, (int64_t)b * p.vocab + token);
  };
  const auto each = [&](auto f) {
    for (int i = tid; i < K * per; i += kThreads) {
      const int b = i / per, j = i - b * per;
      if (state[b] == 0) {
        const int64_t at = (row0 + b) * per + j;
        const int id = ldg(w.ids + at);
        if (id >= 0) offer(f, b, key_of(b, ldg(w.values + at)), id);
      } else if (state[b] == 1 && j == 0) {
        offer(f, b, scores[b], p.eos);
      }
    }
  };
  const int found = choose(best, K, each, [&](int rank, double, int64_t id) {
    const int b = (int)(id / p.vocab);
    parents[rank] = b;
    tokens[rank] = (int)(id - (int64_t)b * p.vocab);
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
    const double key = state[b] == 2 ? -__builtin_huge_val()
                                     : key_of(b, state[b] == 1 ? 0.0f : ldg(p.logits + (row0 + b) * p.vocab + token));
    const bool counts = tid < found;  // others come after all, as -inf
    const bool ended = p.ended != nullptr && ldg(p.ended + row0 + b) != 0;
    stg(p.tokens_out + row, token);
    stg(p.parents_out + row, (int)(row0 + b));
    stg(p.scores_out + row, counts ? (float)key : -kInf);
    stg(p.ended_out + row, (int)(ended || token == p.eos));
    if (p.lengths != nullptr) stg(p.lengths_out + row, lengths[b]);
  }
  if (p.history == nullptr) return;
  for (int k = wave; k < K; k += kThreads / kWave) {
    const int64_t from = (row0 + parents[k]) * p.width, to = (row0 + k) * p.width;
    const int shift = p.ended != nullptr && ldg(p.ended + row0 + parents[k]) != 0 ? 0 : 1;
    for (int64_t i = lane; i < p.width; i += kWave)
      stg(p.history_out + to + i, i + shift < p.width ? ldg(p.history + from + i + shift) : tokens[k]);
  }
}

// Tokens of a thread: 8 where the rows are few, so that their pieces fill the device, else 32.
int per_thread(int64_t rows, int vocab) { return rows * ((vocab + 32 * kThreads - 1) / (32 * kThreads)) < 512 ? 8 : 32; }
int pieces_of(int64_t rows, int vocab) {
  const int size = per_thread(rows, vocab) * kThreads;
  return (int)(((int64_t)vocab + size - 1) / size);
}

}  // namespace

size_t beam_workspace_bytes(int64_t rows, int beams, int vocab) {
  return (size_t)rows * pieces_of(rows, vocab) * (2 + 2 * (size_t)beams) * 4;
}

hipError_t launch_beam_select(const BeamSelect& p, int64_t rows, void* workspace, hipStream_t s) {
  if (rows == 0) return hipSuccess;
  BeamWork w{};
  w.pieces = pieces_of(rows, p.vocab);
  const int64_t n = rows * w.pieces;
  w.tops = (float*)workspace;
  w.values = w.tops + 2 * n;
  w.ids = (int*)(w.values + n * p.beams);
  const dim3 grid((unsigned)w.pieces, (unsigned)rows), block(kThreads);
  const auto kernel = per_thread(rows, p.vocab) == 8 ? k_beam_rows<8> : k_beam_rows<32>;
  UOCR_LAUNCH("beam_rows", kernel, grid, block, 0, s, p, w);
  UOCR_LAUNCH("beam_join", k_beam_join, dim3((unsigned)(rows / p.beams)), block, 0, s, p, w);
  return hipGetLastError();
}

}  // namespace uocr
