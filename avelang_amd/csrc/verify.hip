// Which nodes of a drafted tree the target model accepts, and the token behind them.
//
//   row sums     one launch over all rows and pieces of the vocabulary: largest logit, its lowest index, sum of exp((x - largest) / temperature)
//   rejections   (drafts with distributions only) sum of max(p - q, 0) of the rows whose first child is rejected, then, a workgroup a row, the
//                children that are left
//   walk         a workgroup a sequence: whether a node is accepted once its parent is and its elder siblings are not does not depend on the
//                rest of the walk, so all nodes' probabilities are fetched at once; then the path, then the token: among the sums of the
//                pieces first, and in one piece element by element
//
// Everything behind a logit is fp64: a token is chosen by where a number lies among the running sums of 10^5 probabilities, and in fp32 one
// draw in some hundred to thousand would go to a neighbour by rounding.
#include <algorithm>

#include "fp4_common.hpp"
#include "kv_cache.hpp"

namespace ave {
namespace {

constexpr int kPiece = kVocabPiece;
constexpr int kRowThreads = 256, kWalkThreads = 1024;

struct PieceSum {
  double sum;   // of exp((x - top) / temperature)
  float top;    // -inf: no number
  int at;       // the lowest index of top
};
struct VerifyArgs {
  ave_fp4_draft d;
  int pieces;
  PieceSum* sums;      // [rows][pieces]
  double* rest;        // [rows][pieces]: sums of max(p - t q, 0), where a row's children are rejected
  double* times;       // [rows]: that t, 0 without rejections
  int* choice;         // [rows]: the accepted child, -1
};

struct Span {
  int first, n;
};
__device__ inline Span span_of(const VerifyArgs& p, int b) {
  Span s;
  int end = p.d.cu_q[b + 1];
  s.first = p.d.cu_q[b];
  s.first = s.first < 0 ? 0 : s.first > p.d.rows ? p.d.rows : s.first;
  end = end < s.first ? s.first : end > p.d.rows ? p.d.rows : end;
  s.n = end - s.first;
  return s;
}
// The sequence of a row (every wave by itself), -1: nobody's.  64 probes at a time; if offsets fall, any sequence that has the row, or none.
__device__ inline int sequence_of(const VerifyArgs& p, int row) {
  const int lane = threadIdx.x & 63;
  int from = 0, many = p.d.batch;   // the last sequence that starts at or before the row is among these
  while (many > 0) {
    const int step = (many + 63) / 64, b = from + lane * step;
    const uint64_t below = __ballot(lane * step < many && p.d.cu_q[b] <= row);
    if (!below) return -1;
    const int last = 63 - __clzll((long long)below);
    from += last * step;
    many = step == 1 ? 0 : min(step, many - last * step);
  }
  if (p.d.batch <= 0) return -1;
  // (an empty sequence starts where the next one does, and comes before it)
  const Span s = span_of(p, __builtin_amdgcn_readfirstlane(from));
  return row >= s.first && row < s.first + s.n ? __builtin_amdgcn_readfirstlane(from) : -1;
}
// 1 / temperature in units of log2(e); 0: the largest logit
__device__ inline double inverse_temperature(const VerifyArgs& p, int b) {
  const float t = p.d.temperature ? p.d.temperature[b] : 1.0f;
  return t > 0.0f ? 1.4426950408889634 / (double)fminf(t, 3.402823466e38f) : 0.0;
}

// 2^y for y <= 0: 2^n times the Taylor polynomial of e^f, |f| <= ln 2 / 2, whose first missing term is below 2e-16
__device__ inline double exp2_of(double y) {
  y = fmax(y, -1100.0);
  const double n = rint(y), f = (y - n) * 0.6931471805599453;
  double r = 1.0 / 479001600.0;
  r = fma(r, f, 1.0 / 39916800.0);
  r = fma(r, f, 1.0 / 3628800.0);
  r = fma(r, f, 1.0 / 362880.0);
  r = fma(r, f, 1.0 / 40320.0);
  r = fma(r, f, 1.0 / 5040.0);
  r = fma(r, f, 1.0 / 720.0);
  r = fma(r, f, 1.0 / 120.0);
  r = fma(r, f, 1.0 / 24.0);
  r = fma(r, f, 1.0 / 6.0);
  r = fma(r, f, 0.5);
  r = fma(r, f, 1.0);
  r = fma(r, f, 1.0);
  return ldexp(r, (int)n);
}
// exp((x - top) / temperature); x <= top, either may be -inf (then 0)
__device__ inline double weight_of(float x, float top, double per) {
  return x == -INFINITY ? 0.0 : exp2_of(((double)x - (double)top) * per);
}

__device__ inline float number(float x) { return x != x ? -INFINITY : fminf(x, 3.402823466e38f); }
template <bool F32>
__device__ inline float logit(const VerifyArgs& p, int row, int i) {
  if constexpr (F32) return number(static_cast<const float*>(p.d.logits)[(int64_t)row * p.d.logits_stride + i]);
  else return number(__builtin_bit_cast(float, (unsigned)static_cast<const uint16_t*>(p.d.logits)[(int64_t)row * p.d.logits_stride + i] << 16));
}
// N consecutive logits from index i on, -inf behind the last
template <bool F32, int N>
__device__ inline void logits(const VerifyArgs& p, int row, int i, float (&x)[N]) {
  constexpr int kOf = F32 ? 4 : 8;   // elements of 16 bytes
  static_assert(N % kOf == 0, "");
  const int64_t at = (int64_t)row * p.d.logits_stride + i;
  const char* from = static_cast<const char*>(p.d.logits) + at * (F32 ? 4 : 2);
  if (i + N <= p.d.vocab && reinterpret_cast<uintptr_t>(from) % 16 == 0) {
    v4i raw[N / kOf];
#pragma unroll
    for (int k = 0; k < N / kOf; ++k) raw[k] = reinterpret_cast<const v4i*>(from)[k];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if constexpr (F32) x[k] = number(__builtin_bit_cast(float, (int)raw[k / 4][k % 4]));
      else x[k] = number(__builtin_bit_cast(float, k % 2 ? (unsigned)raw[k / 8][k % 8 / 2] & 0xFFFF0000u : (unsigned)raw[k / 8][k % 8 / 2] << 16));
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = i + k < p.d.vocab ? logit<F32>(p, row, i + k) : -INFINITY;
  }
}
__device__ inline double draft_prob(const VerifyArgs& p, int row, int i) {
  const float q = p.d.draft_probs[(int64_t)row * p.d.draft_probs_stride + i];
  return q > 0.0f ? (double)q : 0.0;
}

// ---- over a workgroup ------------------------------------------------------------------------------------------------------------------
__device__ inline double wave_sum(double v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}
// of every thread's v, in all threads; `scratch` has an element a wave and is free again when the next call's barrier has passed
template <int THREADS>
__device__ inline double block_sum(double v, double* scratch) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x / 64] = v;
  __syncthreads();
  double all = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) all += scratch[w];
  return all;
}

// ---- a row's sums ------------------------------------------------------------------------------------------------------------------------
template <bool F32>
__global__ __launch_bounds__(kRowThreads) void row_sums_kernel(VerifyArgs p) {
  constexpr int kEach = kPiece / kRowThreads, kOnce = 8;   // elements of a thread, together in memory
  __shared__ double scratch[kRowThreads / 64];
  __shared__ float tops[kRowThreads / 64];
  __shared__ int ats[kRowThreads / 64];
  const int row = blockIdx.x / (unsigned)p.pieces, piece = blockIdx.x % (unsigned)p.pieces, b = sequence_of(p, row);
  if (b < 0) return;
  const double per = inverse_temperature(p, b);
  float x[kEach / kOnce][kOnce];
#pragma unroll
  for (int k = 0; k < kEach / kOnce; ++k) logits<F32>(p, row, piece * kPiece + (k * kRowThreads + threadIdx.x) * kOnce, x[k]);
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < kEach; ++k) top = fmaxf(top, x[k / kOnce][k % kOnce]);
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x / 64] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowThreads / 64; ++w) top = fmaxf(top, tops[w]);
  int at = INT32_MAX;
  double sum = 0.0;
#pragma unroll
  for (int k = kEach - 1; k >= 0; --k) {
    if (x[k / kOnce][k % kOnce] == top) at = piece * kPiece + (k / kOnce * kRowThreads + threadIdx.x) * kOnce + k % kOnce;
    if (per > 0.0) sum += weight_of(x[k / kOnce][k % kOnce], top, per);
  }
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) at = min(at, __shfl_xor(at, m, 64));
  if ((threadIdx.x & 63) == 0) ats[threadIdx.x / 64] = at;
  sum = block_sum<kRowThreads>(sum, scratch);
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 0; w < kRowThreads / 64; ++w) at = min(at, ats[w]);
    p.sums[(size_t)row * p.pieces + piece] = {sum, top, at};
  }
}

struct RowSum {
  double sum;
  float top;
  int at;
};
// Of all pieces, by one wave, in all of its lanes.  (The order of the sum depends on the number of pieces alone.)
__device__ inline RowSum row_sum(const VerifyArgs& p, int row, double per) {
  const PieceSum* s = p.sums + (size_t)row * p.pieces;
  const int lane = threadIdx.x & 63;
  RowSum r{0.0, -INFINITY, INT32_MAX};
  for (int c = lane; c < p.pieces; c += 64)
    if (s[c].top > r.top) r.top = s[c].top, r.at = s[c].at;
  float top = r.top;
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
  r.at = r.top == top && top != -INFINITY ? r.at : INT32_MAX;
  r.top = top;
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) r.at = min(r.at, __shfl_xor(r.at, m, 64));
  if (per > 0.0) {
    for (int c = lane; c < p.pieces; c += 64) r.sum += s[c].top == -INFINITY ? 0.0 : s[c].sum * weight_of(s[c].top, top, per);
    r.sum = wave_sum(r.sum);
  }
  return r;
}

// ---- rejections, where drafts come with distributions ----------------------------------------------------------------------------------------
// Children of node v of a sequence from node `from` on: the next one, or n (every wave by itself)
__device__ inline int next_child(const VerifyArgs& p, const Span& s, int v, int from) {
  const int lane = threadIdx.x & 63;
  for (int c0 = from; c0 < s.n; c0 += 64) {
    const int c = c0 + lane;
    const uint64_t any = __ballot(c < s.n && c > v && p.d.parents[s.first + c] == v);
    if (any) return c0 + __ffsll((unsigned long long)any) - 1;
  }
  return s.n;
}
__device__ inline double uniform_of(const VerifyArgs& p, int row) {
  const float u = p.d.uniform[row];
  return u > 0.0f ? fmin((double)u, 1.0) : 0.0;
}
// Is child c accepted, with t and s = sum of max(p - t q, 0)?
template <bool F32>
__device__ inline bool accepts(const VerifyArgs& p, int row, const RowSum& r, double per, int child_row, double t, double s) {
  const int token = p.d.tokens[child_row];
  if (token < 0 || token >= p.d.vocab || !(r.sum > 0.0)) return false;
  const double q = draft_prob(p, row, token), w = weight_of(logit<F32>(p, row, token), r.top, per) / r.sum;
  return uniform_of(p, child_row) * q * s < fmax(w - t * q, 0.0);
}

template <bool F32>
__global__ __launch_bounds__(kRowThreads) void rest_sums_kernel(VerifyArgs p) {
  constexpr int kEach = kPiece / kRowThreads, kOnce = 8;
  __shared__ double scratch[kRowThreads / 64];
  const int row = blockIdx.x / (unsigned)p.pieces, piece = blockIdx.x % (unsigned)p.pieces, b = sequence_of(p, row);
  if (b < 0) return;
  const double per = inverse_temperature(p, b);
  const Span s = span_of(p, b);
  const int v = row - s.first, child = next_child(p, s, v, v + 1);
  if (child >= s.n || per == 0.0) return;
  const RowSum r = row_sum(p, row, per);
  if (!(r.sum > 0.0) || accepts<F32>(p, row, r, per, s.first + child, 0.0, 1.0)) return;
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < kEach / kOnce; ++k) {
    const int i = piece * kPiece + (k * kRowThreads + threadIdx.x) * kOnce;
    float x[kOnce];
    logits<F32>(p, row, i, x);
#pragma unroll
    for (int j = 0; j < kOnce; ++j)
      if (i + j < p.d.vocab) sum += fmax(weight_of(x[j], r.top, per) / r.sum - draft_prob(p, row, i + j), 0.0);
  }
  sum = block_sum<kRowThreads>(sum, scratch);
  if (threadIdx.x == 0) p.rest[(size_t)row * p.pieces + piece] = sum;
}

// A row's children one after the other
template <bool F32>
__global__ __launch_bounds__(kWalkThreads) void children_kernel(VerifyArgs p) {
  constexpr int kEach = kPiece / kWalkThreads;
  __shared__ double scratch[kWalkThreads / 64];
  const int row = blockIdx.x, b = sequence_of(p, row);
  if (b < 0) return;
  const double per = inverse_temperature(p, b);
  if (per == 0.0) return;
  const Span s = span_of(p, b);
  const int v = row - s.first;
  const RowSum r = row_sum(p, row, per);
  double t = 0.0, left = 1.0;
  int found = -1, tried = 0;
  for (int child = next_child(p, s, v, v + 1); child < s.n; child = next_child(p, s, v, child + 1)) {
    if (tried == 1) {
      t = 1.0, left = 0.0;
      for (int c = 0; c < p.pieces; ++c) left += p.rest[(size_t)row * p.pieces + c];
    } else if (tried > 1) {
      t += left, left = 0.0;
      for (int c = 0; c < p.pieces; ++c) {
        double sum = 0.0;
        const int i = c * kPiece + threadIdx.x * kEach;
        float x[kEach];
        logits<F32>(p, row, i, x);
#pragma unroll
        for (int j = 0; j < kEach; ++j)
          if (i + j < p.d.vocab) sum += fmax(weight_of(x[j], r.top, per) / r.sum - t * draft_prob(p, row, i + j), 0.0);
        left += block_sum<kWalkThreads>(sum, scratch);
      }
    }
    if (accepts<F32>(p, row, r, per, s.first + child, t, left)) {
      found = child;
      break;
    }
    ++tried;
  }
  // nothing accepted: what the next token is drawn from
  if (found < 0 && r.sum > 0.0 && tried > 1) {
    t += left;
    for (int c = 0; c < p.pieces; ++c) {
      double sum = 0.0;
      const int i = c * kPiece + threadIdx.x * kEach;
      float x[kEach];
      logits<F32>(p, row, i, x);
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        if (i + j < p.d.vocab) sum += fmax(weight_of(x[j], r.top, per) / r.sum - t * draft_prob(p, row, i + j), 0.0);
      sum = block_sum<kWalkThreads>(sum, scratch);
      if (threadIdx.x == 0) p.rest[(size_t)row * p.pieces + c] = sum;
    }
  } else if (tried == 1) {
    t = 1.0;
  }
  if (threadIdx.x == 0) p.choice[row] = found, p.times[row] = found < 0 ? t : 0.0;
}

// ---- the walk ----------------------------------------------------------------------------------------------------------------------------------
template <bool F32>
__global__ __launch_bounds__(kWalkThreads) void walk_kernel(VerifyArgs p) {
  constexpr int kEach = kPiece / kWalkThreads, kWaves = kWalkThreads / 64;
  __shared__ double scratch[kWaves];
  __shared__ double wave_at[kWaves + 1];
  __shared__ int said[4];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  const Span s = span_of(p, b);
  const double per = inverse_temperature(p, b);
  if (s.n == 0) {
    if (threadIdx.x == 0) p.d.accepted[b] = 0;
    return;
  }
  if (wave == 0) {
    int at = 0, kept = 1;
    double taken = 0.0;
    RowSum r = row_sum(p, s.first, per);
    const auto accept = [&](int child) {
      at = child, taken = 0.0;
      if (lane == 0) {
        p.d.path[s.first + kept] = child;
        p.d.emitted[s.first + kept - 1] = p.d.tokens[s.first + child];
      }
      ++kept;
      r = row_sum(p, s.first + child, per);
    };
    if (lane == 0) p.d.path[s.first] = 0;
    if (p.d.draft_probs && per > 0.0) {
      for (int child; (child = p.choice[s.first + at]) > at && child < s.n;) accept(child);
    } else {
      for (int child = next_child(p, s, 0, 1); child < s.n; child = next_child(p, s, at, child + 1)) {
        const int token = p.d.tokens[s.first + child];
        if (token < 0 || token >= p.d.vocab) continue;
        if (per == 0.0) {
          if (token == r.at) accept(child);
          continue;
        }
        // a token that an elder sibling had has been taken out
        bool again = false;
        for (int c0 = at + 1; c0 < child; c0 += 64) {
          const int c = c0 + lane;
          again = again || __any(c < child && p.d.parents[s.first + c] == at && p.d.tokens[s.first + c] == token);
        }
        if (again || !(r.sum > 0.0)) continue;
        const double mine = weight_of(logit<F32>(p, s.first + at, token), r.top, per) / r.sum;
        if (uniform_of(p, s.first + child) * (1.0 - taken) < mine) accept(child);
        else taken += mine;
      }
    }
    for (int i = kept + lane; i < s.n; i += 64) p.d.path[s.first + i] = -1, p.d.emitted[s.first + i] = -1;
    if (lane == 0) p.d.accepted[b] = kept, said[0] = at, said[1] = kept, said[2] = r.at;
    if (lane == 0) scratch[0] = r.sum, scratch[1] = (double)r.top;
  }
  __syncthreads();
  const int at = said[0], kept = said[1], row = s.first + at;
  int32_t* out = p.d.emitted + s.first + kept - 1;
  RowSum r{scratch[0], (float)scratch[1], said[2]};
  __syncthreads();
  if (per == 0.0 || !(r.sum > 0.0)) {
    if (threadIdx.x == 0) *out = r.top == -INFINITY ? -1 : r.at;
    return;
  }
  // The next token: weights in units of the row's largest, which are p r.sum.  `how`: 0 p, 1 p without the children's tokens, 2 max(p - t q, 0)
  const double t = p.d.draft_probs ? p.times[row] : 0.0;
  int how = p.d.draft_probs ? (t > 0.0 ? 2 : 0) : next_child(p, s, at, at + 1) < s.n ? 1 : 0;
  const auto weights = [&](int c, double (&w)[kEach]) {   // of this thread's elements of piece c
    const int i = c * kPiece + threadIdx.x * kEach;
    float x[kEach];
    logits<F32>(p, row, i, x);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      w[j] = i + j < p.d.vocab ? weight_of(x[j], r.top, per) / r.sum : 0.0;
      if (how == 2 && i + j < p.d.vocab) w[j] = fmax(w[j] - t * draft_prob(p, row, i + j), 0.0);
    }
    if (how == 1)
      for (int k = next_child(p, s, at, at + 1); k < s.n; k = next_child(p, s, at, k + 1)) {
        const int gone = p.d.tokens[s.first + k] - i;
#pragma unroll
        for (int j = 0; j < kEach; ++j)
          if (gone == j) w[j] = 0.0;
      }
  };
  const auto piece_sum = [&](int c) -> double {
    if (how == 2) return p.rest[(size_t)row * p.pieces + c];
    if (how == 1) {   // recomputed where a token is gone
      bool hit = false;
      for (int k = next_child(p, s, at, at + 1); k < s.n; k = next_child(p, s, at, k + 1)) {
        const int token = p.d.tokens[s.first + k];
        hit = hit || (token >= 0 && token / kPiece == c);
      }
      if (hit) {
        double w[kEach], sum = 0.0;
        weights(c, w);
#pragma unroll
        for (int j = 0; j < kEach; ++j) sum += w[j];
        return block_sum<kWalkThreads>(sum, scratch);
      }
    }
    const PieceSum q = p.sums[(size_t)row * p.pieces + c];
    return q.top == -INFINITY ? 0.0 : q.sum * weight_of(q.top, r.top, per) / r.sum;
  };
  double all = 0.0;
  for (int c = 0; c < p.pieces; ++c) all += piece_sum(c);
  if (!(all > 0.0) && how > 0) {
    how = 0;
    for (int c = 0; c < p.pieces; ++c) all += piece_sum(c);
  }
  const double want = uniform_of(p, s.first) * all;
  int piece = -1;
  double before = 0.0, sum = 0.0;
  for (int c = 0; c < p.pieces; ++c) {
    const double mine = piece_sum(c);
    if (mine > 0.0) {   // (the last one with anything, if rounding leaves `want` at the sum of all)
      if (piece >= 0) before = sum;
      piece = c;
    }
    sum += mine;
    if (sum > want) break;
  }
  if (piece < 0) {
    if (threadIdx.x == 0) *out = -1;
    return;
  }
  double w[kEach], mine = 0.0;
  weights(piece, w);
#pragma unroll
  for (int j = 0; j < kEach; ++j) mine += w[j];
  double upto = mine;   // inclusive running sum over the wave's lanes
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double other = __shfl_up(upto, m, 64);
    if (lane >= m) upto += other;
  }
  if (lane == 63) wave_at[wave] = upto;
  if (threadIdx.x == 0) said[3] = -1;
  __syncthreads();
  double start = before;
  for (int k = 0; k < wave; ++k) start += wave_at[k];
  start += upto - mine;
  // the first element whose running sum is above `want`; if rounding leaves none, the last one that has a weight
  int first = INT32_MAX, last = -1;
  double run = start;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    run += w[j];
    if (w[j] > 0.0) {
      last = piece * kPiece + (int)threadIdx.x * kEach + j;
      if (run > want) first = min(first, last);
    }
  }
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) first = min(first, __shfl_xor(first, m, 64)), last = max(last, __shfl_xor(last, m, 64));
  __syncthreads();
  int* const firsts = reinterpret_cast<int*>(scratch);   // (two ints an element)
  if (lane == 0) firsts[2 * wave] = first, firsts[2 * wave + 1] = last;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 0; k < kWaves; ++k) first = min(first, firsts[2 * k]), last = max(last, firsts[2 * k + 1]);
    *out = first != INT32_MAX ? first : last;
  }
}

VerifyArgs args_of(const ave_fp4_draft& d, void* ws, size_t* bytes) {
  VerifyArgs p{};
  p.d = d;
  p.pieces = (d.vocab + kPiece - 1) / kPiece;
  char* at = static_cast<char*>(ws);
  size_t used = 0;
  const auto take = [&](size_t n) {
    char* r = at + used;
    used += (n + 255) / 256 * 256;
    return r;
  };
  const size_t all = (size_t)d.rows * p.pieces;
  p.sums = reinterpret_cast<PieceSum*>(take(all * sizeof(PieceSum)));
  if (d.draft_probs) {
    p.rest = reinterpret_cast<double*>(take(all * sizeof(double)));
    p.times = reinterpret_cast<double*>(take((size_t)d.rows * sizeof(double)));
    p.choice = reinterpret_cast<int*>(take((size_t)d.rows * sizeof(int)));
  }
  if (bytes) *bytes = used;
  return p;
}

template <bool F32>
hipError_t launch(const VerifyArgs& p, hipStream_t s) {
  const int rows = p.d.rows;
  const dim3 each((unsigned)p.pieces * (unsigned)rows);
  if (rows > 0) hipLaunchKernelGGL((row_sums_kernel<F32>), each, dim3(kRowThreads), 0, s, p);
  if (rows > 0 && p.d.draft_probs) {
    hipLaunchKernelGGL((rest_sums_kernel<F32>), each, dim3(kRowThreads), 0, s, p);
    hipLaunchKernelGGL((children_kernel<F32>), dim3((unsigned)rows), dim3(kWalkThreads), 0, s, p);
  }
  hipLaunchKernelGGL((walk_kernel<F32>), dim3((unsigned)p.d.batch), dim3(kWalkThreads), 0, s, p);
  return hipGetLastError();
}

}  // namespace

size_t verify_draft_workspace_bytes(const ave_fp4_draft& d) {
  size_t bytes = 0;
  args_of(d, nullptr, &bytes);
  return bytes;
}

hipError_t launch_verify_draft(const ave_fp4_draft& d, void* workspace, hipStream_t s) {
  const VerifyArgs p = args_of(d, workspace, nullptr);
  return d.logits_f32 ? launch<true>(p, s) : launch<false>(p, s);
}

}  // namespace ave
