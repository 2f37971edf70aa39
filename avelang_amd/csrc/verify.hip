// Which nodes of a drafted tree the target model accepts, and the token behind them.
//
//   row sums   a workgroup for a piece of a row: largest logit, its lowest index, sum of exp((x - largest) / temperature)
//   children   (drafts with distributions only) rows whose first child is rejected and that have more: sums of max(p - t q, 0), child after child
//   way        a wave goes from node to node: whether a node is accepted, once its parent is and its elder siblings are not, does not depend on the rest
//              of the way, so the probabilities of 64 nodes are fetched at once, a lane each
//   left sums  what pieces of the last node's row leave to draw from, in fp64
//   draw       the piece in which the random number lies, then the element
//
// With little to read the last three are one launch, whose workgroups find the way each by itself.  With much, the children of node 0 are decided on first,
// from its row alone, and then only rows that descend from the accepted one are read.
//
// Bound by HBM where there is much to read: 64 trees of 16 nodes, 131072 tokens in bf16, 63 us of which 23 are the wanted 377 of 1024 rows at 4.2 TB/s
// (all rows at 4.9 TB/s would be 55); else by the way from one launch to the next and by chains of loads: six nodes of 32768 tokens 9 us; eight chains of six
// with distributions, 50001 tokens, 23.  The fp64 sums over 64 rows of 131072 take 14 us, of which vector instructions are 8 (38 an element, 17 of them in fp64, at
// four cycles a wave); the rest are the launch's start and end and waits for the row.
//
// Rejections with distributions: r_0 = p, r_(k+1) = max(r_k - q, 0) / sum is max(p - t_k q, 0) / s_k with t_0 = 0, s_0 = 1, t_(k+1) = t_k + s_k and
// s_k = sum max(p - t_k q, 0), so that a row needs its logits, q and two numbers.
//
// Precision.  A token is drawn by where a number lies among the running sums of 10^5 probabilities; in fp32 one draw in some hundred to
// thousand would go to a neighbour by rounding, so what is drawn from is summed in fp64, and with distributions the row sums are, too.  Without, a node's
// acceptance is one comparison: the row sums behind it are formed in fp32 (kSumError), and where the comparison comes out nearer than that, the row
// is summed again in fp64.  Probabilities are exact to 2^-42 of themselves, so a remainder that rejections leave is exact to 2^-42 of p: one to which they come with a
// probability of 2^-40 is not told from rounding.
#include <algorithm>

#include "fp4_common.hpp"
#include "kernels.hpp"
#include "kv_cache.hpp"

namespace ave {
namespace {

constexpr int kPiece = kVocabPiece;
constexpr int kThreads = 256, kOnce = 8;          // elements of a thread that are together in memory
constexpr int kShort = kThreads * kOnce;           // elements that a workgroup draws from

struct PieceSum {
  double sum;   // of exp((x - top) / temperature)
  float top;    // -inf: no number
  int at;       // the lowest index of top
};
constexpr int kGone = 16;
// What a sequence's token is drawn from
struct Draw {
  double times;   // t of max(p - t q, 0)
  double sum;     // of the row, in units of its largest weight
  float top;
  int gone[kGone], many;   // the children's tokens, so many; -1: more, to be looked for
  int row, how, out;       // out: of `emitted`; how: kAll: p, kWithout: p without the children's tokens, kRest: max(p - t q, 0); kNothing: the token is there already
};
enum { kAll, kWithout, kRest, kNothing };
constexpr int kMany = -2;

struct Wanted {
  double per;   // inverse temperature
  int row;
};

struct VerifyArgs {
  ave_fp4_draft d;
  int pieces, shorts;   // of kPiece and of kShort elements
  PieceSum* sums;   // [rows][pieces]
  double* left;     // [batch][shorts]: sums of what is drawn from
  Draw* draws;      // [batch]
  double* rest;     // [rows][pieces]: sums of max(p - q, 0)
  double* times;    // [rows]: t when all children are rejected
  int* choice;      // [rows]: the accepted child, -1: none; kMany: there are several and nobody has looked
  Wanted* wanted;   // [rows]: the rows that descend from the accepted children of nodes 0, in any order, and
  int* many;        // how many
  int* done;        // [batch]: pieces of the last row that are summed up; with distributions also [rows] behind that: pieces of `rest`
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
__device__ inline int uniform_int(int x) { return __builtin_amdgcn_readfirstlane(x); }
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
  const Span s = span_of(p, uniform_int(from));
  return row >= s.first && row < s.first + s.n ? uniform_int(from) : -1;
}
// 1 / temperature in units of log2(e); 0: the largest logit
__device__ inline double inverse_temperature(const VerifyArgs& p, int b) {
  const float t = p.d.temperature ? p.d.temperature[b] : 1.0f;
  return t > 0.0f ? 1.4426950408889634 / (double)fminf(t, 3.402823466e38f) : 0.0;
}

// exp((x - top) / temperature) for x <= top.  2^y = 2^n 2^f with n the nearest integer (out of the low bits of y + 1.5 2^52) and the Taylor
// polynomial of 2^f, |f| <= 1/2, whose first missing term is 2^-42 of it; 2^n by adding to the exponent.  0 for -inf, and for what is below 2^-1020, next to where
// numbers of 64 bits end: a finite mask leaves nothing.
__device__ inline double weight_of(float x, double top, double per) {
  constexpr double kRound = 6755399441055744.0;
  const double y = ((double)x - top) * per, up = y + kRound, f = y - (up - kRound);
  double r = 7.0549116208011233e-9;   // (ln 2)^k / k!
  r = fma(r, f, 1.0178086009239699e-7);
  r = fma(r, f, 1.3215486790144307e-6);
  r = fma(r, f, 1.5252733804059841e-5);
  r = fma(r, f, 1.5403530393381609e-4);
  r = fma(r, f, 1.3333558146428443e-3);
  r = fma(r, f, 9.6181291076284772e-3);
  r = fma(r, f, 5.5504108664821580e-2);
  r = fma(r, f, 0.24022650695910071);
  r = fma(r, f, 0.69314718055994531);
  r = fma(r, f, 1.0);
  const uint64_t bits = __builtin_bit_cast(uint64_t, r) + ((uint64_t)(unsigned)__builtin_bit_cast(uint64_t, up) << 52);
  return y >= -1020.0 ? __builtin_bit_cast(double, bits) : 0.0;
}

// A NaN counts as -inf, infinity as the largest number.  (The lesser of a NaN and a number is the number: a NaN has to be told apart by itself.)
__device__ inline float number(float x) { return x == x ? fminf(x, 3.402823466e38f) : -INFINITY; }
template <bool F32>
__device__ inline float logit(const VerifyArgs& p, int row, int i) {
  if constexpr (F32) return static_cast<const float*>(p.d.logits)[(int64_t)row * p.d.logits_stride + i];
  else return __builtin_bit_cast(float, (unsigned)static_cast<const uint16_t*>(p.d.logits)[(int64_t)row * p.d.logits_stride + i] << 16);
}
// Eight consecutive logits from index i on as they are in memory, -inf behind the last
template <bool F32>
struct Eight {
  int word[F32 ? 8 : 4];
};
template <bool F32>
__device__ inline Eight<F32> load8(const VerifyArgs& p, int row, int i) {
  typedef int Four __attribute__((ext_vector_type(4), aligned(2)));   // (rows of an odd vocabulary start anywhere)
  const char* from = static_cast<const char*>(p.d.logits) + ((int64_t)row * p.d.logits_stride + i) * (F32 ? 4 : 2);
  Eight<F32> r;
  if (i + kOnce <= p.d.vocab) {
#pragma unroll
    for (int k = 0; k < (F32 ? 2 : 1); ++k) {
      const Four x = reinterpret_cast<const Four*>(from)[k];
#pragma unroll
      for (int e = 0; e < 4; ++e) r.word[4 * k + e] = x[e];
    }
  } else {
#pragma unroll
    for (int k = 0; k < kOnce; ++k) {
      const int x = __builtin_bit_cast(int, i + k < p.d.vocab ? logit<F32>(p, row, i + k) : -INFINITY);
      if constexpr (F32) r.word[k] = x;
      else r.word[k / 2] = k % 2 ? r.word[k / 2] | x : (int)((unsigned)x >> 16);
    }
  }
  return r;
}
template <bool F32>
__device__ inline void unpack(const Eight<F32>& r, float (&x)[kOnce]) {
#pragma unroll
  for (int k = 0; k < kOnce; ++k) {
    if constexpr (F32) x[k] = __builtin_bit_cast(float, r.word[k]);
    else x[k] = __builtin_bit_cast(float, k % 2 ? (unsigned)r.word[k / 2] & 0xFFFF0000u : (unsigned)r.word[k / 2] << 16);
  }
}
template <bool F32>
__device__ inline void logits(const VerifyArgs& p, int row, int i, float (&x)[kOnce]) {
  unpack<F32>(load8<F32>(p, row, i), x);
}
__device__ inline double draft_prob(const VerifyArgs& p, int row, int i) {
  const float q = p.d.draft_probs[(int64_t)row * p.d.draft_probs_stride + i];
  return q > 0.0f ? (double)q : 0.0;
}
__device__ inline void draft_probs(const VerifyArgs& p, int row, int i, float (&q)[kOnce]) {   // eight, 0 behind the last
  typedef float Four __attribute__((ext_vector_type(4), aligned(4)));
  const float* from = p.d.draft_probs + (int64_t)row * p.d.draft_probs_stride + i;
  if (i + kOnce <= p.d.vocab) {
    const Four a = reinterpret_cast<const Four*>(from)[0], b = reinterpret_cast<const Four*>(from)[1];
#pragma unroll
    for (int k = 0; k < kOnce; ++k) q[k] = k < 4 ? a[k] : b[k - 4];
  } else {
#pragma unroll
    for (int k = 0; k < kOnce; ++k) q[k] = i + k < p.d.vocab ? from[k] : 0.0f;
  }
}
__device__ inline double random_of(const VerifyArgs& p, int row) {
  const float u = p.d.uniform[row];
  return u > 0.0f ? fmin((double)u, 1.0) : 0.0;
}

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

// ---- over a wave, over a workgroup ---------------------------------------------------------------------------------------------------------
__device__ inline double wave_sum(double v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}
__device__ inline double lane_double(double v, int lane) {   // lane: the same in all lanes
  const uint64_t x = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)x, lane) |
                                        (uint64_t)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(x >> 32), lane) << 32);
}
// of every thread's v, in all threads; `scratch` has an element a wave
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

// ---- a row's sums ----------------------------------------------------------------------------------------------------------------------------
// The relative error of a row's sum in fp32: a difference and a product of a rounding each before an exponential of an argument down to -126 (3 2^-24 126
// ln 2), the exponential's own and 32 additions (2^-23, 2^-19): 1.8e-5 at most.
constexpr double kSumError = 1.0 / 32768.0;

// EXACT: in fp64.  ROWS: 0 all, 1 the first of each sequence, 2 those that are wanted (by a workgroup one after the other)
template <bool F32, bool EXACT, int ROWS>
__global__ __launch_bounds__((EXACT ? 2 : 1) * kThreads) void row_sums_kernel(VerifyArgs p) {
  constexpr int THREADS = (EXACT ? 2 : 1) * kThreads, kEach = kPiece / THREADS;
  __shared__ double scratch[THREADS / 64];
  __shared__ float tops[THREADS / 64];
  __shared__ int lowest;
  if constexpr (ROWS < 2) {   // for the launches behind this one
    const unsigned counts = (unsigned)p.d.batch + (EXACT ? (unsigned)p.d.rows : 0u);
    for (unsigned i = blockIdx.x * THREADS + threadIdx.x; i < counts; i += gridDim.x * THREADS) p.done[i] = 0;
    if (ROWS == 1 && blockIdx.x == 0 && threadIdx.x == 0) *p.many = 0;
  }
  const unsigned all = ROWS == 2 ? (unsigned)min(*p.many, p.d.rows) * (unsigned)p.pieces : blockIdx.x + 1;
  Wanted now{};
  Eight<F32> next[kEach / kOnce];
  const auto fetch = [&](unsigned item) {
    now = p.wanted[item / (unsigned)p.pieces];
#pragma unroll
    for (int k = 0; k < kEach / kOnce; ++k) next[k] = load8<F32>(p, now.row, (int)(item % (unsigned)p.pieces) * kPiece + (k * THREADS + threadIdx.x) * kOnce);
  };
  if (ROWS == 2 && blockIdx.x < all) fetch(blockIdx.x);
  for (unsigned item = blockIdx.x; item < all; item += gridDim.x) {
    const int piece = (int)(item % (unsigned)p.pieces);
    int row = (int)(item / (unsigned)p.pieces), b = row;
    if constexpr (ROWS == 1) {
      const Span s = span_of(p, b);
      if (s.n == 0) return;
      row = s.first;
    }
    double per;
    float x[kEach / kOnce][kOnce];
    if constexpr (ROWS == 2) {   // the present row's are here, the next one's under way
      row = now.row, per = now.per;
#pragma unroll
      for (int k = 0; k < kEach / kOnce; ++k) unpack<F32>(next[k], x[k]);
      if (item + gridDim.x < all) fetch(item + gridDim.x);
    } else {
#pragma unroll
      for (int k = 0; k < kEach / kOnce; ++k) next[k] = load8<F32>(p, row, piece * kPiece + (k * THREADS + threadIdx.x) * kOnce);   // all under way
      if constexpr (ROWS == 0) b = sequence_of(p, row);
      if (b < 0) return;
      per = inverse_temperature(p, b);
#pragma unroll
      for (int k = 0; k < kEach / kOnce; ++k) unpack<F32>(next[k], x[k]);
    }
    if (threadIdx.x == 0) lowest = INT32_MAX;
    float top;
    double sum;
    const auto reduce = [&] {
      float mine = -INFINITY;
#pragma unroll
      for (int k = 0; k < kEach; ++k) mine = fmaxf(mine, x[k / kOnce][k % kOnce]);
      top = mine;
#pragma unroll
      for (int m = 32; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
      if ((threadIdx.x & 63) == 0) tops[threadIdx.x / 64] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < THREADS / 64; ++w) top = fmaxf(top, tops[w]);
      sum = 0.0;
      if (per > 0.0 && top != -INFINITY) {
        if constexpr (EXACT) {
#pragma unroll
          for (int k = 0; k < kEach; ++k) sum += weight_of(x[k / kOnce][k % kOnce], top, per);
        } else {
          const float per32 = (float)fmin(per, 3.4e38);
          float s = 0.0f;
#pragma unroll
          for (int k = 0; k < kEach; ++k) s += __builtin_amdgcn_exp2f((x[k / kOnce][k % kOnce] - top) * per32);
          sum = (double)s;
        }
      }
      sum = block_sum<THREADS>(sum, scratch);
      return mine;
    };
    float mine = reduce();
    if (!(sum < 1e300) || top == INFINITY) {   // a NaN or an infinity in the piece
#pragma unroll
      for (int k = 0; k < kEach; ++k) x[k / kOnce][k % kOnce] = number(x[k / kOnce][k % kOnce]);
      mine = reduce();
    }
    if (mine == top) {
      int at = INT32_MAX;
#pragma unroll
      for (int k = kEach - 1; k >= 0; --k)
        if (x[k / kOnce][k % kOnce] == top) at = piece * kPiece + (k / kOnce * THREADS + threadIdx.x) * kOnce + k % kOnce;
      atomicMin(&lowest, at);
    }
    __syncthreads();
    if (threadIdx.x == 0) p.sums[(size_t)row * p.pieces + piece] = {sum, top, lowest};
    if constexpr (ROWS == 2) __syncthreads();   // before the next one's `lowest`
    if (EXACT && piece == 0 && threadIdx.x < 64) {   // (with distributions)
      const Span s = span_of(p, b);
      const int v = row - s.first, child = next_child(p, s, v, v + 1);
      const bool several = child < s.n && next_child(p, s, v, child + 1) < s.n;
      if (threadIdx.x == 0) p.choice[row] = several && per > 0.0 ? kMany : -1;
    }
  }
}

struct RowSum {
  double sum;
  float top;
  int at;
};
// Of the rows that the lanes name (-1: none), each in its lane, by a wave; exact: in fp64.  A row's sum depends on its pieces alone, bit for bit.
__device__ inline RowSum sums_of_rows(const VerifyArgs& p, int row, double per, bool exact) {
  RowSum mine{0.0, -INFINITY, INT32_MAX};
  if (!exact) {   // a row a lane, sixteen pieces at a time under way
    const float per32 = (float)fmin(per, 3.4e38);
#pragma unroll 1
    for (int c0 = 0; row >= 0 && c0 < p.pieces; c0 += 16) {
      PieceSum q[16];
#pragma unroll
      for (int c = 0; c < 16; ++c) q[c] = p.sums[(size_t)row * p.pieces + min(c0 + c, p.pieces - 1)];
      float top = mine.top;
#pragma unroll
      for (int c = 0; c < 16; ++c) top = fmaxf(top, q[c].top);
      if (top == -INFINITY) continue;
      const auto scale = [&](float x) { return x == -INFINITY ? 0.0 : (double)__builtin_amdgcn_exp2f((x - top) * per32); };
      if (mine.top != top) {
        mine.sum *= scale(mine.top);
#pragma unroll
        for (int c = 15; c >= 0; --c) mine.at = q[c].top == top ? q[c].at : mine.at;
      }
      mine.top = top;
#pragma unroll
      for (int c = 0; c < 16; ++c) mine.sum += c0 + c < p.pieces ? q[c].sum * scale(q[c].top) : 0.0;
    }
    if (!(per > 0.0)) mine.sum = 0.0;
    return mine;
  }
  // a piece a lane, the lanes of a row next to each other, as many rows at a time as that leaves (with a row a lane up to sixteen exponentials of 25 dependent
  // instructions follow each other: eight chains of six with distributions, 50001 tokens, 24.3 us that way, 23.3 this way)
  const int lane = threadIdx.x & 63, wide = p.pieces >= 64 ? 64 : p.pieces > 1 ? 1 << (32 - __clz(p.pieces - 1)) : 1, at_once = 64 / wide;
  const auto of_round = [&](int r0) { return __shfl(row, min(r0 + lane / wide, 63), 64); };
  const auto fetch = [&](int of, int c) { return of >= 0 && c < p.pieces ? p.sums[(size_t)of * p.pieces + c] : PieceSum{0.0, -INFINITY, INT32_MAX}; };
  const auto scale = [&](float x, float top) { return x == -INFINITY ? 0.0 : weight_of(x, top, per); };
  const uint64_t named = __ballot(row >= 0);
  const int end = named ? 64 - __clzll((long long)named) : 0;
  int of = of_round(0);
  PieceSum next = fetch(of, lane % wide);
#pragma unroll 1
  for (int r0 = 0; r0 < end; r0 += at_once) {
    PieceSum q = next;
    const int now = of;
    of = of_round(r0 + at_once);
    if (r0 + at_once < end) next = fetch(of, lane % wide);
#pragma unroll 1
    for (int c = lane % wide + 64; c < p.pieces; c += 64) {   // (more than 64 pieces: 524288 tokens)
      const PieceSum more = fetch(now, c);
      const float top = fmaxf(q.top, more.top);
      q.at = more.top > q.top ? more.at : q.at;
      if (per > 0.0) q.sum = q.sum * scale(q.top, top) + more.sum * scale(more.top, top);
      q.top = top;
    }
    float top = q.top;
#pragma unroll 1
    for (int m = wide / 2; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
    double sum = per > 0.0 ? q.sum * scale(q.top, top) : 0.0;
    int at = q.top == top && top != -INFINITY ? q.at : INT32_MAX;
#pragma unroll 1
    for (int m = wide / 2; m > 0; m >>= 1) {
      sum += __shfl_xor(sum, m, 64);
      at = min(at, __shfl_xor(at, m, 64));
    }
    const int from = (lane - r0) * wide;   // where this lane's row is, in its round
    sum = __shfl(sum, from & 63, 64), top = __shfl(top, from & 63, 64), at = __shfl(at, from & 63, 64);
    if (lane >= r0 && lane < r0 + at_once) mine = {sum, top, at};
  }
  return mine;
}
// Largest logit and its lowest index, by a wave
__device__ inline RowSum row_top(const VerifyArgs& p, int row) {
  const PieceSum* s = p.sums + (size_t)row * p.pieces;
  RowSum r{0.0, -INFINITY, INT32_MAX};
  for (int c = threadIdx.x & 63; c < p.pieces; c += 64)
    if (s[c].top > r.top) r.top = s[c].top, r.at = s[c].at;
  float top = r.top;
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
  if (r.top != top || top == -INFINITY) r.at = INT32_MAX;
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) r.at = min(r.at, __shfl_xor(r.at, m, 64));
  r.top = top;
  return r;
}
// Sum of a row in fp64, by a wave
template <bool F32>
__device__ inline double exact_sum(const VerifyArgs& p, int row, float top, double per) {
  double sum = 0.0;
  for (int i = (threadIdx.x & 63) * kOnce; i < p.d.vocab; i += 64 * kOnce) {
    float x[kOnce];
    logits<F32>(p, row, i, x);
#pragma unroll
    for (int k = 0; k < kOnce; ++k) sum += weight_of(number(x[k]), top, per);
  }
  return wave_sum(sum);
}

__device__ inline RowSum of_lane(const RowSum& r, int lane) {   // lane: the same in all lanes
  return {lane_double(r.sum, lane), __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, r.top), lane)), __builtin_amdgcn_readlane(r.at, lane)};
}

// ---- the way through the tree ------------------------------------------------------------------------------------------------------------------
struct Way {
  int at, kept, tried, token;   // the last node, how many are kept, how many of its children were rejected; temperature 0: the token
  double times;                 // with distributions: t
  RowSum row;                   // of the last node (FIRST: of lanes' nodes)
};
// By one wave.  FIRST: one step only (at: the accepted child of node 0, or 0).  write: this workgroup writes path and emitted.  draw: where the tokens of the
// last node's children go.
template <bool F32, bool FIRST>
__device__ inline Way walk(const VerifyArgs& p, const Span& s, double per, bool write, Draw* draw = nullptr) {
  const int lane = threadIdx.x & 63;
  const bool probs = p.d.draft_probs != nullptr;
  Way w{0, 1, 0, -1, 0.0, {0.0, -INFINITY, INT32_MAX}};
  double taken = 0.0;   // by rejected children, of the present row
  write = write && lane == 0;
  if (write) p.d.path[s.first] = 0;
  // Up to 64 nodes all rows' sums are on their way, a node a lane, while it is looked up whose children the nodes are
  const bool few = s.n <= 64;
  if (few) w.row = sums_of_rows(p, lane < (FIRST ? 1 : s.n) ? s.first + lane : -1, per, probs);
  for (int c0 = 0; c0 < s.n; c0 += 64) {
    // a node a lane: its parent's row, what the target gives its token, what the draft gave it
    const int j = c0 + lane;
    int parent = -1, token = -1;
    double u = 0.0, mine = 0.0, q = 0.0;
    RowSum r{0.0, -INFINITY, INT32_MAX};
    if (j < s.n && j > 0) parent = p.d.parents[s.first + j], token = p.d.tokens[s.first + j];
    if (parent >= j) parent = -1;
    bool there = false;
    float x = -INFINITY;
    if (parent >= w.at && (!FIRST || parent == 0)) {
      const int row = s.first + parent;
      u = random_of(p, s.first + j);
      there = token >= 0 && token < p.d.vocab;
      if (there) x = logit<F32>(p, row, token);
      if (there && probs) q = draft_prob(p, row, token);
    }
    if (few) {
      const int from = parent > 0 ? parent : 0;
      r = {__shfl(w.row.sum, from, 64), __shfl(w.row.top, from, 64), __shfl(w.row.at, from, 64)};
    } else {
      r = sums_of_rows(p, parent >= w.at && (!FIRST || parent == 0) ? s.first + parent : -1, per, probs);
    }
    if (parent >= w.at && (!FIRST || parent == 0)) {   // (the others cannot be reached)
      if (per > 0.0) mine = r.sum > 0.0 ? weight_of(there ? number(x) : -INFINITY, r.top, per) / r.sum : 0.0;
      if (!there) token = -1;
    } else {
      parent = -1;
    }
    uint64_t mask = __ballot(parent == w.at);
    while (mask) {
      const int k = __ffsll((unsigned long long)mask) - 1, child = c0 + k, child_token = __builtin_amdgcn_readlane(token, k);
      mask &= mask - 1;
      bool accepted = false;
      const double p_child = lane_double(mine, k), u_child = lane_double(u, k);
      if (per == 0.0) {
        accepted = child_token >= 0 && child_token == __builtin_amdgcn_readlane(r.at, k);
      } else if (probs) {
        if (w.tried == 0) {
          accepted = child_token >= 0 && u_child * lane_double(q, k) < p_child;
        } else {   // by children_kernel
          const int chosen = p.choice[s.first + w.at];
          if (chosen > w.at && chosen < s.n) {   // this child or a later one
            if (chosen > child) continue;
            accepted = chosen == child;
          }
        }
      } else if (child_token >= 0) {   // a token that an elder sibling had has been taken out
        bool again = __any(lane < k && parent == w.at && token == child_token);
        for (int b0 = w.at + 1; b0 < c0 && !again; b0 += 64)
          again = __any(b0 + lane < c0 && p.d.parents[s.first + b0 + lane] == w.at && p.d.tokens[s.first + b0 + lane] == child_token);
        if (!again) {
          const double bound = u_child * (1.0 - taken);
          double now = p_child, against = bound;
          if (fabs(bound - p_child) <= kSumError * (bound + p_child + u_child * taken)) {
            // nearer than the row's sum is exact: all of it again, over the same tokens
            const int row = s.first + w.at;
            const RowSum of_row = row_top(p, row);
            const double sum = exact_sum<F32>(p, row, of_row.top, per);
            double gone = 0.0;
            for (int b0 = w.at + 1; b0 < child; b0 += 64) {
              const int c = b0 + lane;
              const int t = c < child && p.d.parents[s.first + c] == w.at ? p.d.tokens[s.first + c] : -1;
              bool first = t >= 0 && t < p.d.vocab;
              for (int e = w.at + 1; first && e < c; ++e) first = p.d.parents[s.first + e] != w.at || p.d.tokens[s.first + e] != t;
              gone += wave_sum(first ? weight_of(number(logit<F32>(p, row, t)), of_row.top, per) / sum : 0.0);
            }
            now = weight_of(number(logit<F32>(p, row, child_token)), of_row.top, per) / sum;
            against = u_child * (1.0 - gone);
          }
          accepted = against < now && now > 0.0 && u_child < 1.0;   // (no r is above 1; `against` may be off by the last bit of a sum of 1)
          if (!accepted) taken += p_child;
        }
      }
      if (accepted) {
        if (write) p.d.path[s.first + w.kept] = child, p.d.emitted[s.first + w.kept - 1] = child_token;
        w.at = child, ++w.kept, w.tried = 0, taken = 0.0;
        if constexpr (FIRST) return w;
        mask = __ballot(parent == w.at && lane > k);
      } else {
        ++w.tried;
      }
    }
    if (!FIRST && s.n <= 64) {
      const uint64_t children = __ballot(parent == w.at && token >= 0);
      const int many = __popcll(children), to = __popcll(children & ((1ull << lane) - 1));
      if (many <= kGone && (children >> lane & 1)) draw->gone[to] = token;
      if (lane == 0) draw->many = many <= kGone ? many : -1;
    }
  }
  if (!FIRST && s.n > 64 && lane == 0) draw->many = -1;
  if (!FIRST && !few) w.row = sums_of_rows(p, lane == 0 ? s.first + w.at : -1, per, probs);
  if (!FIRST) w.row = of_lane(w.row, few ? w.at : 0);
  if (probs && per > 0.0) w.times = w.tried > 1 ? p.times[s.first + w.at] : (double)w.tried;   // (p.times is there with distributions only)
  return w;
}

// With much to read: which rows are wanted after node 0's
template <bool F32>
__global__ __launch_bounds__(64) void first_step_kernel(VerifyArgs p) {
  const int b = blockIdx.x;
  const Span s = span_of(p, b);
  if (s.n == 0) return;
  const double per = inverse_temperature(p, b);
  const int top = walk<F32, true>(p, s, per, false).at;
  for (int i = threadIdx.x; i < s.n; i += 64) {
    int at = i;   // up to the accepted child, or past it
    while (at > top) {
      const int up = p.d.parents[s.first + at];
      at = up < at ? up : -1;
    }
    const uint64_t mine = __ballot(top > 0 && at == top);   // (the wave's lanes that are here: the first ones)
    if (mine) {
      const int lane = threadIdx.x;
      int to = 0;
      if (lane == 0) to = atomicAdd(p.many, __popcll(mine));
      to = uniform_int(to) + __popcll(mine & ((1ull << lane) - 1));
      if ((mine >> lane & 1) && to >= 0 && to < p.d.rows) p.wanted[to] = {per, s.first + i};
    }
  }
}

// Elements i .. i + 7 of what is drawn from: what they are made of, to be asked for before any is used,
template <bool F32>
struct Source {
  Eight<F32> x;
  float q[kOnce];
};
template <bool F32>
__device__ inline Source<F32> source_of(const VerifyArgs& p, const Draw& d, int i) {
  Source<F32> r;
  r.x = load8<F32>(p, d.row, i);
  if (d.how == kRest) draft_probs(p, d.row, i, r.q);
  return r;
}
// and they, in units of the row's largest weight (kRest: of 1).  By whole waves, whose lanes' elements follow each other.
template <bool F32>
__device__ inline void weights_of(const VerifyArgs& p, const Span& s, const Draw& d, double per, int i, const Source<F32>& from, double (&w)[kOnce]) {
  float x[kOnce];
  unpack<F32>(from.x, x);
#pragma unroll
  for (int j = 0; j < kOnce; ++j) w[j] = weight_of(number(x[j]), d.top, per);
  if (d.how == kRest) {
    const double over = 1.0 / d.sum;
#pragma unroll
    for (int j = 0; j < kOnce; ++j) w[j] = fmax(w[j] * over - d.times * (from.q[j] > 0.0f ? (double)from.q[j] : 0.0), 0.0);
  }
  if (d.how == kWithout) {
    const int first = uniform_int(i);
    const auto without = [&](int token) {
      if ((unsigned)token - (unsigned)first >= 64u * kOnce) return;   // none of this wave's
#pragma unroll
      for (int j = 0; j < kOnce; ++j)
        w[j] = token - i == j ? 0.0 : w[j];
    };
    if (d.many >= 0) {
      for (int c = 0; c < d.many; ++c) without(d.gone[c]);
    } else {
      const int at = d.row - s.first;
      for (int c = next_child(p, s, at, at + 1); c < s.n; c = next_child(p, s, at, c + 1)) without(p.d.tokens[s.first + c]);
    }
  }
}

// Inclusive running sum over the wave's lanes
__device__ inline double wave_running(double v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double other = __shfl_up(v, m, 64);
    if ((threadIdx.x & 63) >= m) v += other;
  }
  return v;
}
// The next token, by a workgroup, whose threads share the kShort elements among which it lies
template <bool F32>
__device__ inline void draw_token(const VerifyArgs& p, const Span& s, const Draw& of, double per, double random, int b) {
  __shared__ double wave_at[kThreads / 64];
  __shared__ int firsts[kThreads / 64], lasts[kThreads / 64];
  __shared__ Draw all_of_it;
  const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  bool nothing_left = false;
  const auto piece_sum = [&](int c) -> double { return c < p.shorts ? p.left[(size_t)b * p.shorts + c] : 0.0; };
  // every wave: pieces a lane, 64 at a time
  double mine0, upto0;   // of the first 64
  const auto sum_of_all = [&] {
    mine0 = piece_sum(lane), upto0 = wave_running(mine0);
    double sum = lane_double(upto0, 63);
    for (int c0 = 64; c0 < p.shorts; c0 += 64) sum += lane_double(wave_running(piece_sum(c0 + lane)), 63);
    return sum;
  };
  double all = sum_of_all();
  if (!(all > 0.0)) {   // nothing is left: all of the row, summed up here
    nothing_left = true;
    __syncthreads();
    if (threadIdx.x == 0) {
      all_of_it = of;
      all_of_it.how = kAll;
    }
    __syncthreads();
    for (int c = 0; c < p.shorts; ++c) {
      double w[kOnce], sum = 0.0;
      const int i = c * kShort + (int)threadIdx.x * kOnce;
      weights_of<F32>(p, s, all_of_it, per, i, source_of<F32>(p, all_of_it, i), w);
#pragma unroll
      for (int j = 0; j < kOnce; ++j) sum += w[j];
      sum = block_sum<kThreads>(sum, wave_at);
      if (threadIdx.x == 0) p.left[(size_t)b * p.shorts + c] = sum;
    }
    __threadfence();
    __syncthreads();
    all = sum_of_all();
  }
  const double want = random < 1.0 ? random * all : INFINITY;   // (no sum is above the whole, nor does rounding make one)
  int piece = 0;
  double before = 0.0, sum = 0.0;   // before: the sum of the pieces in front
  for (int c0 = 0; c0 < p.shorts; c0 += 64) {
    const double mine = c0 == 0 ? mine0 : piece_sum(c0 + lane), upto = c0 == 0 ? upto0 : wave_running(mine);
    const uint64_t some = __ballot(mine > 0.0), over = __ballot(mine > 0.0 && sum + upto > want);
    if (some) {   // (the last one with anything, if rounding leaves `want` at the sum of all)
      const int k = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)some);
      piece = c0 + k, before = sum + lane_double(upto, k) - lane_double(mine, k);
    }
    if (over) break;
    sum += lane_double(upto, 63);
  }
  const Draw& d = nothing_left ? all_of_it : of;
  double w[kOnce], mine = 0.0;
  const int i = piece * kShort + (int)threadIdx.x * kOnce;
  weights_of<F32>(p, s, d, per, i, source_of<F32>(p, d, i), w);
#pragma unroll
  for (int j = 0; j < kOnce; ++j) mine += w[j];
  const double upto = wave_running(mine);
  if (lane == 63) wave_at[wave] = upto;
  __syncthreads();
  double run = before;
  for (int k = 0; k < wave; ++k) run += wave_at[k];
  run += upto - mine;
  // the first element whose running sum is above `want`; if rounding leaves none, the last one that has a weight
  int first = -1, last = -1;
#pragma unroll
  for (int j = 0; j < kOnce; ++j) {
    run += w[j];
    if (w[j] > 0.0) {
      last = piece * kShort + (int)threadIdx.x * kOnce + j;
      if (run > want && first < 0) first = last;
    }
  }
  const uint64_t over = __ballot(first >= 0), some = __ballot(last >= 0);
  if (over ? lane == __ffsll((unsigned long long)over) - 1 : lane == 0) firsts[wave] = first;
  if (some ? lane == 63 - __clzll((long long)some) : lane == 0) lasts[wave] = last;
  __syncthreads();
  if (threadIdx.x == 0) {
    int token = -1;
    for (int k = 0; k < kThreads / 64 && token < 0; ++k) token = firsts[k];
    for (int k = kThreads / 64 - 1; k >= 0 && token < 0; --k) token = lasts[k];
    p.d.emitted[d.out] = token;
  }
}

// A sequence's way, by one wave, and what its token is drawn from; write: also path, accepted, emitted
template <bool F32>
__device__ inline void find_way(const VerifyArgs& p, const Span& s, double per, int b, bool write, Draw& draw) {
  const int lane = threadIdx.x & 63;
  const Way w = walk<F32, false>(p, s, per, write, &draw);
  const RowSum r = w.row;
  const bool none = per == 0.0 || r.top == -INFINITY;
  const int out = s.first + w.kept - 1;
  if (lane == 0) {
    draw.times = w.times, draw.sum = r.sum, draw.top = r.top, draw.row = s.first + w.at, draw.out = out;
    draw.how = none ? kNothing : w.times > 0.0 ? kRest : w.tried > 0 && !p.d.draft_probs ? kWithout : kAll;
  }
  if (write) {
    for (int i = w.kept + lane; i < s.n; i += 64) p.d.path[s.first + i] = -1, p.d.emitted[s.first + i] = -1;
    if (lane == 0) {
      p.d.accepted[b] = w.kept;
      if (none) p.d.emitted[out] = r.top == -INFINITY ? -1 : r.at;
    }
  }
}
// Sums of SHORTS pieces of kShort elements from `first` on, by a workgroup
template <bool F32, int SHORTS>
__device__ inline void sum_shorts(const VerifyArgs& p, const Span& s, const Draw& d, double per, int b, int first) {
  __shared__ double scratch[kThreads / 64][SHORTS];
  Source<F32> next = source_of<F32>(p, d, first * kShort + (int)threadIdx.x * kOnce);
#pragma unroll 1
  for (int k = 0; k < SHORTS; ++k) {
    const Source<F32> from = next;
    const int i = (first + k) * kShort + (int)threadIdx.x * kOnce;
    if (k + 1 < SHORTS) next = source_of<F32>(p, d, i + kShort);
    double w[kOnce], sum = 0.0;
    weights_of<F32>(p, s, d, per, i, from, w);
#pragma unroll
    for (int j = 0; j < kOnce; ++j) sum += w[j];
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x / 64][k] = sum;
  }
  __syncthreads();
  if (threadIdx.x < SHORTS) {
    double all = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) all += scratch[w][threadIdx.x];
    const int c = first + (int)threadIdx.x;
    if (c < p.shorts) p.left[(size_t)b * p.shorts + c] = all;
  }
}

// Few pieces: every workgroup finds the way by itself and sums up one piece, and the last one of a sequence draws
template <bool F32>
__global__ __launch_bounds__(kThreads) void walk_and_draw_kernel(VerifyArgs p) {
  __shared__ Draw draw;
  __shared__ int before_me;
  const int piece = blockIdx.x % (unsigned)p.shorts, b = blockIdx.x / (unsigned)p.shorts;
  const Span s = span_of(p, b);
  const double per = inverse_temperature(p, b);
  if (s.n == 0) {
    if (piece == 0 && threadIdx.x == 0) p.d.accepted[b] = 0;
    return;
  }
  const double random = random_of(p, s.first);
  if (threadIdx.x < 64) find_way<F32>(p, s, per, b, piece == 0, draw);
  __syncthreads();
  if (draw.how == kNothing) return;
  sum_shorts<F32, 1>(p, s, draw, per, b, piece);
  if (threadIdx.x == 0) {
    __threadfence();   // the sum, before the count says that it is there
    before_me = atomicAdd(p.done + b, 1);
  }
  __syncthreads();
  if (before_me != p.shorts - 1) return;
  __threadfence();   // the others' sums
  draw_token<F32>(p, s, draw, per, random, b);
}

// Many: a launch each
template <bool F32>
__global__ __launch_bounds__(64) void walk_kernel(VerifyArgs p) {
  __shared__ Draw draw;
  const int b = blockIdx.x;
  const Span s = span_of(p, b);
  if (s.n > 0) find_way<F32>(p, s, inverse_temperature(p, b), b, true, draw);
  __syncthreads();
  if (threadIdx.x != 0) return;
  if (s.n == 0) p.d.accepted[b] = 0, p.draws[b].how = kNothing;
  else p.draws[b] = draw;
}
constexpr int kShorts = kPiece / kShort;
template <bool F32>
__global__ __launch_bounds__(kThreads) void left_sums_kernel(VerifyArgs p) {
  const unsigned of_sequence = (unsigned)(p.shorts + kShorts - 1) / kShorts;
  const int piece = blockIdx.x % of_sequence, b = blockIdx.x / of_sequence;
  const Draw& d = p.draws[b];
  if (d.how != kNothing) sum_shorts<F32, kShorts>(p, span_of(p, b), d, inverse_temperature(p, b), b, piece * kShorts);
}
template <bool F32>
__global__ __launch_bounds__(kThreads) void draw_kernel(VerifyArgs p) {
  const int b = blockIdx.x;
  if (p.draws[b].how == kNothing) return;
  const Span s = span_of(p, b);
  draw_token<F32>(p, s, p.draws[b], inverse_temperature(p, b), random_of(p, s.first), b);
}

// ---- children one after the other, where drafts come with distributions ----------------------------------------------------------------------------
template <bool F32>
__device__ inline bool accepts(const VerifyArgs& p, int row, const RowSum& r, double per, int child_row, double t, double left) {
  const int token = p.d.tokens[child_row];
  if (token < 0 || token >= p.d.vocab || !(r.sum > 0.0)) return false;
  const double q = draft_prob(p, row, token), w = weight_of(number(logit<F32>(p, row, token)), r.top, per) / r.sum;
  return random_of(p, child_row) * q * left < fmax(w - t * q, 0.0);
}

// Rows of two children and more whose first one is rejected: the sum of max(p - q, 0), a piece a workgroup; the last one goes on with the other children.
template <bool F32>
__global__ __launch_bounds__(kThreads) void children_kernel(VerifyArgs p) {
  constexpr int kParts = kPiece / kShort;
  __shared__ double scratch[kThreads / 64];
  __shared__ int before_me;
  const int row = blockIdx.x / (unsigned)p.pieces, piece = blockIdx.x % (unsigned)p.pieces;
  if (p.choice[row] != kMany) return;
  const int b = sequence_of(p, row);
  if (b < 0) return;
  const double per = inverse_temperature(p, b);
  const Span s = span_of(p, b);
  const int v = row - s.first;
  int child = next_child(p, s, v, v + 1);
  if (child >= s.n) return;
  const RowSum r = of_lane(sums_of_rows(p, (threadIdx.x & 63) == 0 ? row : -1, per, true), 0);
  if (accepts<F32>(p, row, r, per, s.first + child, 0.0, 1.0)) return;
  const auto sum_of = [&](int c, double t) {   // of piece c
    double sum = 0.0;
    if (r.sum > 0.0) {
      Draw rest{};
      rest.times = t, rest.sum = r.sum, rest.top = r.top, rest.row = row, rest.how = kRest;
      int i = c * kPiece + (int)threadIdx.x * kOnce;
      Source<F32> next = source_of<F32>(p, rest, i);
#pragma unroll 1
      for (int k = 0; k < kParts; ++k, i += kShort) {
        const Source<F32> from = next;
        if (k + 1 < kParts) next = source_of<F32>(p, rest, i + kShort);
        double w[kOnce];
        weights_of<F32>(p, s, rest, per, i, from, w);
#pragma unroll
        for (int j = 0; j < kOnce; ++j) sum += w[j];
      }
    }
    return block_sum<kThreads>(sum, scratch);
  };
  const double first = sum_of(piece, 1.0);
  if (threadIdx.x == 0) {
    p.rest[(size_t)row * p.pieces + piece] = first;
    __threadfence();   // the sum, before the count says that it is there
    before_me = atomicAdd(p.done + p.d.batch + row, 1);
  }
  __syncthreads();
  if (before_me != p.pieces - 1) return;
  __threadfence();   // the others' sums
  double t = 1.0, left = 0.0;
  for (int c = 0; c < p.pieces; ++c) left += p.rest[(size_t)row * p.pieces + c];
  int found = -1;
  for (child = next_child(p, s, v, child + 1); child < s.n;) {
    if (accepts<F32>(p, row, r, per, s.first + child, t, left)) {
      found = child;
      break;
    }
    t += left;
    child = next_child(p, s, v, child + 1);
    if (child >= s.n) break;
    left = 0.0;
    for (int c = 0; c < p.pieces; ++c) left += sum_of(c, t);
  }
  if (threadIdx.x == 0) p.choice[row] = found, p.times[row] = t;
}

VerifyArgs args_of(const ave_fp4_draft& d, void* ws, size_t* bytes) {
  VerifyArgs p{};
  p.d = d;
  p.pieces = (d.vocab + kPiece - 1) / kPiece, p.shorts = (d.vocab + kShort - 1) / kShort;
  char* at = static_cast<char*>(ws);
  size_t used = 0;
  const auto take = [&](size_t n) {
    char* r = at + used;
    used += (n + 255) / 256 * 256;
    return r;
  };
  const size_t all = (size_t)d.rows * p.pieces;
  p.sums = reinterpret_cast<PieceSum*>(take(all * sizeof(PieceSum)));
  p.left = reinterpret_cast<double*>(take((size_t)d.batch * p.shorts * sizeof(double)));
  p.draws = reinterpret_cast<Draw*>(take((size_t)d.batch * sizeof(Draw)));
  if (d.draft_probs) {
    p.rest = reinterpret_cast<double*>(take(all * sizeof(double)));
    p.times = reinterpret_cast<double*>(take((size_t)d.rows * sizeof(double)));
    p.choice = reinterpret_cast<int*>(take((size_t)d.rows * sizeof(int)));
  } else {
    p.wanted = reinterpret_cast<Wanted*>(take((size_t)d.rows * sizeof(Wanted)));
    p.many = reinterpret_cast<int*>(take(sizeof(int)));
  }
  p.done = reinterpret_cast<int*>(take(((size_t)d.batch + (d.draft_probs ? d.rows : 0)) * sizeof(int)));
  if (bytes) *bytes = used;
  return p;
}

// Node 0's rows first and then those that are wanted, instead of all at once: two launches more, against what need not be read.  us so and at once, trees of
// 16 nodes, 131072 tokens: 8 sequences (32 MB) 37 and 31, 16 40 and 40, 32 48 and 54, 64 65 and 80; 16 sequences of 64 nodes 60 and 74; chains of six, 64
// sequences 51 and 50.
bool in_two_steps(const VerifyArgs& p) {
  return (int64_t)p.d.rows * p.d.vocab * (p.d.logits_f32 ? 4 : 2) > (int64_t)64 << 20 && p.d.rows >= 3 * (int64_t)p.d.batch;
}

template <bool F32>
hipError_t launch(const VerifyArgs& p, hipStream_t s) {
  const unsigned rows = (unsigned)p.d.rows, batch = (unsigned)p.d.batch, pieces = (unsigned)p.pieces;
  if (p.d.draft_probs) {
    if (rows > 0) {
      hipLaunchKernelGGL((row_sums_kernel<F32, true, 0>), dim3(rows * pieces), dim3(2 * kThreads), 0, s, p);
      hipLaunchKernelGGL((children_kernel<F32>), dim3(rows * pieces), dim3(kThreads), 0, s, p);
    }
  } else if (in_two_steps(p)) {
    hipLaunchKernelGGL((row_sums_kernel<F32, false, 1>), dim3(batch * pieces), dim3(kThreads), 0, s, p);
    hipLaunchKernelGGL((first_step_kernel<F32>), dim3(batch), dim3(64), 0, s, p);
    hipLaunchKernelGGL((row_sums_kernel<F32, false, 2>), dim3(std::min(rows * pieces, 8u * (unsigned)compute_units())), dim3(kThreads), 0, s, p);
  } else if (rows > 0) {
    hipLaunchKernelGGL((row_sums_kernel<F32, false, 0>), dim3(rows * pieces), dim3(kThreads), 0, s, p);
  }
  // The way, its sums and the draw at once where that makes no more than one workgroup a compute unit (each finds the way by itself, and its fence costs the
  // others time): one sequence, 131072 tokens, 17 us, with a launch each 23; four 23 and 26, eight 34 and 31, 16 55 and 40.
  if (batch * (unsigned)p.shorts <= (unsigned)compute_units()) {
    hipLaunchKernelGGL((walk_and_draw_kernel<F32>), dim3(batch * (unsigned)p.shorts), dim3(kThreads), 0, s, p);
  } else {
    hipLaunchKernelGGL((walk_kernel<F32>), dim3(batch), dim3(64), 0, s, p);
    hipLaunchKernelGGL((left_sums_kernel<F32>), dim3(batch * pieces), dim3(kThreads), 0, s, p);
    hipLaunchKernelGGL((draw_kernel<F32>), dim3(batch), dim3(kThreads), 0, s, p);
  }
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
