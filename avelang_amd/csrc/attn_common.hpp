// What the kernels of attention over an MXFP4 cache share: how the work of a call is cut into equal parts on the device, where
// partial results go, loads from the cache into LDS, and the queries' and probabilities' forms for the matrix cores.
//
// Work.  An item is a block of ROWS rows -- (new token, query head) pairs of one sequence and one key head, tokens first -- and has
// as many units as there are TILE keys between the first and the last one that any of its rows sees (at least one).  Units are
// numbered by sequence, key head, block, key; every workgroup takes the same number of consecutive ones, so that a long sequence
// beside short ones, or the triangle of a prompt, costs no workgroup more than another.  Lengths are device memory: each workgroup adds the
// units up for itself (one read of seq_lens and cu_q).  A part of an item that does not cover all of it goes to the workspace, and
// a second launch joins the parts in order.  (The arithmetic: attn_units.hpp.)
#pragma once
#include "attn_units.hpp"
#include "fp4_common.hpp"
#include "kv_cache.hpp"
#include "tile_common.hpp"

namespace ave {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef unsigned short us2 __attribute__((ext_vector_type(2)));

// A score that is not there: below every one that is, and exp2(kNone c - m c) is zero for every maximum m that is a score, and for m = 0,
// because c is 1e-30 at least (a softmax scale of zero is taken as 1e-30, which leaves scores without effect just the same).
constexpr float kNone = -3.0e38f;
__device__ inline float softmax_scale(float scale) { return fmaxf(fabsf(scale) * 1.4426950408889634f, 1e-30f); }   // base 2
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

typedef const __attribute__((address_space(4))) int32_t* ConstInts;   // read through the scalar cache where the index is uniform

__device__ inline Sequence sequence(const AttnArgs& p, int b) {
  const ConstInts cu = (ConstInts)p.a.cu_q, lens = (ConstInts)p.a.seq_lens;
  Sequence s;
  if (p.a.cu_q) {
    s.first = cu[b];
    s.first = s.first < 0 ? 0 : s.first > p.a.tokens ? p.a.tokens : s.first;
    int end = cu[b + 1];
    end = end < s.first ? s.first : end > p.a.tokens ? p.a.tokens : end;
    s.n = end - s.first;
  } else {
    s.first = b, s.n = 1;
  }
  const int most = p.a.table_pages << p.page_shift;
  s.len = lens[b];
  s.len = s.len < 0 ? 0 : s.len > most ? most : s.len;
  return s;
}

__device__ inline int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ inline unsigned wave_scan(unsigned v) {   // inclusive prefix sums over the lanes
  v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);   // one, two, four, eight lanes to the right in a row of 16
  v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
  v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
  v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
  v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);   // a row's last lane to the next row
  v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);   // lane 31 to the upper half
  return v;
}
__device__ inline unsigned lane_value(unsigned v, int lane) { return (unsigned)lane_value((int)v, lane); }
__device__ inline Units lane_value(Units v, int lane) {
  return (Units)(unsigned)lane_value((int)(unsigned)v, lane) | (Units)(unsigned)lane_value((int)(unsigned)(v >> 32), lane) << 32;
}
__device__ inline Units wave_scan(Units v) {   // of numbers whose sum is below 2^58: 26 bits and the rest, so that neither sum overflows
  return wave_scan((unsigned)v & 0x3FFFFFFu) + ((Units)wave_scan((unsigned)(v >> 26)) << 26);
}
// Units of one key head of a sequence of many blocks, which the lanes of a wave share
template <int ROWS, int TILE, typename U>
__device__ inline U wave_sequence_units(const AttnArgs& p, const Sequence& s) {
  U u = 0;
  int tile0;
  const int rows = s.n * p.group, lane = threadIdx.x & 63;
  for (int row0 = 0; row0 < rows; row0 += 64 * ROWS) {
    const int mine = row0 + lane * ROWS;
    u += lane_value(wave_scan(mine < rows ? (unsigned)block_units<ROWS, TILE>(p, s, mine, tile0) : 0u), 63);
  }
  return u;
}

// The part of workgroup g.  Every wave finds it by itself (no barrier): 64 sequences at a time, a lane each.
// LONG: sequences may have many blocks of rows; where p.few_long says so the wave takes one sequence after the other.
template <int ROWS, int TILE, typename U, bool LONG = false>
__device__ inline Part<U> take_part(const AttnArgs& p, unsigned g, unsigned workgroups) {
  if constexpr (LONG) {
    if (p.few_long) {
      Part<U> r{};
      const unsigned heads = (unsigned)p.c.kv_heads;
      for (int b = 0; b < p.a.batch; ++b) r.units += heads * wave_sequence_units<ROWS, TILE, U>(p, sequence(p, b));
      cut(p, r, g, workgroups);
      for (r.b = 0;; ++r.b) {   // (the last one if lengths change under the call)
        r.s = sequence(p, r.b);
        r.per_head = wave_sequence_units<ROWS, TILE, U>(p, r.s);
        if (r.u0 < r.b_begin + heads * r.per_head || r.b + 1 >= p.a.batch) break;
        r.b_begin += heads * r.per_head;
      }
      return r;
    }
  }
  const int lane = threadIdx.x & 63;
  const unsigned heads = (unsigned)p.c.kv_heads;
  const auto load = [&](int b) {
    Sequence s{0, 0, 0};
    if (b < p.a.batch) s = sequence(p, b);
    return s;
  };
  Part<U> r{};
  Sequence s = load(lane);
  U mine = sequence_units<ROWS, TILE, U>(p, s), in = wave_scan(mine * heads), total = lane_value(in, 63);
  r.units = total;
  Sequence next = load(64 + lane);
  for (int b0 = 64; b0 < p.a.batch; b0 += 64) {
    const Sequence now = next;
    next = load(b0 + 64 + lane);
    r.units += lane_value(wave_scan(sequence_units<ROWS, TILE, U>(p, now) * heads), 63);
  }
  cut(p, r, g, workgroups);
  if (r.u0 >= r.u1) return r;
  U base = 0;
  int b0 = 0;
  while (r.u0 >= base + total && b0 + 64 < p.a.batch) {   // (u0 is below the number of units: found at the latest in the last 64)
    base += total;
    b0 += 64;
    s = load(b0 + lane);
    mine = sequence_units<ROWS, TILE, U>(p, s);
    in = wave_scan(mine * heads);
    total = lane_value(in, 63);
  }
  const U begin = base + in - mine * heads;
  const uint64_t here = __ballot(begin <= r.u0 && r.u0 < begin + mine * heads);
  const int at = here ? __ffsll((unsigned long long)here) - 1 : 0;
  r.b = b0 + at;
  r.b_begin = lane_value(begin, at);
  r.per_head = lane_value(mine, at);
  r.s = {lane_value(s.first, at), lane_value(s.n, at), lane_value(s.len, at)};
  return r;
}

// An item, and where the units of a walk stand in it
template <typename U>
struct Item {
  Sequence s;
  int head, row0, tile0;
  unsigned units;
  U begin;
};
// The item that holds unit u >= b_begin; moves b, b_begin, the sequence s and its units of one head on to it.  (Where lengths change under the call
// it may end before u, and never begins behind it.)
template <int ROWS, int TILE, typename U, bool LONG = false>
__device__ inline Item<U> item_of(const AttnArgs& p, U u, int& b, U& b_begin, Sequence& s, U& per_head) {
  Item<U> it;
  // (u is below the number of all units; the bounds on b and row0 hold if lengths change under the call, too)
  while (u >= b_begin + per_head * (unsigned)p.c.kv_heads && b + 1 < p.a.batch) {
    b_begin += per_head * (unsigned)p.c.kv_heads;
    b = __builtin_amdgcn_readfirstlane(b + 1);
    s = sequence(p, b);
    per_head = LONG ? wave_sequence_units<ROWS, TILE, U>(p, s) : sequence_units<ROWS, TILE, U>(p, s);
  }
  it.s = s;
  it.head = 0;
  it.begin = b_begin;
  while (u >= it.begin + per_head && it.head + 1 < p.c.kv_heads) it.begin += per_head, ++it.head;
  if constexpr (LONG) {   // 64 blocks at a time, a lane each
    const int lane = threadIdx.x & 63, rows = s.n * p.group;
    for (int row0 = 0;; row0 += 64 * ROWS) {
      const int mine = row0 + lane * ROWS;
      int tile0 = 0;
      const unsigned units = mine < rows ? (unsigned)block_units<ROWS, TILE>(p, s, mine, tile0) : 0u, in = wave_scan(units);
      const unsigned total = lane_value(in, 63);
      const U rest = u - it.begin;
      if (rest < total || row0 + 64 * ROWS >= rows) {
        const uint64_t here = __ballot(rest < in);
        const int at = here ? __ffsll((unsigned long long)here) - 1 : 0;
        it.row0 = row0 + at * ROWS;
        it.units = lane_value(units, at);
        it.tile0 = lane_value(tile0, at);
        it.begin += lane_value(in - units, at);
        return it;
      }
      it.begin += total;
    }
  }
  for (it.row0 = 0;; it.row0 += ROWS) {
    it.units = (unsigned)block_units<ROWS, TILE>(p, it.s, it.row0, it.tile0);
    if (u < it.begin + it.units || it.row0 + ROWS >= it.s.n * p.group) break;
    it.begin += it.units;
  }
  return it;
}

// ---- loads ---------------------------------------------------------------------------------------------------------------------
// Lane l of the wave writes its 16 (4) bytes at LDS address lds + 16 l (4 l), straight from memory; counts on vmcnt.
__device__ inline void to_lds16(const uint8_t* src, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(src) : "m0", "memory");
}
__device__ inline const uint8_t* uniform_pointer(const uint8_t* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  return reinterpret_cast<const uint8_t*>((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)v) | (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32);
}
// A wave-uniform base in scalar registers: five wait states have to pass if a vector instruction (uniform_pointer, a register spilled to lanes) wrote
// them just before, and the compiler, which counts those for its own loads, does not look inside: one by s_mov, four by s_nop.
template <bool ONCE = false>   // ONCE: nobody else will want it (non-temporal)
__device__ inline void to_lds16(const uint8_t* base, unsigned offset, unsigned lds) {   // base is wave-uniform
  if constexpr (ONCE) asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(offset), "s"(base) : "m0", "memory");
  else asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(offset), "s"(base) : "m0", "memory");
}
__device__ inline void to_lds4(const uint8_t* src, unsigned lds) {   // (scales for few rows, which nobody else will want either)
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off nt" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(src) : "m0", "memory");
}
__device__ inline void to_lds4(const uint8_t* base, unsigned offset, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dword %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(offset), "s"(base) : "m0", "memory");
}
template <int N>
__device__ inline void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ inline unsigned lds_address(const void* p) {
  return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}

// Page of tokens 16 i .. 16 i + 15 of a sequence of len > 0 keys (behind the last: the last one's): what the table holds, and a valid one of that
__device__ inline int page_entry(const AttnArgs& p, ConstInts row, int token, int len) { return row[(token < len ? token : len - 1) >> p.page_shift]; }
__device__ inline int page_of(const AttnArgs& p, int entry) {
  const int page = entry < 0 ? 0 : entry;
  return page < p.c.pages ? page : p.c.pages - 1;
}
__device__ inline int page_at(const AttnArgs& p, ConstInts row, int token, int len) { return page_of(p, page_entry(p, row, token, len)); }

// A value that all lanes hold, in a scalar register
__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline float uniform(float x) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x))); }

// Eight bf16, from any address where `aligned` is not set
__device__ inline v4i load8_bf16(const uint16_t* q, bool aligned) {
  if (aligned) return *reinterpret_cast<const v4i*>(q);
  v4i r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (int)((unsigned)q[2 * i] | (unsigned)q[2 * i + 1] << 16);
  return r;
}
__device__ inline float bf16_lo(int x) { return __builtin_bit_cast(float, (unsigned)x << 16); }
__device__ inline float bf16_hi(int x) { return __builtin_bit_cast(float, (unsigned)x & 0xFFFF0000u); }

// max3 as it is: fmaxf makes the compiler pass every operand through another maximum first (signalling NaN).  A NaN loses to a number.
// The compiler does not see inside, so it does not wait for a matrix instruction whose result is an operand: `after` must come from an
// ordinary instruction on that result, for which it has waited.
__device__ inline float max3(float a, float b, float c, float after) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c), "v"(after));
  return r;
}
// Largest of the sixteen results of one matrix instruction, from `first` to `last`, and of `other`
template <int first, int last>
__device__ inline float largest_of(const v16f& s, float other) {
  static_assert((last - first) % 2 == 1 && last > first + 2, "");
  const float after = fmaxf(s[first], s[first + 1]);
  float top = max3(after, s[first + 2], s[first + 3], after), two = other;
#pragma unroll
  for (int t = first + 4; t < last; t += 4) {
    two = max3(two, s[t], s[t + 1], after);
    if (t + 2 < last) top = max3(top, s[t + 2], s[t + 3], after);
  }
  return fmaxf(top, two);
}
// Two 16-bit a * k + c, k a scalar pair
__device__ inline unsigned pk_mad_u16(unsigned a, unsigned k, unsigned c) {
  unsigned r;
  asm("v_pk_mad_u16 %0, %1, %2, %3" : "=v"(r) : "v"(a), "s"(k), "v"(c));
  return r;
}
__device__ inline us2 as_us2(unsigned x) { return __builtin_bit_cast(us2, x); }
__device__ inline unsigned as_u32(us2 x) { return __builtin_bit_cast(unsigned, x); }
__device__ inline unsigned pk_sub_sat(unsigned a, unsigned b) { return as_u32(__builtin_elementwise_sub_sat(as_us2(a), as_us2(b))); }

// ---- queries: two 8-bit parts ------------------------------------------------------------------------------------------------------
// The scaled MFMAs multiply E2M1 keys as they are with 8-bit queries.  A bf16 number has 8 significant bits, an E4M3 number 4:
// q = 2^e hi + 2^(e-5) lo, hi the rounded q / 2^e and lo the rounded rest times 32, is exact down to 2^-19 of the row's largest element
// (e puts that one into [2^7, 2^8)); two MFMAs take the time that one bf16 product of the same length would, and no key is converted.
struct QueryScale {
  float hi, lo;             // 2^e, 2^(e-5)
  int hi_byte, lo_byte;     // the same as E8M0; 0xFF (NaN) for a row with an infinity or a NaN
};
__device__ inline QueryScale query_scale(unsigned amax) {   // of bf16 bits
  int f = (int)(amax >> 7);
  const bool bad = f == 0xFF;
  f = f < 13 ? 13 : f;   // e + 127 = f - 7
  const float hi = __builtin_bit_cast(float, (unsigned)(f - 7) << 23), lo = __builtin_bit_cast(float, (unsigned)(f - 12) << 23);
  return {hi, lo, bad ? 0xFF : f - 7, bad ? 0xFF : f - 12};
}
typedef short v2s __attribute__((ext_vector_type(2)));
// Eight bf16 -> 2 x 4 bytes of each part (the conversions divide and multiply by their scale operand)
__device__ inline void split_query(v4i x, const QueryScale& s, int (&hi)[2], int (&lo)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int x0 = x[2 * i], x1 = x[2 * i + 1];
    v2s h = {0, 0}, l = {0, 0};
    h = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(h, __builtin_bit_cast(v2bf, x0), s.hi, false);
    h = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(h, __builtin_bit_cast(v2bf, x1), s.hi, true);
    hi[i] = __builtin_bit_cast(int, h);
    const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi[i], s.hi, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi[i], s.hi, true);
    l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, bf16_lo(x0) - a[0], bf16_hi(x0) - a[1], s.lo, false);
    l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, bf16_lo(x1) - b[0], bf16_hi(x1) - b[1], s.lo, true);
    lo[i] = __builtin_bit_cast(int, l);
  }
}
// Largest magnitudes of eight bf16 as bit patterns in the two halves of m (NaN > infinity > numbers)
__device__ inline us2 amax_pairs(v4i x, us2 m) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned w = (unsigned)x[i] & 0x7FFF7FFFu;
    m = __builtin_elementwise_max(m, as_us2(w));
  }
  return m;
}
__device__ inline unsigned larger_half(us2 m) {
  const unsigned a = m[0], b = m[1];
  return a > b ? a : b;
}

// Largest value of lanes l, l ^ 16, l ^ 32, l ^ 48 (XOR16) or l, l ^ 32
__device__ inline float max_of_swapped(unsigned a, unsigned b) { return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)); }
template <bool XOR16>
__device__ inline float cross_max(float v) {   // (a vector's element is copied before __builtin_bit_cast, which reads element 0 of it otherwise)
  unsigned a = __builtin_bit_cast(unsigned, v);
  auto r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  v = max_of_swapped(r[0], r[1]);
  if constexpr (XOR16) {
    a = __builtin_bit_cast(unsigned, v);
    r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    v = max_of_swapped(r[0], r[1]);
  }
  return v;
}
template <bool XOR16>
__device__ inline float cross_sum(float v) {
  v += __shfl_xor(v, 32, 64);
  if constexpr (XOR16) v += __shfl_xor(v, 16, 64);
  return v;
}

// A row's place in the output: (token, query head)
__device__ inline size_t row_index(const AttnArgs& p, int first, int head, int row) {
  const int t = p.token_of(row);
  return (size_t)(first + t) * p.a.heads + head * p.group + (row - t * p.group);
}

// What the sums of a finished row are multiplied with, and its lse; m in base 2 (-inf: the row saw nothing).
struct RowEnd {
  float factor, lse;
};
__device__ inline float sink_of(const AttnArgs& p, int query_head) { return p.a.sinks ? p.a.sinks[query_head] * kLog2e : -INFINITY; }
__device__ inline RowEnd row_end(float sink, float m, float l) {   // sink in base 2
  const bool none = m == -INFINITY && l == l;   // (only NaN scores: the sum is NaN)
  const float top = fmaxf(m, sink), fade = none ? 0.0f : __builtin_amdgcn_exp2f(m - top);
  const float total = (none ? 0.0f : l * fade) + (sink == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sink - top));
  return {none ? 0.0f : fade / total, (top + __builtin_amdgcn_logf(total)) * kLn2};
}
__device__ inline void store4_bf16(uint16_t* out, v4f o) {
  reinterpret_cast<unsigned*>(out)[0] = pack_bf16x2(o[0], o[1]);
  reinterpret_cast<unsigned*>(out)[1] = pack_bf16x2(o[2], o[3]);
}
// Four channels of a finished row
__device__ inline void finish_row(const AttnArgs& p, size_t row, int D, int channel, v4f o, float m, float l) {
  const RowEnd e = row_end(sink_of(p, (int)(row % (unsigned)p.a.heads)), m, l);
  store4_bf16(p.a.out + row * D + channel, o * e.factor);
  if (p.a.lse && channel == 0) p.a.lse[row] = e.lse;
}

hipError_t launch_attn_prompt(AttnArgs p, void* workspace, hipStream_t s);
size_t attn_prompt_workspace(const AttnArgs& p);
hipError_t launch_attn_decode(AttnArgs p, int row_tiles, void* workspace, hipStream_t s);
size_t attn_decode_workspace(const AttnArgs& p, int row_tiles);
// rows: of a block; rows_expected: of a sequence and key head
hipError_t launch_attn_combine(const AttnArgs& p, int rows, int64_t rows_expected, int workgroups, hipStream_t s);
// meta, maxima and sums, partial results, in this order
inline size_t attn_meta_bytes(int workgroups) { return ((size_t)workgroups * sizeof(PartMeta) + 255) / 256 * 256; }
inline size_t attn_workspace(int rows, int head_dim, int workgroups) {
  return attn_meta_bytes(workgroups) + (size_t)workgroups * 2 * rows * (2 + head_dim) * 4;
}
inline void place_workspace(AttnArgs& p, int rows, int workgroups, void* ws) {
  p.meta = static_cast<PartMeta*>(ws);
  p.part_ml = reinterpret_cast<float*>(static_cast<char*>(ws) + attn_meta_bytes(workgroups));
  p.part_o = p.part_ml + (size_t)workgroups * 2 * rows * 2;
}
}  // namespace ave
