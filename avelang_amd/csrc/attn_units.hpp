// Attention over an MXFP4 cache: what the rows of a sequence see, and how many units of work that makes.  Plain arithmetic, so that it also
// compiles for the host (without HIP), where a test goes through numbers that are too large for a run.
#pragma once
#include <stdint.h>

#include "../../include/ave_fp4.h"

#ifdef __HIP__
#define AVE_BOTH __host__ __device__
#else
#define AVE_BOTH
#endif

namespace ave {

// Units of a call are numbered in 32 bits (U = unsigned) where they cannot be more (units_bound), else in 64: an item has up to 2^25, a call up to
// 2^31 items.  600000 tokens of 128 heads on 8 over as many keys, all of them seen, come to 5.6e9.  (64 bits for every call: four tokens of 16
// sequences of 1500 keys 10.2 -> 11.1 us, by the longer way to the first load.)  Within an item 32 bits do.
typedef uint64_t Units;

struct PartMeta;

struct AttnArgs {
  ave_fp4_attention a;
  ave_fp4_kv_cache c;
  int group;          // query heads per key head
  int page_shift;
  int whole;          // 1: items are not split; no workspace, no second launch
  int q_aligned;      // every row of q starts at a multiple of 16 bytes
  int few_long;       // few sequences of many blocks of rows each
  int item_units;     // that the start and the end of an item count for beside its tiles
  int min_units_log2; // of a workgroup, so that small calls are not cut into crumbs
  PartMeta* meta;     // workspace: [workgroups]
  float* part_ml;     // [2 workgroups][ROWS][2]: maximum (base 2) and sum
  float* part_o;      // [2 workgroups][ROWS][D]
  unsigned group_mul, group_shift;   // division by `group` of numbers below 2^31: high word of the product, shifted (set_group)

  AVE_BOTH inline int token_of(int row) const { return group == 1 ? row : (int)((unsigned)((uint64_t)(unsigned)row * group_mul >> 32) >> group_shift); }
};
// The same for a tree of drafted tokens: the new tokens of a sequence see all keys before them, or the last p.a.window of what they see, and of each
// other those that their row of bits says.
struct PartStart;
struct TreeArgs : AttnArgs {
  PartStart* starts;      // workspace: [workgroups]
  const uint64_t* seen;   // bit j % 64 of word j / 64 of a token's row: new token j of its sequence
  int64_t seen_stride;    // words between rows
  int words;              // of a row
};
// 2^(31+s) / d rounded up with s = ceil(log2 d) has an error below 2^-31 of a quotient, so that n < 2^31 is divided exactly.
inline void set_group(AttnArgs& p, int group) {
  p.group = group;
  int s = 0;
  while ((1 << s) < group) ++s;
  p.group_mul = group == 1 ? 0 : (unsigned)((((uint64_t)1 << (31 + s)) / (unsigned)group) + 1);
  p.group_shift = group == 1 ? 0 : (unsigned)(s - 1);
}

// What a workgroup leaves for the second launch: its first unit, first and last unit (exclusive) of the item that it starts in, that item's
// first row of q, all rows of its sequence, key head, first row of the block; without work nothing but first units beyond all units
struct PartMeta {
  Units u0, begin, end;
  int first, rows, head, row0;
};

// Of a tree also by itself, for whoever looks through all of them
struct PartStart {
  Units u0, begin;
};

struct Sequence {
  int first, n, len;   // first row of q, new tokens, keys
};

// Keys that new token t of a sequence sees: [lo, hi)
AVE_BOTH inline void visible(const AttnArgs& p, const Sequence& s, int t, int& lo, int& hi) {
  const int pos = s.len - s.n + t;
  hi = p.a.causal ? pos + 1 : s.len;
  hi = hi < 0 ? 0 : hi;
  lo = p.a.window > 0 && pos >= p.a.window ? pos - p.a.window + 1 : 0;
}

// Rows t_first to t_last: [lo_min, hi_max) is what any of them sees at most, all of them see [lo_max, hi_min)
struct Bounds {
  int lo_min, lo_max, hi_min, hi_max;
};
AVE_BOTH inline Bounds bounds(const AttnArgs& p, const Sequence& s, int t_first, int t_last) {
  Bounds r;
  visible(p, s, t_first, r.lo_min, r.hi_min);
  visible(p, s, t_last, r.lo_max, r.hi_max);
  return r;
}
AVE_BOTH inline Bounds bounds(const TreeArgs& p, const Sequence& s, int, int) {   // (a row sees none to all of the n new tokens)
  const int base = s.len - s.n, before = base < 0 ? 0 : base, w = p.a.window;
  const int lo_min = w > 0 && base > w ? base - w : 0, lo_max = w > 0 && s.len > w ? s.len - w : 0;
  return {lo_min, lo_max, before, s.len};
}

// A block of rows: units (those for its start come before its tiles), and the first tile
template <int ROWS, int TILE, typename A>
AVE_BOTH inline int block_units(const A& p, const Sequence& s, int row0, int& tile0) {
  const int rows = s.n * p.group, last = row0 + ROWS < rows ? row0 + ROWS - 1 : rows - 1;
  if (rows <= 0) {
    tile0 = 0;
    return 1 + p.item_units;
  }
  const Bounds b = bounds(p, s, p.token_of(row0), p.token_of(last));
  const int lo = b.lo_min, hi = b.hi_max;
  tile0 = lo / TILE;
  return (hi > lo ? (hi + TILE - 1) / TILE - tile0 : 1) + p.item_units;
}
template <int ROWS, int TILE, typename U, typename A>
AVE_BOTH inline U sequence_units(const A& p, const Sequence& s) {   // of one key head
  U u = 0;
  int tile0;
  for (int row0 = 0; row0 < s.n * p.group; row0 += ROWS) u += (unsigned)block_units<ROWS, TILE>(p, s, row0, tile0);
  return u;
}
// All blocks of a tree's rows have the same units
template <int ROWS, int TILE, typename U>
AVE_BOTH inline U sequence_units(const TreeArgs& p, const Sequence& s) {
  int tile0;
  const unsigned rows = (unsigned)(s.n * p.group);
  return (U)((rows + ROWS - 1) / ROWS) * (unsigned)block_units<ROWS, TILE>(p, s, 0, tile0);
}
// No call has more, whatever its lengths are, as long as its sequences do not share rows of q (if they do, results are anybody's, and no walk
// leaves its bounds): blocks of rows, times the tiles that the page table or the window has for one
inline Units units_bound(const AttnArgs& p, int rows_of_block, int tile) {
  const Units rows = (Units)p.a.tokens * p.group, filled = rows / rows_of_block + p.a.batch, blocks = filled < rows ? filled : rows;
  const Units in_table = ((Units)p.a.table_pages << p.page_shift) / tile + 1, in_window = ((Units)p.a.window + rows_of_block) / tile + 2;
  const Units tiles = p.a.window > 0 && in_window < in_table ? in_window : in_table;
  return blocks * p.c.kv_heads * (tiles + p.item_units);
}

inline Units units_bound(const TreeArgs& p, int rows_of_block, int tile) {   // (a block also sees all new tokens of its sequence)
  AttnArgs q = p;
  if (p.a.window > 0) q.a.window = p.a.window > INT32_MAX - p.a.tokens ? INT32_MAX : p.a.window + p.a.tokens;
  return units_bound(q, rows_of_block, tile);
}

// The part of a workgroup: units [u0, u1) of all `units`, cut into `parts` equal ones; sequence b holds u0, b_begin is its first unit and
// per_head the units of one of its key heads.
template <typename U>
struct Part {
  U u0, u1, units;
  unsigned parts;
  int b;
  U b_begin, per_head;
  Sequence s;
};

// First unit of part g: the first units % parts parts have one unit more
template <typename U>
AVE_BOTH inline U part_start(U each, unsigned more, unsigned g) { return g * each + (g < more ? g : more); }

template <typename U>
AVE_BOTH inline void cut(const AttnArgs& p, Part<U>& r, unsigned g, unsigned workgroups) {
  const U want = (r.units + (1u << p.min_units_log2) - 1) >> p.min_units_log2;
  r.parts = want < workgroups ? (want ? (unsigned)want : 1) : workgroups;
  const U each = r.units / r.parts;
  const unsigned more = (unsigned)(r.units - each * r.parts);
  r.u0 = g < r.parts ? part_start(each, more, g) : r.units;
  r.u1 = g < r.parts ? part_start(each, more, g + 1) : r.units;
}

}  // namespace ave
