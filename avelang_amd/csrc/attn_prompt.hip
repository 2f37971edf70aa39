// Attention of many query rows over a paged MXFP4 cache: prompts and chunks of prompts.
//
// Bound by the matrix cores and by the exponentials beside them.  A workgroup takes blocks of 128 rows -- (token, query head) pairs of one
// key head, 32 a wave -- through 64 keys at a time, in equal parts of the call (attn_common.hpp) or as whole blocks, largest first:
//
//   S^T = K Q^T   scaled MFMA 32x32x64, keys as they are (E2M1 codes and E8M0 scales straight from memory into LDS), queries as two E4M3
//                 parts.  Row 8 i + 4 h + t of a tile of 32 keys is key 16 h + 4 i + t, so that lane half h = lane / 32 of the result holds
//                 keys 16 h .. 16 h + 15 of the tile for query row lane % 32.
//   O^T = V^T P^T bf16 MFMA 32x32x16: P goes from the result's registers into the operand as it is, rounded to bf16 (for the reason in
//                 attn_decode.hip).  Values are converted once a workgroup, codes times their scales (exact), and lie in LDS as bf16 rows that
//                 transposing reads hand out by columns.
//
// What a wave does for 64 keys: 8 scaled and 16 bf16 MFMAs at 128 channels (about 1090 cycles), and beside them 32 each of fma, exponential
// and addition a lane, 16 conversions of P, a quarter of a tile's values converted, requests and addresses (about 950).  Scores, exponentials and
// values come one after the other; three waves a SIMD (four at 64 channels, two at 256), each of another workgroup and at another point, put
// the ones under the others.  That measured faster than two waves with the three interleaved by hand (677 us against 642, 8192 tokens, 32 heads on
// 8 of 128) and than 64 rows a wave in 512 registers (1354: one wave issues an instruction in five cycles).  What then counted:
//   - nobody waits between the requests for the next tile and the products (scales unpacked and table entries checked where they are used, lane
//     constants in LDS instead of spilled: 642 -> 609);
//   - equal ends: workgroups of a compute unit take turns in going first, and an item's start and end count as tiles (609 -> 537);
//   - LDS reads ahead of the products (four long sequences: 348 -> 332); half tiles that nobody sees skipped (533 -> 515).
//   - whole items instead of parts where that leaves little waiting (503 -> 480; six prompts of about 1000 tokens 88 -> 72).
// (Cards differ by some per cent; a figure and the one it is compared with are of one card.)
// 8192 tokens, 32 heads on 8 of 128: 459 us, 1.20 PFLOP/s of 4 D flop a score (the matrix cores also multiply the queries' second part, half as much
// again); 4 sequences of up to 16000 keys, 600 new tokens, 40 heads on 8: 320 us, 1.11 PFLOP/s; six prompts of about 1000 tokens, 64 heads on 8 of 64:
// 67 us, where an item of 128 rows has but 8 tiles for its start and end, and half the work is exponentials.
//
// Trees of drafted tokens (TreeArgs): a row sees its sequence's keys before the nodes, and of the nodes those with a bit; bits are looked at in tiles that hold
// nodes only.  Drafts make 17 to 128 rows a key head, so there are blocks of 64 rows, too (SPLIT 2: waves 0 and 1 take the first 32 keys of a tile, 2 and 3 the
// others, with sums of their own that meet in LDS at the item's end), and always parts: 16 sequences of up to 4096 keys, 16 nodes, 32 heads on 8 of 128 33 us and
// 7.5 the join (vector units 29 % busy, matrix cores 13 %; 6 to 10 us are the start); 8 of up to 3000, 64 nodes, 64 heads on 8 of 64, window 1000 28 and 7.4; one of
// 131072, 64 nodes (blocks of 128 rows) 129 and 12.5, 1.06 PFLOP/s in the first.
#include "attn_common.hpp"
#include "kernels.hpp"

namespace ave {
namespace {

typedef short v4s __attribute__((ext_vector_type(4)));

constexpr float kNoMax = -1.0e30f;   // a maximum of nothing
constexpr int kTile = 64, kWaves = 4, kMostRows = 32 * kWaves, kBuffers = 2;

template <int D>
struct Shape {
  static constexpr int kRow = D / 2, kBlocks = D / 32, kSteps = D / 64, C = D / 32;
  static constexpr int kKeys = kTile * kRow, kScales = kTile * kBlocks, kValues = kTile * D * 2;
  static constexpr int kFar = D == 256 ? 2 : 0;
  static constexpr int kValueBuffers = D == 256 ? 1 : kBuffers;   // (two workgroups a compute unit)
  static constexpr int kBuffer = kKeys + kScales, kLds = kBuffers * kBuffer + kValueBuffers * kValues;   // keys' buffers, then values'
  static constexpr int kThreadBytes = kTile * kRow / (kWaves * 64);   // of values' codes: 8, 16 or 32, within one or two blocks of a token
  // LDS positions.  Keys: 16-byte pieces permuted so that the 16 lanes of a read touch different banks.  Values: a row's 64-byte segments, and
  // the pieces of a segment, permuted by the token for the transposing reads (four tokens, 64 bytes each) and the writes.
  __device__ static int key_swizzle(int t) {
    return D == 64 ? (t >> 4) & 1 : D == 128 ? ((t >> 2) & 1) | ((t >> 4) & 1) << 1 : ((t >> 1) & 1) | ((t >> 2) & 1) << 1 | ((t >> 4) & 1) << 2;
  }
  __device__ static int value_swizzle(int t) { return D == 64 ? 5 * ((t >> 1) & 1) : 5 * (t & 3); }
};

// Values' codes of one thread for one tile, and their scale bytes
template <int D>
struct Values {
  static constexpr int kWords = Shape<D>::kThreadBytes / 4, kScaleBytes = D == 256 ? 2 : 1;
  unsigned code[kWords], scales;   // scales: the four bytes that hold them
  // where those lie behind the wave's first token, and from which bit this lane's own
  __device__ static unsigned scales_at(int lane) { return D == 64 ? lane / 8 * 4 : D == 128 ? lane / 4 * 4 : lane / 2 * 4; }
  __device__ static int shift(int lane) { return D == 64 ? 8 * (lane / 2 % 4) : D == 128 ? 8 * (lane % 4) : 16 * (lane % 2); }
};

template <int N>
struct Index {
  static constexpr int value = N;
};

typedef __attribute__((address_space(3))) v4i LdsInt4;
typedef __attribute__((address_space(3))) unsigned LdsInt;
typedef __attribute__((address_space(3))) v2i LdsInt2;
typedef __attribute__((address_space(3))) v4f LdsFloat4;
typedef __attribute__((address_space(3))) uint16_t LdsShort;
typedef __attribute__((address_space(3))) v4s LdsShort4;
typedef __attribute__((address_space(3))) v8bf Lds8Bf16;
typedef int Loose4 __attribute__((ext_vector_type(4), aligned(4)));   // (results are aligned to 4 bytes)
template <typename T>
__device__ inline T* lds_at(unsigned address) {
  return (T*)(uintptr_t)address;
}

// Waves of a SIMD, each of another workgroup: by registers (a wave's sums are D / 2 of them, its queries D / 4)
template <int D>
constexpr int waves_per_simd() {
  return D == 64 ? 4 : D == 128 ? 3 : 2;
}

// Whole items in falling order, for calls of up to kSequences.  Level k has the k-th last block of each sequence and key head that has so many;
// items are numbered level by level (by sequence, then head, within one), so that causal ones, which have fewer keys the earlier their rows
// stand, come largest first.  `all` is a table of the sequences in LDS, {first, n, len, blocks}; every lane of the wave takes part.
constexpr int kSequences = kWaves * 64;
__device__ inline unsigned items_below(const AttnArgs& p, const v4i* all, unsigned level) {   // of levels below
  const auto of_lane = [&](int b0) {
    const unsigned blocks = (unsigned)all[b0 + (threadIdx.x & 63)][3];
    return blocks < level ? blocks : level;
  };
  unsigned mine = of_lane(0);
  if (p.a.batch > 64)
    for (int b0 = 64; b0 < kSequences; b0 += 64) mine += of_lane(b0);   // (nothing behind the last sequence)
  return (unsigned)p.c.kv_heads * (unsigned)lane_value((int)wave_scan(mine), 63);
}
template <int ROWS, typename U, typename A>
__device__ inline Item<U> ranked_item(const A& p, const v4i* all, unsigned rank, int& b) {   // rank: below the number of items
  const unsigned heads = (unsigned)p.c.kv_heads;
  unsigned level = 0, step = 1;   // the level: the last one with at most `rank` items below it
  while (items_below(p, all, level + step) <= rank) level += step, step *= 2;
  for (; step > 0; step /= 2)
    if (items_below(p, all, level + step) <= rank) level += step;
  const unsigned rest = rank - items_below(p, all, level);
  unsigned index = rest / heads;   // among the sequences that have so many blocks
  const unsigned head = rest - index * heads;
  int b0 = 0;
  v4i mine = all[threadIdx.x & 63];
  uint64_t have = __ballot((unsigned)mine[3] > level);
  if (p.a.batch > 64)
    while (index >= (unsigned)__popcll(have) && b0 + 64 < kSequences) {
      index -= (unsigned)__popcll(have);
      b0 += 64;
      mine = all[b0 + (threadIdx.x & 63)];
      have = __ballot((unsigned)mine[3] > level);
    }
  const unsigned before = __builtin_amdgcn_mbcnt_hi((unsigned)(have >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)have, 0u));
  const uint64_t found = __ballot((unsigned)mine[3] > level && before == index);
  const int at = uniform(found ? __ffsll((unsigned long long)found) - 1 : 0);
  b = b0 + at;
  Item<U> it{};
  it.s = {lane_value(mine[0], at), lane_value(mine[1], at), lane_value(mine[2], at)};
  it.head = uniform((int)head);
  it.row0 = uniform((lane_value(mine[3], at) - 1 - (int)level) * ROWS);
  it.units = (unsigned)uniform(block_units<ROWS, kTile>(p, it.s, it.row0, it.tile0));
  return it;
}

// Of a tree: which of the 16 keys from `key` on a row of a sequence sees (a row behind the last: what that one does)
__device__ inline unsigned tree_bits(const TreeArgs& p, const Sequence& s, int row, int rows, int key) {
  const int t = p.token_of(row < rows ? row : rows - 1);
  return seen_of(p, s, t, first_seen(p, s, t), key);
}

// SMALL: no tensor of the cache spans more than 4 GB, so that 32 bits hold a byte offset (64 prompts of 200 tokens: 84 us, with 64-bit
// bases for every tile 89).
// SPLIT 2: blocks of 64 rows; waves 0 and 1 take the first 32 keys of a tile, 2 and 3 the others, and the two results of a row meet at the item's end.
template <int D, bool SMALL, typename U, typename A, int SPLIT = 1>
__global__ __launch_bounds__(kWaves * 64, (waves_per_simd<D>())) void attn_prompt_kernel(A p) {
  using S = Shape<D>;
  constexpr int C = S::C, kRows = kMostRows / SPLIT;
  __shared__ __align__(512) unsigned char smem[S::kLds];
  __shared__ uint64_t nan_in[kBuffers][Values<D>::kScaleBytes][kWaves];   // which lanes of a wave hold a value with a NaN scale
  __shared__ __align__(16) int nan_any[kBuffers][kWaves];
  __shared__ float other_ml[SPLIT == 2 ? 2 : 1][32][2];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid & 63, h = lane / 32, col = lane % 32;
  // Equal parts, or whole items: then a workgroup takes one of the first gridDim.x, in the next round the one as far from the end, and so on to
  // and fro.  What that may cost is the largest item of the last round (`most` units), less a workgroup's share of that round;
  // up to 24 units it is below the cost of partial results, their launch and the items' second starts (six prompts of 1000 tokens, 64 channels: 71 us,
  // in parts 88; 4 of 2000, 256 channels 173 and 222; one of 8192, 128 channels, 22 units: 591 and 624; 150 of 100 89 and 108).
  __shared__ __align__(16) v4i sequences[kTree<A> ? 1 : kSequences];
  unsigned items = 0, rounds = 0;
  bool by_items = false;
  if (!kTree<A> && p.a.batch <= kSequences) {
    Sequence s{0, 0, 0};
    if (tid < p.a.batch) s = sequence(p, tid);
    sequences[tid] = v4i{s.first, s.n, s.len, (s.n * p.group + kRows - 1) / kRows};
    __syncthreads();
    items = items_below(p, sequences, 0x7FFFFFFFu);
    rounds = (items + gridDim.x - 1) / gridDim.x;
    if (rounds == 0) {
      by_items = true;
    } else {
      int any;
      const uint64_t all = gridDim.x, last = items - (rounds - 1) * gridDim.x;
      const uint64_t most = ranked_item<kRows, U>(p, sequences, (rounds - 1) * gridDim.x, any).units;
      by_items = most <= 8 || 2 * all * most <= 48 * all + last * (most + ranked_item<kRows, U>(p, sequences, items - 1, any).units);
    }
  }
  // workgroups of an XCD (every eighth) take neighbouring parts, which read the same keys
  unsigned g = gridDim.x % 8 == 0 ? blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8 : blockIdx.x;
  Part<U> part{};
  TreeWalk<U> walk{};
  if constexpr (kTree<A>) walk = tree_part<D, kRows, kTile, U>(p, blockIdx.x, gridDim.x, waves_per_simd<D>(), g, by_items, part.u0, part.u1, part.units);
  else if (!by_items) part = take_part<kRows, kTile, U, true>(p, g, gridDim.x);
  const unsigned lds = (unsigned)__builtin_amdgcn_readfirstlane((int)lds_address(smem));
  const float c = uniform(softmax_scale(p.a.scale));
  // this lane's places in LDS, of the first half of the first buffer: its key (row 8 i + 4 h' + t' of a result is key 16 h' + 4 i + t'), the
  // key's scales, and by 32 channels the values
  // (k steps of 64 or 32 channels on they differ by an exclusive or alone).  They wait in LDS, as registers are short.
  __shared__ __align__(16) v4i places[64], far_q[2 * S::kFar + 1][S::kFar ? kWaves * 64 : 1];
  if (tid < 64) {
    const int t = 16 * ((col >> 2) & 1) + 4 * (col >> 3) + (col & 3), r = lane % 16 / 4;   // r: token within four
    const unsigned key_at = lds + t * S::kRow + (h ^ S::key_swizzle(t)) * 16, scale_at = lds + S::kKeys + t * S::kBlocks;
    const unsigned value_at = lds + kBuffers * S::kBuffer + (16 * h + r) * (2 * D) + ((2 * ((lane / 16) & 1) + (lane % 4) / 2) ^ S::value_swizzle(r)) * 16 + (lane & 1) * 8;
    places[lane] = v4i{(int)key_at, (int)scale_at, (int)value_at, 8 * h};
  }
  __syncthreads();
  const auto lane_here = [&] {   // for what is derived from the lane where it is used, and not kept in registers all the time
    int x = lane;
    asm volatile("" : "+v"(x));
    return x;
  };
  int b = part.b;
  U b_begin = part.b_begin, per_head = part.per_head;
  Sequence seq = part.s;
  if (tid == 0 && (part.u0 >= part.u1 || (kTree<A> && by_items))) {   // no part, nothing to join
    PartMeta& m = p.meta[g];
    m.u0 = m.begin = m.end = part.units;
    if constexpr (kTree<A>) p.starts[g] = {part.units, part.units};
  }
  // Among waves that could issue, the oldest goes first, so that of equal parts the workgroups that a compute unit got last would end
  // long after the others (452 us the first, 677 the last).  The later a workgroup came, the more of its tiles it takes at a higher priority.
  const int late = blockIdx.x * waves_per_simd<D>() / gridDim.x;
  int turn = 0;
  bool first_item = true;
  Item<U> it{};
  U u = part.u0;
  for (unsigned round = 0; by_items && !kTree<A> ? round < rounds : u < part.u1; ++round) {
    unsigned from = 0, to;   // units of the item
    if constexpr (kTree<A>) {
      if (!first_item) tree_next<kRows, kTile, U>(p, walk);
      b = walk.b;
      it.s = walk.s, it.head = walk.head, it.row0 = walk.row0, it.tile0 = walk.tile0, it.units = walk.units, it.begin = walk.begin;
      if (!by_items && first_item && tid == 0) {
        p.meta[g] = {part.u0, it.begin, it.begin + it.units, it.s.first, it.s.n * p.group, it.head, it.row0};
        p.starts[g] = {part.u0, it.begin};
      }
      if (!by_items && u - it.begin >= it.units) break;   // (lengths that change under the call: no walk without end, and the second launch finds its record)
      from = by_items ? 0 : (unsigned)(u - it.begin);
      to = by_items || part.u1 - it.begin >= it.units ? it.units : (unsigned)(part.u1 - it.begin);
      u = by_items ? part.u1 : it.begin + to;
      first_item = false;
    } else if (by_items) {
      const unsigned rank = round * gridDim.x + (round % 2 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
      if (rank >= items) break;
      it = ranked_item<kRows, U>(p, sequences, rank, b);
      to = it.units;
    } else {
      if (!first_item && it.row0 + kRows < it.s.n * p.group) {   // the next block of the same key head
        it.row0 += kRows;
        it.begin = u;
        it.units = (unsigned)block_units<kRows, kTile>(p, it.s, it.row0, it.tile0);
      } else {
        it = item_of<kRows, kTile, U, true>(p, u, b, b_begin, seq, per_head);
      }
      if (first_item && tid == 0) p.meta[g] = {part.u0, it.begin, it.begin + it.units, it.s.first, it.s.n * p.group, it.head, it.row0};
      if (u - it.begin >= it.units) break;   // (lengths that change under the call: no walk without end, and the second launch finds its record)
      from = (unsigned)(u - it.begin), to = part.u1 - it.begin < it.units ? (unsigned)(part.u1 - it.begin) : it.units;
      u = it.begin + to;
      first_item = false;
    }
    const unsigned start = (unsigned)p.item_units;   // unit of the item's first tile
    const unsigned first = from > start ? from : start;
    const int rows = it.s.n * p.group, tile0 = it.tile0 + (int)(first - start);
    const int tiles = it.s.len > 0 && to > first ? (int)(to - first) : 0;
    const ConstInts table = (ConstInts)(p.a.page_table + (int64_t)b * p.a.page_table_stride);

    // what this wave's rows see: [lo_max, hi_min) all of them, [lo_min, hi_max) any
    const int row0 = uniform(it.row0 + 32 * (SPLIT == 1 ? wave : wave % 2)), keys_from = SPLIT == 1 ? 0 : wave / 2 * 32;   // of a tile
    const bool active = row0 < uniform(rows);
    int lo_max, hi_min, lo_min, hi_max;
    if constexpr (kTree<A>) {
      const Bounds all = bounds(p, it.s, 0, 0);
      lo_max = all.lo_max, hi_min = all.hi_min, lo_min = all.lo_min, hi_max = all.hi_max;
    } else {
      visible(p, it.s, p.token_of(active ? row0 : 0), lo_min, hi_min);
      visible(p, it.s, p.token_of(row0 + 32 < rows ? row0 + 31 : rows - 1), lo_max, hi_max);
    }
    lo_max = uniform(lo_max), hi_min = uniform(hi_min), lo_min = uniform(lo_min), hi_max = uniform(hi_max);

    // ---- a tile's requests: keys and their scales to LDS, values to registers; a wave takes 16 tokens, which lie in one page
    Values<D> next;
    const auto entry_of = [&](int tile) { return page_entry(p, table, tile * kTile + 16 * wave, it.s.len); };   // one tile ahead of its use: nobody waits
    // A tensor's base and offset for this wave's tokens of a tile, `bytes` a token and head
    const auto place = [&](const uint8_t* tensor, int64_t stride, int pg, int tile, unsigned bytes, const uint8_t*& base) -> unsigned {
      const int t = tile * kTile + 16 * wave;
      const unsigned in_page = (unsigned)(it.head * p.c.page_size + (t & (p.c.page_size - 1))) * bytes;
      if constexpr (SMALL) {
        base = tensor;
        return (unsigned)pg * (unsigned)stride + in_page;
      } else {
        base = uniform_pointer(tensor + (int64_t)pg * stride + in_page);
        return 0;
      }
    };
    unsigned key_offset[(16 * S::kRow + 1023) / 1024];   // of this lane within its wave's 16 tokens
#pragma unroll
    for (int i = 0; i < (16 * S::kRow + 1023) / 1024; ++i) {
      constexpr int kPieces = S::kRow / 16;
      const int token = i * (64 / kPieces) + lane / kPieces;
      key_offset[i] = token * S::kRow + ((lane % kPieces) ^ S::key_swizzle(16 * wave + token)) * 16;
    }
    const auto request_keys = [&](int tile, int pg, int buffer) {
      const unsigned at = lds + buffer * S::kBuffer;
      const uint8_t* base;
      unsigned off = place(p.c.k, p.c.k_page_stride, pg, tile, S::kRow, base);
#pragma unroll
      for (int i = 0; i < (16 * S::kRow + 1023) / 1024; ++i)
        if (D > 64 || lane < 32) to_lds16(base, off + key_offset[i], at + wave * (16 * S::kRow) + i * 1024);
      off = place(p.c.k_scale, p.c.k_scale_page_stride, pg, tile, S::kBlocks, base);
      if (lane < 4 * S::kBlocks) to_lds4(base, off + lane * 4, at + S::kKeys + wave * (16 * S::kBlocks));
    };
    const auto request_values = [&](int tile, int pg) {
      const uint8_t* base;
      unsigned off = place(p.c.v, p.c.v_page_stride, pg, tile, S::kRow, base) + lane * S::kThreadBytes;
#pragma unroll
      for (int k = 0; k < Values<D>::kWords; k += 2) {
        const v2i x = *reinterpret_cast<const v2i*>(base + (off + 4 * k));
        next.code[k] = (unsigned)x[0], next.code[k + 1] = (unsigned)x[1];
      }
      off = place(p.c.v_scale, p.c.v_scale_page_stride, pg, tile, S::kBlocks, base) + Values<D>::scales_at(lane);
      next.scales = *reinterpret_cast<const unsigned*>(base + off);
    };
    const auto store_values = [&](int tile, int buffer) {   // what no key occupies, and what has a NaN scale, is zero
      const int here = lane_here(), token = 16 * wave + here / 4;
      const bool there = tile * kTile + token < it.s.len;
      const unsigned at = lds + kBuffers * S::kBuffer + buffer % S::kValueBuffers * S::kValues + token * (2 * D) + ((here % 4 * Values<D>::kWords) ^ S::value_swizzle(token)) * 16;
      uint64_t any = 0;
#pragma unroll
      for (int k = 0; k < Values<D>::kScaleBytes; ++k) {
        constexpr int kOfScale = Values<D>::kWords / Values<D>::kScaleBytes;
        const unsigned scale = next.scales >> (Values<D>::shift(here) + 8 * k) & 255;
        const bool bad = there && scale >= 253, none = bad || !there;
        const float f = __builtin_bit_cast(float, none ? 0x3F800000u : scale << 23);
#pragma unroll
        for (int w = k * kOfScale; w < (k + 1) * kOfScale; ++w) {   // eight channels, one 16-byte piece
          const unsigned x = none ? 0 : next.code[w];
          const v2bf a0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, f, 0), a1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, f, 1);
          const v2bf a2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, f, 2), a3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, f, 3);
          *lds_at<Lds8Bf16>(at ^ 16 * w) = v8bf{a0[0], a0[1], a1[0], a1[1], a2[0], a2[1], a3[0], a3[1]};
        }
        const uint64_t lanes = __ballot(bad);
        any |= lanes;
        if (lane == 0) nan_in[buffer][k][wave] = lanes;
      }
      if (lane == 0) nan_any[buffer][wave] = any != 0;
    };

    // ---- the queries' loads, then the first requests.  Queries: lane (column lane % 32): bytes 0-15 of a step are k = 16 h .., bytes 16-31
    // k = 32 + 16 h ..
    int entry = tiles > 0 ? entry_of(tile0 + 1) : 0;
    v8i q_hi[S::kSteps], q_lo[S::kSteps];   // (of q_lo the first kFar steps lie in LDS instead, as registers are short)
    int q_scale;   // of the first part; of the second in the next byte
    {
      const int first_entry = tiles > 0 ? entry_of(tile0) : 0, here = lane_here(), row = row0 + here % 32;
      const bool real = row < rows;
      const int t = real ? p.token_of(row) : 0, query_head = it.head * p.group + (real ? row - t * p.group : 0);
      const uint16_t* q = p.a.q + (int64_t)(it.s.first + t) * p.a.q_token_stride + (int64_t)query_head * p.a.q_head_stride + here / 32 * 16;
      v4i x[S::kSteps][4];
#pragma unroll
      for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) x[i][k] = v4i{0, 0, 0, 0};
      if (real) {
        if (p.q_aligned) {
#pragma unroll
          for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) x[i][k] = load8_bf16(q + 64 * i + 32 * (k / 2) + 8 * (k % 2), true);
        } else {
#pragma unroll
          for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) x[i][k] = load8_bf16(q + 64 * i + 32 * (k / 2) + 8 * (k % 2), false);
        }
      }
      if (tiles > 0) {
        const int page = page_of(p, first_entry);
        request_keys(tile0, page, 0);
        request_values(tile0, page);
      }
      us2 m = {0, 0};
#pragma unroll
      for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) m = amax_pairs(x[i][k], m);
      const QueryScale s = query_scale(lane_xor_max_bits(larger_half(m), 32));
      const int sign = p.a.scale < 0.0f ? (int)0x80808080u : 0;
#pragma unroll
      for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          int hi[2], lo[2];
          split_query(x[i][k], s, hi, lo);
#pragma unroll
          for (int e = 0; e < 2; ++e) q_hi[i][2 * k + e] = hi[e] ^ sign, q_lo[i][2 * k + e] = lo[e] ^ sign;
        }
#pragma unroll
      for (int i = 0; i < S::kFar; ++i) far_q[2 * i][tid] = q_lo[i].lo, far_q[2 * i + 1][tid] = q_lo[i].hi;
      q_scale = s.hi_byte | s.lo_byte << 8;
    }

    v16f acc[C];
#pragma unroll
    for (int k = 0; k < C; ++k) acc[k] = v16f{};
    float m = kNoMax, l = 0.0f;   // m: base 2

    // ---- 32 keys, half j of a tile.  What the matrix instructions take out of LDS is read ahead of them, by hand: the compiler, short of
    // registers, waits for each piece.
    constexpr int kAhead = 3;   // fragments of values on their way
    struct Keys {
      v4i code[S::kSteps];
      unsigned scale[(S::kBlocks + 3) / 4];
    };
    const auto read_keys = [&](int buffer, int j, const v4i& at_lane, Keys& f) {
      const unsigned at = at_lane[0] + buffer * S::kBuffer, ks = at_lane[1] + buffer * S::kBuffer + 32 * j * S::kBlocks;
      if constexpr (D == 64) {
        f.scale[0] = *lds_at<const LdsShort>(ks);
      } else {
#pragma unroll
        for (int k = 0; k < S::kBlocks / 4; ++k) f.scale[k] = lds_at<const LdsInt>(ks)[k];
      }
#pragma unroll
      for (int k = 0; k < S::kSteps; ++k) f.code[k] = *lds_at<const LdsInt4>((at ^ 32 * k) + 32 * j * S::kRow);
    };
    const auto scores = [&](const Keys& f, int shift) {
      v16f s = {};
#pragma unroll
      for (int k = 0; k < S::kSteps; ++k) {
        const v4i x = f.code[k];
        const v8i x8 = {x[0], x[1], x[2], x[3], 0, 0, 0, 0};
        const int scale = (int)(f.scale[k / 2] >> shift);
        v8i low = q_lo[k];
        if (k < S::kFar) low.lo = far_q[2 * k][tid], low.hi = far_q[2 * k + 1][tid];
        if (k % 2 == 0) {
          s = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x8, low, s, kFmtFp4, 0, 0, scale, 1, q_scale);
          s = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x8, q_hi[k], s, kFmtFp4, 0, 0, scale, 0, q_scale);
        } else {
          s = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x8, low, s, kFmtFp4, 0, 2, scale, 1, q_scale);
          s = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x8, q_hi[k], s, kFmtFp4, 0, 2, scale, 0, q_scale);
        }
      }
      return s;
    };
    const auto read_values = [&](unsigned at, int j, int n) {   // 16 of the 32 keys (n / C), 32 channels (n % C)
      typedef short v8s __attribute__((ext_vector_type(8)));
      at = (at ^ 64 * (n % C)) + (32 * j + 8 * (n / C)) * (2 * D);
      const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<LdsShort4>(at));
      const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<LdsShort4>(at + 4 * 2 * D));
      return __builtin_bit_cast(v8bf, v8s{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
    };
    // Probabilities from scores.  Any reference will do that keeps them in range, so the scores' maximum is looked for only where a lane's
    // sixteen come to more than 2^8 (the first ones that a row sees: to infinity): up to there they have the same relative error, and most
    // steps go without.
    const auto probabilities = [&](int tile, auto which, bool first, v16f& s, unsigned (&prob)[8]) {   // first: of the item
      constexpr int j = decltype(which)::value;
      const int key0 = tile * kTile + 32 * j + keys_from;
      if (key0 < lo_max || key0 + 32 > hi_min) {
        const int here = lane_here();
        if constexpr (kTree<A>) {
          const unsigned seen = tree_bits(p, it.s, row0 + here % 32, rows, key0 + here / 32 * 16);
#pragma unroll
          for (int t = 0; t < 16; ++t) s[t] = seen >> t & 1 ? s[t] : kNone;
        } else {
          int lo, hi;
          visible(p, it.s, p.token_of(row0 + here % 32), lo, hi);   // (a row behind the last: whatever)
          const int from = lo - key0 - here / 32 * 16;
          const unsigned many = (unsigned)(hi > lo ? hi - lo : 0);
#pragma unroll
          for (int t = 0; t < 16; ++t) s[t] = (unsigned)(t - from) < many ? s[t] : kNone;
        }
      }
      float sum;
      const auto exponentials = [&](float reference) {
        sum = 0.0f;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * t], c, -reference)), d = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * t + 1], c, -reference));
          sum += a;
          sum += d;
          prob[t] = pack_bf16x2(a, d);
          asm volatile("" : "+v"(prob[t]));   // here, not where it is used
        }
      };
      bool over = true;
      if (!first) {
        exponentials(m);
        over = !(sum <= 256.0f);
      }
      if (__any(over)) {   // a row by itself: what others hold leaves it as it is
        const float top = cross_max<false>(largest_of<0, 15>(s, kNone)), to_row = fmaxf(m, top > 0.5f * kNone ? top * c : kNoMax);
        const float to = cross_max<false>(over ? 1.0f : 0.0f) != 0.0f ? to_row : m, fade = __builtin_amdgcn_exp2f(m - to);
        l *= fade;
#pragma unroll
        for (int k = 0; k < C; ++k) acc[k] *= fade;
        m = to;
        exponentials(m == kNoMax ? 0.0f : m);
      }
      l += sum;
    };
    const auto add_values = [&](int tile, int buffer, auto which, const unsigned (&prob)[8], int nan, const v4i& place, v8bf (&v)[kAhead], Keys& keys) {
      const unsigned at = place[2] + buffer % S::kValueBuffers * S::kValues;
      constexpr int j = decltype(which)::value;
      // ---- values with a NaN scale, zeros in LDS: NaN for the rows that see them, however little they count
      if (nan) {
        const int here = lane_here(), key = tile * kTile + 32 * j + keys_from + here / 32 * 16;
        uint64_t some;   // four bits for each of this lane's 16 keys
        if constexpr (kTree<A>) {
          const unsigned seen = tree_bits(p, it.s, row0 + here % 32, rows, key);
          some = 0;
#pragma unroll
          for (int t = 0; t < 16; ++t) some |= (seen >> t & 1 ? 0xFull : 0ull) << 4 * t;
        } else {
          int lo, hi;
          visible(p, it.s, p.token_of(row0 + here % 32), lo, hi);
          const int from = lo - key, to = hi - key;
          some = (to > 15 ? ~0ull : to > 0 ? (1ull << 4 * to) - 1 : 0ull) & (from > 15 ? 0ull : from > 0 ? ~0ull << 4 * from : ~0ull);
        }
#pragma unroll
        for (int k = 0; k < C; ++k) {   // lane 4 t + quarter of a wave holds channels of block k
          const int quarter = D == 64 ? 2 * k : D == 128 ? k : k / 2;
          const uint64_t* lanes = nan_in[buffer][D == 256 ? k % 2 : 0] + 2 * j + keys_from / 16;
          const bool hit = ((lane < 32 ? lanes[0] : lanes[1]) & some & (0x1111111111111111ull << quarter)) != 0;
          acc[k] += cross_max<false>(hit ? 1.0f : 0.0f) != 0.0f ? __builtin_nanf("") : 0.0f;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < 2 * C; ++n) {
        const v4i w = {(int)prob[4 * (n / C)], (int)prob[4 * (n / C) + 1], (int)prob[4 * (n / C) + 2], (int)prob[4 * (n / C) + 3]};
        acc[n % C] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[n % kAhead], __builtin_bit_cast(v8bf, w), acc[n % C], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (n + kAhead < 2 * C) v[n % kAhead] = read_values(at, j, n + kAhead);
        if (SPLIT == 1 && j == 0 && n + kAhead == 2 * C) read_keys(buffer, 1, place, keys);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    const auto half_tile = [&](int tile, int buffer, auto which, bool first, int& nan, const v4i& place, Keys& keys) {
      constexpr int j = decltype(which)::value;
      v8bf v[kAhead];
      unsigned prob[8];
      if constexpr (j == 0) read_keys(buffer, 0, place, keys);
      v4i any;
      if constexpr (j == 0) any = *reinterpret_cast<const v4i*>(nan_any[buffer]);
      v16f s = scores(keys, place[3]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < kAhead; ++n) v[n] = read_values(place[2] + buffer % S::kValueBuffers * S::kValues, j, n);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (j == 0) nan = uniform(any[0] | any[1] | any[2] | any[3]);
      probabilities(tile, which, first, s, prob);
      add_values(tile, buffer, which, prob, nan, place, v, keys);
    };

    if (tiles > 0) store_values(tile0, 0);
    wait_loads<0>();
    __syncthreads();
    for (int i = 0; i < tiles; ++i) {
      const int tile = tile0 + i, buffer = i & 1;
      v4i place = places[lane];
      if constexpr (SPLIT == 2) place += v4i{keys_from * S::kRow, keys_from * S::kBlocks, keys_from * 2 * D, 0};
      if constexpr (waves_per_simd<D>() > 1) {
        if (turn < late) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
        turn = turn + 1 < waves_per_simd<D>() ? turn + 1 : 0;
      }
      if (i + 1 < tiles) {
        const int page = page_of(p, entry);
        request_values(tile + 1, page);
        request_keys(tile + 1, page, buffer ^ 1);
        entry = entry_of(tile + 2);
      }
      if constexpr (SPLIT == 2) {
        if (active && tile * kTile + keys_from < hi_max && tile * kTile + keys_from + 32 > lo_min) {
          int nan = 0;
          Keys keys;
          half_tile(tile, buffer, Index<0>{}, i == 0, nan, place, keys);
        }
      } else if (active && tile * kTile < hi_max && tile * kTile + kTile > lo_min) {
        int nan = 0;
        Keys keys;
        half_tile(tile, buffer, Index<0>{}, i == 0, nan, place, keys);
        if (tile * kTile + 32 < hi_max) half_tile(tile, buffer, Index<1>{}, false, nan, place, keys);
      }
      if constexpr (S::kValueBuffers == 1) __syncthreads();
      if (i + 1 < tiles) store_values(tile + 1, buffer ^ 1);
      wait_loads<0>();
      __syncthreads();
    }

    if constexpr (SPLIT == 2) {   // waves 2 and 3 leave their sums in the values' place, waves 0 and 1 add them to their own
      constexpr int kAtOnce = S::kValues * S::kValueBuffers / (2 * 64 * 64);   // blocks of 32 channels that fit there
      const unsigned at = lds + kBuffers * S::kBuffer + wave % 2 * (kAtOnce * 4096) + lane * 16;
      const float sum = cross_sum<false>(l);
      float(&ml)[32][2] = other_ml[wave % 2];
      if (wave >= 2 && lane < 32) ml[lane][0] = m, ml[lane][1] = sum;
      float f0 = 0.0f, f1 = 0.0f;
#pragma unroll
      for (int first = 0; first < C; first += kAtOnce) {
        if (wave >= 2) {
#pragma unroll
          for (int k = first; k < first + kAtOnce && k < C; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *lds_at<LdsFloat4>(at + (4 * (k - first) + i) * 1024) = v4f{acc[k][4 * i], acc[k][4 * i + 1], acc[k][4 * i + 2], acc[k][4 * i + 3]};
        }
        __syncthreads();
        if (wave < 2) {
          if (first == 0) {
            const float m1 = ml[lane % 32][0], top = fmaxf(m, m1);
            f0 = __builtin_amdgcn_exp2f(m - top), f1 = __builtin_amdgcn_exp2f(m1 - top);
            l = lane < 32 ? sum * f0 + ml[lane % 32][1] * f1 : 0.0f;   // (both halves of the wave are added up below)
            m = top;
          }
#pragma unroll
          for (int k = first; k < first + kAtOnce && k < C; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const v4f x = *lds_at<const LdsFloat4>(at + (4 * (k - first) + i) * 1024);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[k][4 * i + e] = acc[k][4 * i + e] * f0 + x[e] * f1;
            }
        }
        __syncthreads();   // (the next ones, and the results, go by way of the same LDS)
      }
    }

    // ---- results: lane (column lane % 32) has channels 32 k + 8 i + 4 (lane / 32) .. + 3 of its row
    const bool done = from == 0 && to == it.units;
    if (active && (SPLIT == 1 || wave < 2)) {
      const float sum = cross_sum<false>(l), m2 = m == kNoMax ? -INFINITY : m;
      const int here = lane_here(), row = row0 + here % 32, ch0 = here / 32 * 4;
      const bool real = row < rows;
      if (done) {   // by way of LDS, whose values nobody needs any more, so that whole rows are stored (16 bytes a row at a time: 6000 cycles an item)
        float factor = 0.0f;
        if (real) {
          const RowEnd e = row_end(sink_of(p, it.head * p.group + (row - p.token_of(row) * p.group)), m2, sum);
          if (p.a.lse && ch0 == 0) p.a.lse[row_index(p, it.s.first, it.head, row)] = e.lse;
          factor = e.factor;
        }
        constexpr int kWide = D < 128 ? D : 128, kPieces = kWide / 8, kAtOnce = 64 / kPieces;   // channels at a time, 16-byte pieces of them, rows of a store
        const unsigned own = lds + kBuffers * S::kBuffer + wave * (32 * 2 * kWide);
#pragma unroll
        for (int wide = 0; wide < D / kWide; ++wide) {
#pragma unroll
          for (int k = 0; k < kWide / 32; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const v16f& a = acc[wide * (kWide / 32) + k];
              *lds_at<LdsInt2>(own + here % 32 * (2 * kWide) + ((4 * k + i) ^ (here % kPieces)) * 16 + ch0 * 2) =
                  v2i{(int)pack_bf16x2(a[4 * i] * factor, a[4 * i + 1] * factor), (int)pack_bf16x2(a[4 * i + 2] * factor, a[4 * i + 3] * factor)};
            }
#pragma unroll
          for (int n = 0; n < 32 / kAtOnce; ++n) {
            const int r = n * kAtOnce + here / kPieces;
            const v4i x = *lds_at<const LdsInt4>(own + r * (2 * kWide) + ((here % kPieces) ^ (r % kPieces)) * 16);
            if (row0 + r < rows) *reinterpret_cast<Loose4*>(p.a.out + row_index(p, it.s.first, it.head, row0 + r) * D + wide * kWide + here % kPieces * 8) = x;
          }
        }
      } else if (real) {
        const size_t slot = 2 * (size_t)g + (from == 0 ? 1 : 0), at = slot * kRows + (row - it.row0);
        float* out = p.part_o + at * D + ch0;
#pragma unroll
        for (int k = 0; k < C; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<v4f*>(out + 32 * k + 8 * i) = v4f{acc[k][4 * i], acc[k][4 * i + 1], acc[k][4 * i + 2], acc[k][4 * i + 3]};
        if (ch0 == 0) p.part_ml[at * 2] = m2, p.part_ml[at * 2 + 1] = sum;
      }
    }
    if (done) __syncthreads();   // before the next item's values
  }
}

int workgroups_of(const AttnArgs& p) {
  const int d = p.c.head_dim;
  return compute_units() * (d == 64 ? waves_per_simd<64>() : d == 128 ? waves_per_simd<128>() : waves_per_simd<256>());
}
template <int D, int SPLIT, typename A>
void launch(const A& p, int workgroups, hipStream_t s) {
  const dim3 grid((unsigned)workgroups), block(kWaves * 64);
  const int64_t last = p.c.pages - 1, page = (int64_t)p.c.kv_heads * p.c.page_size * D / 2;   // bytes of codes; of scales a 16th
  const auto small = [&](int64_t stride, int64_t bytes) { return last * stride + bytes <= (int64_t)1 << 32; };
  const bool all = small(p.c.k_page_stride, page) && small(p.c.v_page_stride, page) && small(p.c.k_scale_page_stride, page / 16) && small(p.c.v_scale_page_stride, page / 16);
  if (units_bound(p, kMostRows / SPLIT, kTile) >> 32) hipLaunchKernelGGL((attn_prompt_kernel<D, false, Units, A, SPLIT>), grid, block, 0, s, p);   // (a call of seconds)
  else if (all) hipLaunchKernelGGL((attn_prompt_kernel<D, true, unsigned, A, SPLIT>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((attn_prompt_kernel<D, false, unsigned, A, SPLIT>), grid, block, 0, s, p);
}

}  // namespace

size_t attn_prompt_workspace(const AttnArgs& p) { return attn_workspace(kMostRows, p.c.head_dim, workgroups_of(p)); }

namespace {
int64_t rows_of(const AttnArgs& p) { return p.a.cu_q ? (int64_t)p.a.max_q * p.group : p.group; }
// Rows of a block, for trees: 64 where there are no more, and where few blocks of few tiles leave waves without work.  us in blocks of 64 and of 128, 32
// heads on 8 of 128: 16 sequences of 4096 keys, 16 nodes (64 rows) 40 and 42; 4 of 4096, 64 nodes (256 rows) 40 and 45, 16 of them 86 and 79; one of
// 131072, 64 nodes 132 and 116; 64 heads on 8 of 64, 64 sequences of 1000, 16 nodes (128 rows) 37 and 47, 128 of 300 49 and 29.  (The bound on a sequence's keys is
// what the page table or the window can hold.)
int tree_block(const TreeArgs& p) {
  const int64_t rows = rows_of(p), items = (int64_t)p.a.batch * p.c.kv_heads * ((rows + kMostRows - 1) / kMostRows), slots = workgroups_of(p);
  const int64_t in_table = (int64_t)p.a.table_pages << p.page_shift, in_window = p.a.window > 0 ? (int64_t)p.a.window + p.a.max_q : in_table;
  const int64_t tiles = (in_window < in_table ? in_window : in_table) / kTile + 1;
  return rows <= kMostRows / 2 || (2 * items <= slots && items * tiles <= 8 * slots) ? kMostRows / 2 : kMostRows;
}

template <int D>
hipError_t launch_of(AttnArgs p, void* ws, hipStream_t s) {
  const int workgroups = workgroups_of(p);
  p.whole = 0;
  // In parts: 2048 new tokens of 2 sequences of 16384 keys, 128 channels, with 1 950 us, 2 950, 3 947, 4 948; 300 prompts of 60 tokens, whose items have
  // but one tile, 100, 107, 118, 118; 64 channels 106, 113, 112, 115.  (It also counts in the choice of whole items, whose bound was measured with it.)
  p.item_units = D == 64 ? 2 : 3;
  p.min_units_log2 = 2;
  p.few_long = p.a.batch <= 8;   // (one sequence, 4096 new tokens on 65536 keys: 3734 us so, 3771 otherwise; 8 with 40 on 2300: 54 and 49; 300 prompts of 60: 315 and 118)
  place_workspace(p, kMostRows, workgroups, ws);
  launch<D, 1>(p, workgroups, s);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  return launch_attn_combine(p, kMostRows, rows_of(p), workgroups, s);
}
template <int D>
hipError_t launch_of(TreeArgs p, void* ws, hipStream_t s) {
  const int workgroups = workgroups_of(p), rows = tree_block(p);
  p.whole = 0;
  p.item_units = 3;
  p.min_units_log2 = 2;
  p.starts = static_cast<PartStart*>(ws);
  place_workspace(p, rows, workgroups, static_cast<char*>(ws) + attn_starts_bytes(workgroups));
  if (rows < kMostRows) launch<D, 2>(p, workgroups, s);
  else launch<D, 1>(p, workgroups, s);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  return launch_attn_join(p, rows, rows_of(p), workgroups, s);
}
}  // namespace

size_t attn_prompt_workspace(const TreeArgs& p) { return attn_starts_bytes(workgroups_of(p)) + attn_workspace(tree_block(p), p.c.head_dim, workgroups_of(p)); }

template <typename A>
hipError_t launch_attn_prompt(A p, void* ws, hipStream_t s) {
  if (p.c.head_dim == 64) return launch_of<64>(p, ws, s);
  if (p.c.head_dim == 128) return launch_of<128>(p, ws, s);
  return launch_of<256>(p, ws, s);
}
template hipError_t launch_attn_prompt(AttnArgs p, void* ws, hipStream_t s);
template hipError_t launch_attn_prompt(TreeArgs p, void* ws, hipStream_t s);

}  // namespace ave
