// Attention of few query rows over a paged MXFP4 cache: single tokens of a decode batch, a handful of tokens of a draft.
//
// Bound by HBM: a token's key and value are 34 bytes per 32 channels, read once.  A workgroup walks its share of the call's
// units (64 keys, attn_common.hpp); its waves take the units of an item in turn, each through LDS stages of its own that are filled
// straight from memory, and meet at the item's end only.
//
//   S^T = K Q^T   scaled MFMA 16x16x128, keys as they are (E2M1, E8M0), queries as two E4M3 parts.  Which token is row r of key
//                 tile j is free: token 16 (r / 4) + 4 j + r % 4, so that lane group g = lane / 16 of the result holds the scores of
//                 tokens 16 g .. 16 g + 15 for query row lane % 16.
//   P             bf16 of exp(s - max), the running maximum shared by the four groups; sums per lane, in fp32, of what is not rounded
//   O^T = V^T P^T bf16 MFMA 16x16x32: lane group g multiplies its own 16 tokens, so P stays in its registers.  A transposing LDS read
//                 (4 bits) gives a lane 16 tokens' codes of one channel, two per conversion.  The E8M0 scales of the values differ from
//                 token to token, the contracted axis: they go into P as integer additions to the bf16 exponent, one copy of P per
//                 32 channels -- exact, saturating at zero.
//
// P is rounded to bf16 because the values' codes reach the matrix cores as bf16 without loss and the result is bf16 anyway: 2^-9 of a
// probability, averaged over the keys.  Scores, maxima, sums and results are fp32.
//
// 32 heads on 8 of 128: 64 sequences of 2048 to 4096 keys 52 us (4.1 TB/s; of 16384 keys each 6.0, of 256 channels 6.1, of 64 5.4), one of
// 131072 38 us.  A plain read of as many bytes takes 36 and 25 us; the rest is the second launch (7 with the gap in front of it) and the way from the
// lengths by the table to the first keys.  Non-temporal hints on what nobody else reads gave 4 us (58.5 and 43 before, 16384 keys 215 to 199).  For
// up to 16 rows four waves with two stages each, two workgroups a compute unit, read ahead best (eight waves, one workgroup: 63 and 45 us where this
// came to 58 and 42); items that stay whole get eight waves, which halve their way.
#include "attn_common.hpp"
#include "kernels.hpp"

namespace ave {
namespace {

template <int D>
struct Shape {
  static constexpr int kRow = D / 2, kBlocks = D / 32;                     // bytes of a token's codes and scales
  static constexpr int kCodes = 64 * kRow, kScales = 64 * kBlocks;         // of a stage
  static constexpr int kStage = 2 * kCodes + 2 * kScales;
  static constexpr int kLoads = 2 * (kCodes / 1024) + (D == 64 ? 1 : 2 * kScales / 256);
  // 16-byte pieces of a row are permuted in LDS so that the 16 lanes of a read touch different banks
  __device__ static int key_swizzle(int t) { return D == 64 ? (t >> 4) & 1 : D == 128 ? (t >> 4) & 3 : ((t >> 1) & 1) | ((t >> 4) & 3) << 1; }
  __device__ static int value_swizzle(int t) { return D == 64 ? (t >> 3) & 1 : D == 128 ? (t >> 2) & 3 : (t >> 1) & 7; }
};


// (values, not the elements of an array: a choice of elements would keep the array in memory)
__device__ inline const uint8_t* pick(bool first, const uint8_t* a, const uint8_t* b) { return first ? a : b; }

// Requests for stages.  ONE_PAGE: pages of 64 tokens and more, so that a stage lies in one page and its addresses are a scalar base and
// a lane's fixed offset (four groups of 16 tokens in pages of their own cost four times the scalar arithmetic: 64 sequences of 16384 keys 190 us in pages of 64, 204 in
// pages of 16).
template <int D, bool ONE_PAGE>
struct Request {
  using S = Shape<D>;
  static constexpr int kPieces = S::kRow / 16, kTokens = 1024 / S::kRow;   // pieces of a row, tokens of an instruction
  static constexpr int kN = S::kCodes / 1024;
  static constexpr int kGroups = ONE_PAGE ? 1 : 4, kGroupTokens = 64 / kGroups;
  unsigned key[kN], value[kN];   // byte offsets of this lane's pieces within a group of tokens that lie in one page

  __device__ inline Request() {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int t = i * kTokens + lane / kPieces;
      key[i] = t % kGroupTokens * S::kRow + ((lane % kPieces) ^ S::key_swizzle(t)) * 16;
      value[i] = t % kGroupTokens * S::kRow + ((lane % kPieces) ^ S::value_swizzle(t)) * 16;
    }
  }

  // The 64 keys and values from token t0 on (a multiple of 64) of a sequence of len > 0 keys into the stage at `lds`
  __device__ inline void stage(const AttnArgs& p, ConstInts table, int len, int head, int t0, unsigned lds) const {
    const int lane = threadIdx.x & 63;
    int page[kGroups];
    unsigned row[kGroups];   // within a page (all heads): below 2^30 / kRow
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      page[i] = page_at(p, table, t0 + kGroupTokens * i, len);
      row[i] = (unsigned)(head * p.c.page_size + ((t0 + kGroupTokens * i) & (p.c.page_size - 1)));
    }
    // codes: 1 KB an instruction
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const uint8_t* base[kGroups];
#pragma unroll
      for (int i = 0; i < kGroups; ++i)
        base[i] = (kv ? p.c.v + page[i] * p.c.v_page_stride : p.c.k + page[i] * p.c.k_page_stride) + row[i] * (unsigned)S::kRow;
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const unsigned off = kv ? value[i] : key[i], at = lds + kv * S::kCodes + i * 1024;
        if constexpr (ONE_PAGE) to_lds16<true>(base[0], off, at);
        else if constexpr (kTokens > 16) to_lds16(pick(lane < 32, base[2 * i % kGroups], base[(2 * i + 1) % kGroups]) + off, at);   // two groups
        else to_lds16<true>(base[i * kTokens / 16 % kGroups], off, at);
      }
    }
    // scales: a lane's four bytes belong to the tokens of one group
    const auto scales = [&](const uint8_t* from, int64_t stride, int offset) {   // of the stage's kScales bytes
      const uint8_t* base[kGroups];
#pragma unroll
      for (int i = 0; i < kGroups; ++i) base[i] = from + page[i] * stride + row[i] * (unsigned)S::kBlocks;
      if constexpr (ONE_PAGE) return base[0] + offset;
      const int t = offset / S::kBlocks;
      return pick(t < 32, pick(t < 16, base[0], base[1 % kGroups]), pick(t < 48, base[2 % kGroups], base[3 % kGroups])) + offset % (16 * S::kBlocks);
    };
    if constexpr (D == 64) {   // keys' scales by lanes 0-31, values' by 32-63
      const uint8_t *a = scales(p.c.k_scale, p.c.k_scale_page_stride, lane % 32 * 4), *b = scales(p.c.v_scale, p.c.v_scale_page_stride, lane % 32 * 4);
      to_lds4(lane < 32 ? a : b, lds + 2 * S::kCodes);
    } else {
#pragma unroll
      for (int i = 0; i < S::kScales / 256; ++i) {
        to_lds4(scales(p.c.k_scale, p.c.k_scale_page_stride, i * 256 + lane * 4), lds + 2 * S::kCodes + i * 256);
        to_lds4(scales(p.c.v_scale, p.c.v_scale_page_stride, i * 256 + lane * 4), lds + 2 * S::kCodes + S::kScales + i * 256);
      }
    }
  }
};

// The queries of a block of rows: 16 rows a tile, a tile's parts in the layout of the 16x16x128 MFMA (lane: column lane % 16; bytes 0-15 are
// k = 16 g .., bytes 16-31 k = 64 + 16 g ..).  D = 64: one MFMA takes both parts, the second in the place of k >= 64.
template <int D, int NT>
struct Queries {
  static constexpr int kSteps = D == 64 ? 1 : D / 128;
  v8i hi[NT][kSteps], lo[NT][D == 64 ? 1 : kSteps];
  int s_hi[NT], s_lo[NT];
  v4i x[NT][D / 32];   // eight channels each: pairs of them at 16 g + 64 i

  __device__ inline void request(const AttnArgs& p, const Sequence& s, int head, int row0, int rows) {
    const int lane = threadIdx.x & 63, g = lane / 16;
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      const int row = row0 + ct * 16 + lane % 16;
      const bool real = row < rows;
      const int t = real ? p.token_of(row) : 0;
      const uint16_t* q = p.a.q + (int64_t)(s.first + t) * p.a.q_token_stride + (int64_t)(head * p.group + (real ? row - t * p.group : 0)) * p.a.q_head_stride;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        x[ct][i] = v4i{0, 0, 0, 0};
        if (real) x[ct][i] = load8_bf16(q + (i / 2) * 64 + g * 16 + (i % 2) * 8, p.q_aligned);
      }
    }
  }
  __device__ inline void convert(const AttnArgs& p) {
    const int g = (threadIdx.x & 63) / 16;
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      us2 m = {0, 0};
#pragma unroll
      for (int i = 0; i < D / 32; ++i) m = amax_pairs(x[ct][i], m);
      const QueryScale s = query_scale(lane_xor_max_bits(lane_xor_max_bits(larger_half(m), 16), 32));
      const int sign = p.a.scale < 0.0f ? (int)0x80808080u : 0;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        int h[2], l[2];
        split_query(x[ct][i], s, h, l);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if constexpr (D == 64) hi[ct][0][i * 2 + k] = h[k] ^ sign, hi[ct][0][4 + i * 2 + k] = l[k] ^ sign;
          else hi[ct][i / 4][i % 4 * 2 + k] = h[k] ^ sign, lo[ct][i / 4][i % 4 * 2 + k] = l[k] ^ sign;
        }
      }
      s_hi[ct] = D == 64 && g >= 2 ? s.lo_byte : s.hi_byte;
      s_lo[ct] = s.lo_byte;
    }
  }
};

// LDS of a workgroup (stages, or the waves' results when they meet), and how many workgroups fit the 160 KB of a compute unit
template <int D, int NT, int NW, int NS>
constexpr int lds_bytes() {
  constexpr int kRing = NW * NS * Shape<D>::kStage, kJoin = NW * NT * 16 * (D + 4) * 4;
  return kRing > kJoin ? kRing : kJoin;
}
template <int D, int NT, int NW, int NS>
constexpr int workgroups_per_cu() {
  return lds_bytes<D, NT, NW, NS>() <= 78 * 1024 ? 2 : 1;
}

template <int D, int NT, int NW, int NS, bool ONE_PAGE, typename U, typename A>
__global__ __launch_bounds__(NW * 64, (workgroups_per_cu<D, NT, NW, NS>() * NW / 4)) void attn_decode_kernel(A p) {
  using S = Shape<D>;
  constexpr int ROWS = NT * 16, TILE = 64, C = D / 16;   // C: channel tiles of 16
  constexpr bool kEarly = NT == 1;            // registers for a whole stage beside the rest
  constexpr int kPitch = D + 4;                          // floats of a row of a wave's result in LDS
  __shared__ __align__(16) unsigned char smem[lds_bytes<D, NT, NW, NS>()];
  __shared__ float join_ml[NW][ROWS][2];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63, g = lane / 16, col = lane % 16;
  const Part<U> part = take_part<ROWS, TILE, U>(p, blockIdx.x, gridDim.x);
  const unsigned ring = (unsigned)__builtin_amdgcn_readfirstlane(lds_address(smem)) + wave * NS * S::kStage;
  const unsigned char* ring_ptr = smem + wave * NS * S::kStage;
  const float c = softmax_scale(p.a.scale);
  const Request<D, ONE_PAGE> request;
  int b = part.b;
  U b_begin = part.b_begin, per_head = part.per_head;
  Sequence seq = part.s;
  bool first_item = true;
  if (!p.whole && threadIdx.x == 0 && part.u0 >= part.u1) {   // no work
    PartMeta& m = p.meta[blockIdx.x];
    m.u0 = m.begin = m.end = part.units;
  }
  for (U u = part.u0; u < part.u1;) {
    const Item<U> it = item_of<ROWS, TILE, U>(p, u, b, b_begin, seq, per_head);
    if (!p.whole && first_item && threadIdx.x == 0) p.meta[blockIdx.x] = {part.u0, it.begin, it.begin + it.units, it.s.first, it.s.n * p.group, it.head, it.row0};
    if (u - it.begin >= it.units) break;   // (lengths that change under the call: no walk without end, and the second launch finds its record)
    unsigned from = (unsigned)(u - it.begin), to = it.units;   // units of the item
    if (!p.whole) {
      if (part.u1 - it.begin < to) to = (unsigned)(part.u1 - it.begin);
      u = it.begin + to;
    } else {   // the items that start in this part, as wholes
      u = it.begin + it.units;
      if (it.begin < part.u0) {
        first_item = false;
        continue;
      }
      from = 0;
    }
    const int rows = it.s.n * p.group;
    const int tile0 = it.tile0 + (int)from, tiles = (int)(to - from);
    const ConstInts table = (ConstInts)(p.a.page_table + (int64_t)b * p.a.page_table_stride);

    // what the rows see
    int lo_row[NT], hi_row[NT], lo_max, hi_min;   // hi_row: of a tree the row's token
    {
      const int last = it.row0 + ROWS < rows ? it.row0 + ROWS - 1 : rows - 1;
      const Bounds all = bounds(p, it.s, p.token_of(it.row0), p.token_of(last));
      lo_max = all.lo_max, hi_min = all.hi_min;
#pragma unroll
      for (int ct = 0; ct < NT; ++ct) {
        const int row = it.row0 + ct * 16 + col, t = p.token_of(row < rows ? row : last);
        if constexpr (kTree<A>) lo_row[ct] = rows > 0 ? first_seen(p, it.s, t) : 0, hi_row[ct] = t;
        else visible(p, it.s, t, lo_row[ct], hi_row[ct]);
      }
    }
    const int mine = it.s.len > 0 && tiles > wave ? (tiles - wave + NW - 1) / NW : 0;   // tiles wave, wave + NW, ...
    Queries<D, NT> q;
    q.request(p, it.s, it.head, it.row0, rows);
    int requested = 0;
    for (; requested < (kEarly ? NS : NS - 1) && requested < mine; ++requested)
      request.stage(p, table, it.s.len, it.head, (tile0 + wave + requested * NW) * TILE, ring + requested * S::kStage);

    q.convert(p);

    v4f acc[NT][C];
    float m[NT], l[NT];
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      m[ct] = kNone, l[ct] = 0.0f;
#pragma unroll
      for (int i = 0; i < C; ++i) acc[ct][i] = v4f{0, 0, 0, 0};
    }

    for (int i = 0; i < mine; ++i) {
      const int t0 = (tile0 + wave + i * NW) * TILE;
      const auto request_next = [&] {
        if (requested < mine) {
          request.stage(p, table, it.s.len, it.head, (tile0 + wave + requested * NW) * TILE, ring + (requested % NS) * S::kStage);
          ++requested;
        }
      };
      if constexpr (!kEarly) request_next();
      const int behind = requested - 1 - i;   // stages requested behind this one: below NS
      if (NS > 3 && behind >= 3) wait_loads<(NS > 3 ? 3 : 0) * S::kLoads>();
      else if (NS > 2 && behind >= 2) wait_loads<(NS > 2 ? 2 : 0) * S::kLoads>();
      else if (NS > 1 && behind >= 1) wait_loads<(NS > 1 ? 1 : 0) * S::kLoads>();
      else wait_loads<0>();
      const unsigned char* st = ring_ptr + (i % NS) * S::kStage;
      const unsigned char *keys = st, *values = st + S::kCodes, *ks = st + 2 * S::kCodes, *vs = ks + S::kScales;

      // ---- the stage out of LDS
      constexpr int kSteps = Queries<D, NT>::kSteps, kScaleWords = S::kScales / 16, kCheck = (S::kScales + 255) / 256;
      const auto read_key = [&](int j, int step, v4i& x, int& scale) {
        const int t = 16 * (col / 4) + 4 * j + col % 4, block = D == 64 ? g % 2 : step * 4 + g;
        x = *reinterpret_cast<const v4i*>(keys + t * S::kRow + (block ^ S::key_swizzle(t)) * 16);
        scale = ks[t * S::kBlocks + block];
      };
      const auto read_value = [&](int ch) {
        const int t = 16 * g + col;
        const unsigned char* at = values + t * S::kRow + (ch / 2 ^ S::value_swizzle(t)) * 16 + ch % 2 * 8;
        return __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) v2i*)at);
      };
      const auto read_scale = [&](int k) { return reinterpret_cast<const unsigned*>(vs)[g * kScaleWords + k]; };   // of this group's 16 tokens
      v4i key[4][kSteps];
      int key_scale[4][kSteps];
      v2i value[C];
      unsigned value_scale[kScaleWords], check[kCheck];
#pragma unroll
      for (int k = 0; k < kCheck; ++k) {   // each word of the stage once, over the lanes
        const int at = k * 256 + lane * 4;
        check[k] = *reinterpret_cast<const unsigned*>(vs + (at < S::kScales ? at : 0));
      }
      if constexpr (kEarly) {   // all of it into registers: the buffer is free for the stage after next
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int step = 0; step < kSteps; ++step) read_key(j, step, key[j][step], key_scale[j][step]);
#pragma unroll
        for (int ch = 0; ch < C; ++ch) value[ch] = read_value(ch);
#pragma unroll
        for (int k = 0; k < kScaleWords; ++k) value_scale[k] = read_scale(k);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        request_next();
      }

      // ---- scores
      v4f s[NT][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int ct = 0; ct < NT; ++ct) s[ct][j] = v4f{0, 0, 0, 0};
#pragma unroll
        for (int step = 0; step < kSteps; ++step) {
          if constexpr (!kEarly) read_key(j, step, key[j][step], key_scale[j][step]);
          const v4i x = key[j][step];
          const v8i x8 = {x[0], x[1], x[2], x[3], 0, 0, 0, 0};
          const int sk = key_scale[j][step];
#pragma unroll
          for (int ct = 0; ct < NT; ++ct) {
            if constexpr (D != 64)
              s[ct][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x8, q.lo[ct][step], s[ct][j], kFmtFp4, 0, 0, sk, 0, q.s_lo[ct]);
            s[ct][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x8, q.hi[ct][step], s[ct][j], kFmtFp4, 0, 0, sk, 0, q.s_hi[ct]);
          }
        }
      }

      // ---- probabilities
      const bool all_seen = t0 >= lo_max && t0 + TILE <= hi_min;
      unsigned prob[NT][8], bias[NT][8];   // pairs of tokens 16 g + 2 i, + 1; what is taken from their exponents
      unsigned seen[NT];                   // of a tree: a bit for each of this group's 16 tokens
#pragma unroll
      for (int ct = 0; ct < NT; ++ct) {
        seen[ct] = 0xFFFFu;
        if constexpr (kTree<A>) {
          if (!all_seen) {
            seen[ct] = seen_of(p, it.s, hi_row[ct], lo_row[ct], t0 + 16 * g);
#pragma unroll
            for (int j = 0; j < 16; ++j) s[ct][j / 4][j % 4] = seen[ct] >> j & 1 ? s[ct][j / 4][j % 4] : kNone;
          }
        } else if (!all_seen) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const int key = t0 + 16 * g + 4 * j + t;
              s[ct][j][t] = key >= lo_row[ct] && key < hi_row[ct] ? s[ct][j][t] : kNone;
            }
        }
        float top = kNone;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float two = fmaxf(s[ct][j][0], s[ct][j][1]);
          top = fmaxf(top, max3(two, s[ct][j][2], s[ct][j][3], two));
        }
        top = fmaxf(m[ct], cross_max<true>(top));
        if (__any(top > m[ct])) {
          const float fade = __builtin_amdgcn_exp2f((m[ct] - top) * c);
          l[ct] *= fade;
#pragma unroll
          for (int k = 0; k < C; ++k) acc[ct][k] *= fade;
          m[ct] = top;
        }
        const float shift = m[ct] == kNone ? 0.0f : -m[ct] * c;
        float pr[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          pr[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ct][j / 4][j % 4], c, shift));
          l[ct] += pr[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          prob[ct][j] = pack_bf16x2(pr[2 * j], pr[2 * j + 1]);
          // 127 in the exponent's place, or more than everything for a probability of zero, which stays zero
          bias[ct][j] = pk_mad_u16(pk_sub_sat(0x00010001u, prob[ct][j]), 0xC07FC07Fu, 0x3F803F80u);
        }
      }

      // ---- values: a scale byte from 253 on (NaN) anywhere in the stage?  (also in what no key occupies: no row sees that)
      bool nan = false;
#pragma unroll
      for (int k = 0; k < kCheck; ++k) {
        const unsigned x = ~check[k];
        nan = nan || ((x - 0x03030303u) & ~x & 0x80808080u) != 0;
      }
      nan = __any(nan);
      // the scale bytes of tokens 16 g + 2 k and + 1 for a block of channels, in 16 bits each
      const auto scale_pair = [&](int blk, int k) -> unsigned {
        if constexpr (D == 64) {
          const unsigned w = kEarly ? value_scale[k] : read_scale(k);
          return __builtin_amdgcn_perm(w, w, blk ? 0x0c030c01u : 0x0c020c00u);
        } else {
          constexpr int kWords = S::kBlocks / 4;
          const int at = 2 * k * kWords + blk / 4;
          const unsigned w0 = kEarly ? value_scale[at] : read_scale(at), w1 = kEarly ? value_scale[at + kWords] : read_scale(at + kWords);
          return __builtin_amdgcn_perm(w1, w0, 0x0c040c00u + 0x00010001u * (blk % 4));
        }
      };
      if (nan) {   // a row that sees a value with a NaN scale, however little it counts: its block of channels is NaN
#pragma unroll
        for (int ct = 0; ct < NT && !kTree<A>; ++ct) {
          const int from = lo_row[ct] - t0 - 16 * g, to = hi_row[ct] - t0 - 16 * g;
          seen[ct] = (to > 15 ? 0xFFFFu : to > 0 ? (1u << to) - 1 : 0u) & (from > 15 ? 0u : from > 0 ? ~0u << from : ~0u);
        }
#pragma unroll
        for (int blk = 0; blk < S::kBlocks; ++blk) {
          unsigned bad = 0;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const unsigned over = pk_sub_sat(scale_pair(blk, k), 0x00FC00FCu);   // 1 to 3 in a half where NaN
            const unsigned two = (over | over >> 1) & 0x00010001u;
            bad |= ((two | two >> 15) & 3u) << 2 * k;
          }
#pragma unroll
          for (int ct = 0; ct < NT; ++ct) {
            const float poison = cross_max<true>(bad & seen[ct] ? 1.0f : 0.0f) != 0.0f ? __builtin_nanf("") : 0.0f;
            acc[ct][2 * blk] += poison;
            acc[ct][2 * blk + 1] += poison;
          }
        }
      }
#pragma unroll
      for (int blk = 0; blk < S::kBlocks; ++blk) {
        // P with the scales of this block of channels
        v4i ps[NT][2];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const unsigned e = scale_pair(blk, k);
#pragma unroll
          for (int ct = 0; ct < NT; ++ct) {
            const unsigned r = pk_sub_sat(pk_mad_u16(e, 0x00800080u, prob[ct][k]), bias[ct][k]);
            ps[ct][k / 4][k % 4] = (int)r;
          }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int ch = blk * 2 + half;
          const v2i w = kEarly ? value[ch] : read_value(ch);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const unsigned x = (unsigned)w[k];
            const v2bf a0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, 1.0f, 0), a1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, 1.0f, 1);
            const v2bf a2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, 1.0f, 2), a3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, 1.0f, 3);
            const v8bf a = {a0[0], a0[1], a1[0], a1[1], a2[0], a2[1], a3[0], a3[1]};
#pragma unroll
            for (int ct = 0; ct < NT; ++ct)
              acc[ct][ch] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(v8bf, ps[ct][k]), acc[ct][ch], 0, 0, 0);
          }
        }
      }
    }

    // ---- the waves' results joined
    __syncthreads();   // (no load is under way any more: every wave has waited for its last one)
    float* mine_o = reinterpret_cast<float*>(smem) + (size_t)wave * ROWS * kPitch;
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      const float sum = cross_sum<true>(l[ct]);
      if (g == 0) {
        join_ml[wave][ct * 16 + col][0] = m[ct] == kNone ? -INFINITY : m[ct] * c;
        join_ml[wave][ct * 16 + col][1] = sum;
      }
#pragma unroll
      for (int k = 0; k < C; ++k) *reinterpret_cast<v4f*>(mine_o + (ct * 16 + col) * kPitch + k * 16 + g * 4) = acc[ct][k];
    }
    __syncthreads();
    const bool done = from == 0 && to == it.units;
    const int valid = rows - it.row0 < ROWS ? rows - it.row0 : ROWS;
    const size_t slot = 2 * (size_t)blockIdx.x + (from == 0 ? 1 : 0);   // the item that the part starts in, the one that it ends in
    for (int at = threadIdx.x; at < valid * (D / 4); at += NW * 64) {
      const int row = at / (D / 4), ch = at % (D / 4) * 4;
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) top = fmaxf(top, join_ml[w][row][0]);
      v4f o = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float mw = join_ml[w][row][0];
        const float f = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - top);
        sum += join_ml[w][row][1] * f;
        o += *reinterpret_cast<const v4f*>(reinterpret_cast<const float*>(smem) + ((size_t)w * ROWS + row) * kPitch + ch) * f;
      }
      if (done) {
        finish_row(p, row_index(p, it.s.first, it.head, it.row0 + row), D, ch, o, top, sum);
      } else {
        *reinterpret_cast<v4f*>(p.part_o + (slot * ROWS + row) * D + ch) = o;
        if (ch == 0) p.part_ml[(slot * ROWS + row) * 2] = top, p.part_ml[(slot * ROWS + row) * 2 + 1] = sum;
      }
    }
    __syncthreads();   // before the next item's loads
    first_item = false;
  }
}

template <int D, int NT, int NW, int NS, typename U = unsigned, typename A>
hipError_t launch_form(A p, bool whole, void* ws, hipStream_t s) {
  constexpr int ROWS = NT * 16;
  const int workgroups = compute_units() * workgroups_per_cu<D, NT, NW, NS>();
  p.whole = whole;
  p.item_units = 0;
  p.min_units_log2 = p.whole ? 0 : log2_of(NW);
  if (!p.whole) place_workspace(p, ROWS, workgroups, ws);
  const dim3 grid((unsigned)workgroups), block(NW * 64);
  if constexpr (sizeof(U) == 4) {
    if (p.c.page_size >= 64) hipLaunchKernelGGL((attn_decode_kernel<D, NT, NW, NS, true, U, A>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((attn_decode_kernel<D, NT, NW, NS, false, U, A>), grid, block, 0, s, p);
  } else {   // (pages of any size by the general form)
    hipLaunchKernelGGL((attn_decode_kernel<D, NT, NW, NS, false, U, A>), grid, block, 0, s, p);
  }
  if (hipError_t e = hipGetLastError(); e != hipSuccess || p.whole) return e;
  return launch_attn_combine(p, ROWS, p.a.cu_q ? (int64_t)p.a.max_q * p.group : p.group, workgroups, s);
}

// Short items stay whole: one launch, no partial results.  Cut in parts they cost a second launch and 128 bytes of partial results for each
// row and 32 channels; whole they keep one workgroup each busy, which matters where there are few of them.  32 query heads on 8 of 128, one
// sequence: single tokens 500 keys 8.5 us whole, 11.1 cut, 1500 keys 13.5 and 11.0; 8 tokens 12.5 and 16.3, 19.0 and 16.1; of 256 channels 500
// keys 13.2 and 12.9.  16 sequences, 8 tokens, 1500 keys: 21.2 and 30.8, of 64 channels 15.8 and 26.9, of 256 44.0 and 40.9; 64 sequences of
// 1500, single tokens: 31.9 and 27.4.  The bound on an item's keys is what the page table or the window can hold.
bool keep_whole(const AttnArgs& p, int row_tiles) {
  const int64_t in_table = (int64_t)p.a.table_pages << p.page_shift, in_window = p.a.window > 0 ? (int64_t)p.a.window + p.a.max_q : in_table;
  const bool many = 2 * (int64_t)p.a.batch * p.c.kv_heads >= compute_units() && (row_tiles > 1 || p.c.head_dim == 64);
  return (in_window < in_table ? in_window : in_table) <= (p.c.head_dim == 256 ? 512 : 1024) * (many ? 2 : 1);
}

// More units than 32 bits hold (a call of seconds): one form for each number of channels, of two row tiles
template <typename A>
bool in_64_bits(const A& p, int row_tiles) { return units_bound(p, row_tiles * 16, 64) >> 32 != 0; }

}  // namespace

template <typename A>
size_t attn_decode_workspace(const A& p, int row_tiles) {
  return keep_whole(p, row_tiles) ? 0 : attn_workspace((in_64_bits(p, row_tiles) ? 2 : row_tiles) * 16, p.c.head_dim, 2 * compute_units());
}

template <typename A>
hipError_t launch_attn_decode(A p, int row_tiles, void* ws, hipStream_t s) {
  const bool whole = keep_whole(p, row_tiles);
  if (in_64_bits(p, row_tiles)) {
    if (p.c.head_dim == 64) return launch_form<64, 2, 4, 4, Units>(p, whole, ws, s);
    if (p.c.head_dim == 128) return launch_form<128, 2, 4, 2, Units>(p, whole, ws, s);
    return launch_form<256, 2, 4, 2, Units>(p, whole, ws, s);
  }
  // (trees: two row tiles come with up to 1024 keys only, where items of 64 and 128 channels stay whole, and four do not come)
  switch (p.c.head_dim * 8 + row_tiles) {
    case 64 * 8 + 1: return whole ? launch_form<64, 1, 8, 4>(p, whole, ws, s) : launch_form<64, 1, 4, 4>(p, whole, ws, s);
    case 64 * 8 + 2:
      if constexpr (!kTree<A>)
        if (!whole) return launch_form<64, 2, 4, 4>(p, whole, ws, s);
      return launch_form<64, 2, 8, 4>(p, whole, ws, s);
    case 128 * 8 + 1: return whole ? launch_form<128, 1, 8, 2>(p, whole, ws, s) : launch_form<128, 1, 4, 2>(p, whole, ws, s);
    case 128 * 8 + 2:
      if constexpr (!kTree<A>)
        if (!whole) return launch_form<128, 2, 4, 2>(p, whole, ws, s);
      return launch_form<128, 2, 8, 2>(p, whole, ws, s);
    case 128 * 8 + 4:
      if constexpr (!kTree<A>) return launch_form<128, 4, 4, 4>(p, whole, ws, s);
      return hipErrorInvalidValue;
    case 256 * 8 + 1: return launch_form<256, 1, 4, 2>(p, whole, ws, s);
    default: return launch_form<256, 2, 4, 2>(p, whole, ws, s);
  }
}

template size_t attn_decode_workspace(const AttnArgs& p, int row_tiles);
template hipError_t launch_attn_decode(AttnArgs p, int row_tiles, void* ws, hipStream_t s);
template size_t attn_decode_workspace(const TreeArgs& p, int row_tiles);
template hipError_t launch_attn_decode(TreeArgs p, int row_tiles, void* ws, hipStream_t s);

// ---- parts of split items, joined -----------------------------------------------------------------------------------------------
namespace {

// blockIdx.x: a boundary between two workgroups of the first launch; the first boundary inside an item joins the item's parts.  A thread
// takes four channels of a row.  GROUPS > 1 (few rows of many parts): the threads of a row are GROUPS groups that take every so many parts and
// meet in LDS; GROUPS = 1 (prompts: many rows of two or three parts): 1024 / D rows at once.
template <int D, int GROUPS>
__global__ __launch_bounds__(256) void attn_combine_kernel(AttnArgs p, int ROWS) {
  constexpr int T = D / 4, R = 256 / T / GROUPS;
  __shared__ v4f sums[GROUPS][T];
  __shared__ float ml[GROUPS][2];
  const int g = blockIdx.x + 1;
  const PartMeta* m = p.meta + g;
  const Units begin = m->begin, end = m->end;
  if (begin >= m->u0 || m[-1].u0 > begin) return;
  const int rows = m->rows, row0 = m->row0, valid = rows - row0 < ROWS ? rows - row0 : ROWS;
  const int group = GROUPS > 1 ? threadIdx.x / T : 0, ch = threadIdx.x % T * 4, most = (int)gridDim.x + 1 - g;   // workgroups from g on
  for (int first = blockIdx.y * R; first < valid; first += gridDim.y * R) {
    const int row = first + (GROUPS > 1 ? 0 : threadIdx.x / T);
    float top = -INFINITY, sum = 0.0f;
    v4f o = {0, 0, 0, 0};
    // part 0: of the workgroup that the item starts in; part i: of workgroup g + i - 1, if that starts inside the item
    if (row < valid) {
#pragma unroll 4
      for (int i = group; i <= most; i += GROUPS) {
        if (i > 0 && m[i - 1].u0 >= end) break;
        const size_t at = (i == 0 ? 2 * (size_t)(g - 1) + 1 : 2 * (size_t)(g + i - 1)) * ROWS + row;
        const float mi = p.part_ml[at * 2], li = p.part_ml[at * 2 + 1];
        const v4f oi = *reinterpret_cast<const v4f*>(p.part_o + at * D + ch);
        const float t = fmaxf(top, mi), f0 = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - t), f1 = mi == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mi - t);
        sum = sum * f0 + li * f1;
        o = o * f0 + oi * f1;
        top = t;
      }
    }
    if constexpr (GROUPS > 1) {
      sums[group][threadIdx.x % T] = o;
      if (ch == 0) ml[group][0] = top, ml[group][1] = sum;
      __syncthreads();
      if (group == 0) {
        top = -INFINITY, sum = 0.0f, o = v4f{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) top = fmaxf(top, ml[k][0]);
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) {
          const float f = ml[k][0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[k][0] - top);
          sum += ml[k][1] * f;
          o += sums[k][threadIdx.x] * f;
        }
        finish_row(p, row_index(p, m->first, m->head, row0 + row), D, ch, o, top, sum);
      }
      __syncthreads();
    } else if (row < valid) {
      finish_row(p, row_index(p, m->first, m->head, row0 + row), D, ch, o, top, sum);
    }
  }
}

template <int D>
void launch_combine_of(const AttnArgs& p, int rows, int64_t expected, int workgroups, hipStream_t s) {
  const unsigned x = (unsigned)workgroups - 1, at_once = 1024 / D, of_block = (unsigned)(expected < rows ? expected : rows);
  // Many threads for a row of many parts (48 query heads on one, 131072 keys, 256 parts of one item: the call takes 61 us so, 132 with a thread
  // for a row's four channels), many rows at once for prompts (600 new tokens of 4 sequences to 16000 keys: 356 us so, 394 with many threads for a
  // row).  Items as far as the host knows; a part is at most one workgroup's.
  const int64_t items = (int64_t)p.a.batch * p.c.kv_heads * ((expected + rows - 1) / rows);
  if (of_block <= 32 || workgroups >= 8 * items)
    hipLaunchKernelGGL((attn_combine_kernel<D, 1024 / D>), dim3(x, of_block < 32 ? of_block : 32), dim3(256), 0, s, p, rows);
  else
    hipLaunchKernelGGL((attn_combine_kernel<D, 1>), dim3(x, (of_block + at_once - 1) / at_once), dim3(256), 0, s, p, rows);
}

}  // namespace

hipError_t launch_attn_combine(const AttnArgs& p, int rows, int64_t rows_expected, int workgroups, hipStream_t s) {
  if (workgroups < 2) return hipSuccess;
  const int64_t expected = rows_expected < 1 ? 1 : rows_expected;
  if (p.c.head_dim == 64) launch_combine_of<64>(p, rows, expected, workgroups, s);
  else if (p.c.head_dim == 128) launch_combine_of<128>(p, rows, expected, workgroups, s);
  else launch_combine_of<256>(p, rows, expected, workgroups, s);
  return hipGetLastError();
}

// ---- the same for trees ---------------------------------------------------------------------------------------------------------------
// Every workgroup finds the split items by itself -- those that begin in front of a boundary between workgroups of the first launch and behind, or at, the
// one before -- and takes so many rows of one after the other.  (With a workgroup for each boundary and block of rows, as above, most end at once, but hold
// their places for the time of a load: 64 nodes on 131072 keys, 16 items in 768 parts, 29.7 us that way, 12.5 this way.)  Bound by the parts' bytes and
// the chain of records, item and parts: 7.5 us where 16 sequences of up to 4096 keys, 16 nodes, 32 heads on 8 of 128 were taken in parts.
namespace {

constexpr int kMostItems = 1024;   // boundaries: workgroups of the first launch

template <int D, int GROUPS>
__global__ __launch_bounds__(256) void attn_join_kernel(TreeArgs p, int ROWS, int workgroups) {
  constexpr int T = D / 4, R = 256 / T / GROUPS;
  __shared__ v4f sums[GROUPS][R][T];
  __shared__ float ml[GROUPS][R][2];
  __shared__ uint16_t items[kMostItems];
  __shared__ uint64_t counts[kMostItems / 64];   // which of 64 workgroups
  __shared__ Units u0[kMostItems];
  const int wave = threadIdx.x / 64, lane = threadIdx.x & 63;
  bool first[kMostItems / 256];
  PartStart start[kMostItems / 256];
#pragma unroll
  for (int k = 0; k < kMostItems / 256; ++k) {
    const int g = k * 256 + threadIdx.x;
    start[k] = p.starts[g < workgroups ? g : workgroups - 1];
  }
#pragma unroll
  for (int k = 0; k < kMostItems / 256; ++k) u0[k * 256 + threadIdx.x] = start[k].u0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kMostItems / 256; ++k) {
    const int g = k * 256 + threadIdx.x;
    first[k] = g > 0 && g < workgroups && start[k].begin < start[k].u0 && u0[g > 0 ? g - 1 : 0] <= start[k].begin;
    const uint64_t here = __ballot(first[k]);
    if (lane == 0) counts[k * 4 + wave] = here;
  }
  __syncthreads();
  int many = 0;
#pragma unroll
  for (int k = 0; k < kMostItems / 64; ++k) {
    const uint64_t here = counts[k];
    if (k % 4 == wave && first[k / 4]) items[many + __popcll(here & ((1ull << lane) - 1))] = (uint16_t)(k * 64 + lane);
    many += __popcll(here);
  }
  __syncthreads();
  const int blocks = (ROWS + R - 1) / R, group = threadIdx.x / T / R, mine = threadIdx.x / T % R, ch = threadIdx.x % T * 4;
  for (int work = blockIdx.x; work < many * blocks; work += gridDim.x) {
    const int g = items[work / blocks];
    const PartMeta* m = p.meta + g;
    const Units end = m->end;
    const int row0 = m->row0, valid = m->rows - row0 < ROWS ? m->rows - row0 : ROWS, row = work % blocks * R + mine, most = workgroups - g;
    // parts: of the workgroup that the item starts in, and of those from g on that start inside the item
    int parts = 1;
    for (int g0 = 0; g0 < most; g0 += 64) {
      const int more = __popcll(__ballot(g0 + lane < most && u0[g0 + lane < most ? g + g0 + lane : g] < end));
      parts += more;
      if (more < 64) break;
    }
    float top = -INFINITY, sum = 0.0f;
    v4f o = {0, 0, 0, 0};
    if (row < valid) {
#pragma unroll 8
      for (int i = group; i < parts; i += GROUPS) {
        const size_t at = (i == 0 ? 2 * (size_t)(g - 1) + 1 : 2 * (size_t)(g + i - 1)) * ROWS + row;
        const float mi = p.part_ml[at * 2], li = p.part_ml[at * 2 + 1];
        const v4f oi = *reinterpret_cast<const v4f*>(p.part_o + at * D + ch);
        const float t = fmaxf(top, mi), f0 = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - t), f1 = mi == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mi - t);
        sum = sum * f0 + li * f1;
        o = o * f0 + oi * f1;
        top = t;
      }
    }
    if constexpr (GROUPS > 1) {
      sums[group][mine][threadIdx.x % T] = o;
      if (ch == 0) ml[group][mine][0] = top, ml[group][mine][1] = sum;
      __syncthreads();
      if (group == 0) {
        top = -INFINITY, sum = 0.0f, o = v4f{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) top = fmaxf(top, ml[k][mine][0]);
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) {
          const float f = ml[k][mine][0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[k][mine][0] - top);
          sum += ml[k][mine][1] * f;
          o += sums[k][mine][threadIdx.x % T] * f;
        }
      }
      __syncthreads();
    }
    if (group == 0 && row < valid) finish_row(p, row_index(p, m->first, m->head, row0 + row), D, ch, o, top, sum);
  }
}

template <int D>
void launch_join_of(const TreeArgs& p, int rows, int64_t expected, int workgroups, hipStream_t s) {
  const int64_t items = (int64_t)p.a.batch * p.c.kv_heads * ((expected + rows - 1) / rows);   // as far as the host knows
  const unsigned grid = 4u * (unsigned)compute_units();
  if (workgroups >= 8 * items) hipLaunchKernelGGL((attn_join_kernel<D, 4>), dim3(grid), dim3(256), 0, s, p, rows, workgroups);
  else hipLaunchKernelGGL((attn_join_kernel<D, 1>), dim3(grid), dim3(256), 0, s, p, rows, workgroups);
}

}  // namespace

hipError_t launch_attn_join(const TreeArgs& p, int rows, int64_t rows_expected, int workgroups, hipStream_t s) {
  if (workgroups < 2) return hipSuccess;
  if (workgroups > kMostItems) return launch_attn_combine(p, rows, rows_expected, workgroups, s);   // (more compute units than this was written for)
  const int64_t expected = rows_expected < 1 ? 1 : rows_expected;
  if (p.c.head_dim == 64) launch_join_of<64>(p, rows, expected, workgroups, s);
  else if (p.c.head_dim == 128) launch_join_of<128>(p, rows, expected, workgroups, s);
  else launch_join_of<256>(p, rows, expected, workgroups, s);
  return hipGetLastError();
}

}  // namespace ave
