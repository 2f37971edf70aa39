// Attention over a paged MXFP4 key/value cache: which kernel takes a call.
#include "attn_common.hpp"

namespace ave {
namespace {

AttnArgs args_of(const ave_fp4_attention& a, const ave_fp4_kv_cache& c) {
  AttnArgs p{};
  p.a = a, p.c = c;
  set_group(p, a.heads / c.kv_heads);
  p.q_aligned = reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && a.q_token_stride % 8 == 0 && a.q_head_stride % 8 == 0;
  p.page_shift = log2_of(c.page_size);
  return p;
}

// Row tiles of 16 of the kernel for few rows; 0: the kernel for prompts.  Up to 32 rows the former is ahead (64 sequences of 4096 keys,
// 8 new tokens, 32 query heads on 8 of 128: 82 us to 122), from 33 the latter (64 query heads: 265 to 147), but for single tokens on
// one key head of 128 channels (48 query heads, 16 sequences of 16384 keys: 45 to 46 us, one of 131072: 61 to 101).
// Between 17 and 127 rows neither is near its floor: reads and products of these four take 46, 57, 6 and 3 us.  Four row tiles leave one wave a
// SIMD and many parts of one item to join; a block of 128 rows with 64 in it leaves two of four waves without work.
int decode_row_tiles(const AttnArgs& p) {
  const int new_tokens = p.a.cu_q ? p.a.max_q : 1;
  const int64_t rows = (int64_t)new_tokens * p.group;
  const int most = p.c.head_dim == 128 && new_tokens == 1 ? 64 : 32;
  return rows > most ? 0 : rows > 32 ? 4 : rows > 16 ? 2 : 1;
}

}  // namespace

size_t attention_workspace_bytes(const ave_fp4_attention& a, const ave_fp4_kv_cache& c) {
  const AttnArgs p = args_of(a, c);
  if (const int tiles = decode_row_tiles(p)) return attn_decode_workspace(p, tiles);
  return attn_prompt_workspace(p);
}

hipError_t launch_attention(const ave_fp4_attention& a, const ave_fp4_kv_cache& c, void* workspace, hipStream_t s) {
  const AttnArgs args = args_of(a, c);
  if (const int tiles = decode_row_tiles(args)) return launch_attn_decode(args, tiles, workspace, s);
  return launch_attn_prompt(args, workspace, s);
}

}  // namespace ave
