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

// Row tiles of 16 of the kernel for few rows; 0: the kernel for prompts
int decode_row_tiles(const AttnArgs& p) {
  const int64_t rows = (int64_t)(p.a.cu_q ? p.a.max_q : 1) * p.group;
  const int most = p.c.head_dim == 256 ? 32 : 64;
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
