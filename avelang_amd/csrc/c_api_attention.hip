// C ABI of the operators around the MXFP4 key/value cache: argument checks and launches.
#include <hip/hip_runtime.h>

#include "../../include/ave_fp4.h"
#include "c_api_common.hpp"
#include "kv_cache.hpp"

using ave::aligned;
using ave::fail_inval;
using ave::finish;

namespace {

int check_head_dim(int d) {
  return d == 64 || d == 128 || d == 256 ? 0 : fail_inval("head_dim must be 64, 128 or 256, got %d.", d);
}

int check_cache(const ave_fp4_kv_cache* c) {
  if (!c) return fail_inval("null cache.");
  if (int rc = check_head_dim(c->head_dim)) return rc;
  if (c->kv_heads <= 0) return fail_inval("kv_heads must be positive, got %d.", c->kv_heads);
  if (c->page_size < 16 || c->page_size > 4096 || (c->page_size & (c->page_size - 1)) != 0)
    return fail_inval("page_size must be a power of two from 16 to 4096, got %d.", c->page_size);
  if (c->pages <= 0 || (int64_t)c->pages * c->page_size > INT32_MAX)
    return fail_inval("the cache must have between 1 and 2^31 - 1 slots, got %d pages of %d.", c->pages, c->page_size);
  if ((int64_t)c->kv_heads * c->page_size * (c->head_dim / 2) > (1 << 30))
    return fail_inval("a page must not exceed 2^30 bytes, got %d heads of %d tokens.", c->kv_heads, c->page_size);
  if (!c->k || !c->k_scale || !c->v || !c->v_scale) return fail_inval("null device pointer.");
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || c->k_page_stride % 16 || c->v_page_stride % 16)
    return fail_inval("the cache's codes must be 16-byte aligned, pages included.");
  if (!aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) || c->k_scale_page_stride % 4 || c->v_scale_page_stride % 4)
    return fail_inval("the cache's scales must be 4-byte aligned, pages included.");
  const int64_t codes = (int64_t)c->kv_heads * c->page_size * (c->head_dim / 2), scales = codes / 16;
  if (c->pages > 1 && (c->k_page_stride < codes || c->v_page_stride < codes || c->k_scale_page_stride < scales || c->v_scale_page_stride < scales))
    return fail_inval("the cache's pages overlap.");
  return 0;
}

int check_heads(const ave_fp4_heads* h, const char* name, bool output) {
  if (h->heads <= 0) return fail_inval("%s must have heads, got %d.", name, h->heads);
  if (!h->data) return fail_inval("null device pointer (%s).", name);
  if (output && h->is_f32) return fail_inval("%s must be bf16.", name);
  if (!aligned(h->data, h->is_f32 ? 4 : 2)) return fail_inval("%s must be aligned to its elements.", name);
  return 0;
}

int check_how(const ave_fp4_norm_rope* how, int head_dim) {
  if (!how) return 0;
  if (!how->cos != !how->sin) return fail_inval("cos and sin come together.");
  if (how->cos) {
    if (how->rotary_dim <= 0 || how->rotary_dim > head_dim || how->rotary_dim % 16 != 0)
      return fail_inval("rotary_dim must be a multiple of 16 up to head_dim = %d, got %d.", head_dim, how->rotary_dim);
    if (how->table_rows <= 0) return fail_inval("cos and sin must have rows.");
    if (!how->positions) return fail_inval("rotation needs positions.");
    if (!aligned(how->cos, 4) || !aligned(how->sin, 4)) return fail_inval("cos and sin must be 4-byte aligned.");
  }
  const size_t a = how->weight_is_f32 ? 4 : 2;
  if (!aligned(how->q_weight, a) || !aligned(how->k_weight, a)) return fail_inval("norm weights must be aligned to their elements.");
  return 0;
}

}  // namespace

extern "C" {

int ave_fp4_qk_norm_rope(const ave_fp4_heads* q, const ave_fp4_heads* k, int tokens, int head_dim, const ave_fp4_norm_rope* how,
                         const ave_fp4_heads* q_out, const ave_fp4_heads* k_out, void* hip_stream) {
  ave::clear_error();
  if (tokens < 0) return fail_inval("tokens must be non-negative, got %d.", tokens);
  if (int rc = check_head_dim(head_dim)) return rc;
  if (int rc = check_how(how, head_dim)) return rc;
  if (!q != !q_out || !k != !k_out || (!q && !k)) return fail_inval("queries, keys or both, each with its output.");
  if (tokens == 0) return 0;
  ave::HeadArgs p;
  if (q) {
    if (int rc = check_heads(q, "q", false)) return rc;
    if (int rc = check_heads(q_out, "q_out", true)) return rc;
    if (q->heads != q_out->heads) return fail_inval("q has %d heads and q_out %d.", q->heads, q_out->heads);
    p.q = *q, p.q_out = *q_out;
  }
  if (k) {
    if (int rc = check_heads(k, "k", false)) return rc;
    if (int rc = check_heads(k_out, "k_out", true)) return rc;
    if (k->heads != k_out->heads) return fail_inval("k has %d heads and k_out %d.", k->heads, k_out->heads);
    p.k = *k, p.k_out = *k_out;
  }
  if (q && k && q->is_f32 != k->is_f32) return fail_inval("q and k must have one type.");
  if (how) p.how = *how;
  p.tokens = tokens, p.head_dim = head_dim;
  return finish(ave::launch_heads(p, static_cast<hipStream_t>(hip_stream)), "norm and rotation kernel");
}

int ave_fp4_append_kv_mxfp4(const ave_fp4_heads* k, const ave_fp4_heads* v, int tokens, const int32_t* slots, const ave_fp4_norm_rope* how,
                            const ave_fp4_kv_cache* cache, const ave_fp4_heads* q, const ave_fp4_heads* q_out, void* hip_stream) {
  ave::clear_error();
  if (tokens < 0) return fail_inval("tokens must be non-negative, got %d.", tokens);
  if (int rc = check_cache(cache)) return rc;
  if (int rc = check_how(how, cache->head_dim)) return rc;
  if (!k || !v) return fail_inval("keys and values are required.");
  if (!q != !q_out) return fail_inval("queries come with their output.");
  if (tokens == 0) return 0;
  ave::HeadArgs p;
  if (int rc = check_heads(k, "k", false)) return rc;
  if (int rc = check_heads(v, "v", false)) return rc;
  if (k->heads != cache->kv_heads || v->heads != cache->kv_heads)
    return fail_inval("the cache has %d heads, k %d and v %d.", cache->kv_heads, k->heads, v->heads);
  if (k->is_f32 != v->is_f32 || (q && q->is_f32 != k->is_f32)) return fail_inval("q, k and v must have one type.");
  if (q) {
    if (int rc = check_heads(q, "q", false)) return rc;
    if (int rc = check_heads(q_out, "q_out", true)) return rc;
    if (q->heads != q_out->heads) return fail_inval("q has %d heads and q_out %d.", q->heads, q_out->heads);
    p.q = *q, p.q_out = *q_out;
  }
  if (!slots) return fail_inval("null device pointer (slots).");
  p.k = *k, p.v = *v, p.cache = *cache, p.slots = slots;
  if (how) p.how = *how;
  p.tokens = tokens, p.head_dim = cache->head_dim;
  return finish(ave::launch_heads(p, static_cast<hipStream_t>(hip_stream)), "key/value append kernel");
}

int ave_fp4_gather_kv_mxfp4(const ave_fp4_kv_cache* cache, const int32_t* slots, int tokens, uint16_t* k, uint16_t* v, void* hip_stream) {
  ave::clear_error();
  if (tokens < 0) return fail_inval("tokens must be non-negative, got %d.", tokens);
  if (int rc = check_cache(cache)) return rc;
  if (tokens == 0) return 0;
  if (!slots || !k || !v) return fail_inval("null device pointer.");
  if (!aligned(k, 16) || !aligned(v, 16)) return fail_inval("k and v must be 16-byte aligned.");
  return finish(ave::launch_gather_kv(*cache, slots, tokens, k, v, static_cast<hipStream_t>(hip_stream)), "key/value gather kernel");
}

static int check_attention(const ave_fp4_attention* a, const ave_fp4_kv_cache* cache) {
  if (!a) return fail_inval("null arguments.");
  if (int rc = check_cache(cache)) return rc;
  if (a->tokens < 0 || a->batch < 0) return fail_inval("tokens and batch must be non-negative, got %d and %d.", a->tokens, a->batch);
  if (a->heads <= 0 || a->heads % cache->kv_heads != 0)
    return fail_inval("query heads must be a multiple of the cache's %d, got %d.", cache->kv_heads, a->heads);
  if (a->heads / cache->kv_heads > 1024) return fail_inval("at most 1024 query heads share a key head, got %d.", a->heads / cache->kv_heads);
  // the kernels' ints also count what lies behind the last row (the blocks of 64 lanes) and the last key (two tiles that are looked for ahead)
  if ((int64_t)a->tokens * a->heads > INT32_MAX - (1 << 14))
    return fail_inval("tokens times heads must fit 31 bits with 2^14 to spare, got %d x %d.", a->tokens, a->heads);
  if (a->table_pages < 0 || (int64_t)a->table_pages * cache->page_size > INT32_MAX - 255)
    return fail_inval("the page table must cover at most 2^31 - 256 tokens, got %d pages of %d.", a->table_pages, cache->page_size);
  if (a->max_q < 0) return fail_inval("max_q must be non-negative, got %d.", a->max_q);
  if (a->window < 0) return fail_inval("window must be non-negative, got %d.", a->window);
  if (a->window > 0 && !a->causal) return fail_inval("a window needs causal attention.");
  if (!a->cu_q && a->tokens != a->batch) return fail_inval("without cu_q every sequence has one token: %d tokens, %d sequences.", a->tokens, a->batch);
  return 0;
}

size_t ave_fp4_attention_mxfp4_workspace_bytes(const ave_fp4_attention* a, const ave_fp4_kv_cache* cache) {
  ave::clear_error();
  if (check_attention(a, cache) != 0 || a->tokens == 0 || a->batch == 0) return 0;
  return ave::attention_workspace_bytes(*a, *cache);
}

int ave_fp4_attention_mxfp4(const ave_fp4_attention* a, const ave_fp4_kv_cache* cache, void* workspace, size_t workspace_bytes,
                            void* hip_stream) {
  ave::clear_error();
  if (int rc = check_attention(a, cache)) return rc;
  if (a->tokens == 0 || a->batch == 0) return 0;
  if (!a->q || !a->out || !a->seq_lens || (!a->page_table && a->table_pages > 0)) return fail_inval("null device pointer.");
  if (!aligned(a->q, 2) || !aligned(a->out, 4)) return fail_inval("q must be 2-byte and out 4-byte aligned.");
  const size_t need = ave::attention_workspace_bytes(*a, *cache);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail_inval("the workspace must have %zu bytes, got %zu.", need, workspace ? workspace_bytes : (size_t)0);
  if (need > 0 && !aligned(workspace, 16)) return fail_inval("the workspace must be 16-byte aligned.");
  return finish(ave::launch_attention(*a, *cache, workspace, static_cast<hipStream_t>(hip_stream)), "attention kernel");
}

}  // extern "C"
