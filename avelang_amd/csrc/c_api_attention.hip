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

namespace {
struct Range {
  uintptr_t from, to;
};
template <typename T>
Range range(const T* p, int64_t n) {
  const uintptr_t from = reinterpret_cast<uintptr_t>(p);
  return {from, p ? from + (uintptr_t)n * sizeof(T) : from};
}
bool overlap(const Range& a, const Range& b) { return a.from < b.to && b.from < a.to; }
// Rows of so many bytes, so many bytes apart: what is between them is nobody's
struct Rows {
  uintptr_t from;
  int64_t rows, stride, bytes;
};
bool overlap(const Rows& r, const Range& o) {
  if (!r.from || r.rows <= 0 || r.bytes <= 0 || o.from >= o.to) return false;
  const __int128 stride = r.stride < 0 ? -(__int128)r.stride : r.stride, from = r.from + (r.stride < 0 ? (r.rows - 1) * (__int128)r.stride : 0);
  // the first row that ends behind the range's start
  const __int128 ahead = (__int128)o.from - from - r.bytes, row = ahead < 0 || stride == 0 ? 0 : ahead / stride + 1;
  return row < r.rows && from + row * stride < (__int128)o.to && (__int128)o.from < from + row * stride + r.bytes;
}
template <size_t I, size_t O>
bool overlap(const Rows (&in)[I], const Range (&out)[O]) {
  for (const Rows& r : in)
    for (const Range& o : out)
      if (overlap(r, o)) return true;
  return false;
}
// Does an output overlap an input or another output?
template <size_t I, size_t O>
bool overlap(const Range (&in)[I], const Range (&out)[O]) {
  for (size_t o = 0; o < O; ++o) {
    for (size_t i = 0; i < I; ++i)
      if (overlap(in[i], out[o])) return true;
    for (size_t other = 0; other < o; ++other)
      if (overlap(out[other], out[o])) return true;
  }
  return false;
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

static int check_tree(const ave_fp4_attention* a, const ave_fp4_tree* t, const ave_fp4_kv_cache* cache, ave_fp4_attention* with_causal) {
  if (!a || !t) return fail_inval("null arguments.");
  *with_causal = *a;
  with_causal->causal = 1;
  if (int rc = check_attention(with_causal, cache)) return rc;
  if (t->words <= 0 || t->words > 1 << 25) return fail_inval("seen must have between 1 and 2^25 words a row, got %d.", t->words);
  if (t->stride < 0 || (t->stride > 0 && t->stride < t->words)) return fail_inval("rows of seen overlap: %d words, %lld apart.", t->words, (long long)t->stride);
  return 0;
}

size_t ave_fp4_tree_attention_mxfp4_workspace_bytes(const ave_fp4_attention* a, const ave_fp4_tree* tree, const ave_fp4_kv_cache* cache) {
  ave::clear_error();
  ave_fp4_attention args;
  if (check_tree(a, tree, cache, &args) != 0 || args.tokens == 0 || args.batch == 0) return 0;
  return ave::tree_attention_workspace_bytes(args, *tree, *cache);
}

int ave_fp4_tree_attention_mxfp4(const ave_fp4_attention* a, const ave_fp4_tree* tree, const ave_fp4_kv_cache* cache, void* workspace,
                                 size_t workspace_bytes, void* hip_stream) {
  ave::clear_error();
  ave_fp4_attention args;
  if (int rc = check_tree(a, tree, cache, &args)) return rc;
  if (args.tokens == 0 || args.batch == 0) return 0;
  if (!args.q || !args.out || !args.seq_lens || !tree->seen || (!args.page_table && args.table_pages > 0)) return fail_inval("null device pointer.");
  if (!aligned(args.q, 2) || !aligned(args.out, 4) || !aligned(tree->seen, 8)) return fail_inval("q must be 2-byte, out 4-byte and seen 8-byte aligned.");
  const size_t need = ave::tree_attention_workspace_bytes(args, *tree, *cache);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail_inval("the workspace must have %zu bytes, got %zu.", need, workspace ? workspace_bytes : (size_t)0);
  if (need > 0 && !aligned(workspace, 16)) return fail_inval("the workspace must be 16-byte aligned.");
  return finish(ave::launch_tree_attention(args, *tree, *cache, workspace, static_cast<hipStream_t>(hip_stream)), "tree attention kernel");
}

int ave_fp4_draft_tree(const int32_t* parents, const int32_t* cu_q, const int32_t* seq_lens, int tokens, int batch, uint64_t* seen, int words,
                       int32_t* positions, void* hip_stream) {
  ave::clear_error();
  if (tokens < 0 || batch < 0) return fail_inval("tokens and batch must be non-negative, got %d and %d.", tokens, batch);
  if (seen && (words <= 0 || words > 1 << 25)) return fail_inval("seen must have between 1 and 2^25 words a row, got %d.", words);
  if (tokens == 0 || batch == 0 || (!seen && !positions)) return 0;
  if (!parents || !cu_q || (positions && !seq_lens)) return fail_inval("null device pointer.");
  if (!aligned(seen, 8)) return fail_inval("seen must be 8-byte aligned.");
  const Range in[] = {range(parents, tokens), range(cu_q, (int64_t)batch + 1), range(seq_lens, batch)};
  const Range out[] = {range(seen, (int64_t)tokens * words), range(positions, tokens)};
  if (overlap(in, out)) return fail_inval("seen and positions must not overlap the inputs, nor each other.");
  return finish(ave::launch_draft_tree(parents, cu_q, seq_lens, tokens, batch, seen, seen ? words : 0, positions, static_cast<hipStream_t>(hip_stream)),
                "draft tree kernel");
}

static int check_draft(const ave_fp4_draft* d) {
  if (!d) return fail_inval("null arguments.");
  if (d->rows < 0 || d->batch < 0) return fail_inval("rows and batch must be non-negative, got %d and %d.", d->rows, d->batch);
  if (d->vocab <= 0 || d->vocab > 1 << 30) return fail_inval("vocab must be from 1 to 2^30, got %d.", d->vocab);
  const int64_t pieces = (d->vocab + ave::kVocabPiece - 1) / ave::kVocabPiece;
  if (d->rows * pieces >= 1 << 22 || d->batch * pieces >= 1 << 22)   // workgroups of a launch, of up to 1024 threads
    return fail_inval("rows and batch times vocab / %d must be below 2^22, got %d, %d and %d.", ave::kVocabPiece, d->rows, d->batch, d->vocab);
  return 0;
}

size_t ave_fp4_verify_draft_workspace_bytes(const ave_fp4_draft* draft) {
  ave::clear_error();
  if (check_draft(draft) != 0 || draft->batch == 0) return 0;
  return ave::verify_draft_workspace_bytes(*draft);
}

int ave_fp4_verify_draft(const ave_fp4_draft* draft, void* workspace, size_t workspace_bytes, void* hip_stream) {
  ave::clear_error();
  if (int rc = check_draft(draft)) return rc;
  const ave_fp4_draft& d = *draft;
  if (d.batch == 0) return 0;
  if (!d.cu_q || !d.accepted || (d.rows > 0 && (!d.logits || !d.tokens || !d.parents || !d.uniform || !d.path || !d.emitted)))
    return fail_inval("null device pointer.");
  if (!aligned(d.logits, d.logits_f32 ? 4 : 2) || !aligned(d.draft_probs, 4)) return fail_inval("logits and draft_probs must be aligned to their elements.");
  const Range in[] = {range(d.tokens, d.rows), range(d.parents, d.rows), range(d.cu_q, (int64_t)d.batch + 1), range(d.uniform, d.rows), range(d.temperature, d.batch)};
  const Range out[] = {range(d.accepted, d.batch), range(d.path, d.rows), range(d.emitted, d.rows)};
  const int64_t size = d.logits_f32 ? 4 : 2;
  const Rows read[] = {{reinterpret_cast<uintptr_t>(d.logits), d.rows, d.logits_stride * size, d.vocab * size},
                       {reinterpret_cast<uintptr_t>(d.draft_probs), d.rows, d.draft_probs_stride * 4, d.vocab * (int64_t)4}};
  if (overlap(in, out) || overlap(read, out)) return fail_inval("accepted, path and emitted must not overlap the inputs, nor each other.");
  const size_t need = ave::verify_draft_workspace_bytes(d);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail_inval("the workspace must have %zu bytes, got %zu.", need, workspace ? workspace_bytes : (size_t)0);
  if (need > 0 && !aligned(workspace, 16)) return fail_inval("the workspace must be 16-byte aligned.");
  return finish(ave::launch_verify_draft(d, workspace, static_cast<hipStream_t>(hip_stream)), "draft verification kernel");
}

int ave_fp4_keep_kv_mxfp4(const ave_fp4_kv_cache* caches, int layers, const ave_fp4_keep* keep, void* hip_stream) {
  ave::clear_error();
  if (layers <= 0) return fail_inval("there must be layers, got %d.", layers);
  if (!caches || !keep) return fail_inval("null arguments.");
  for (int i = 0; i < layers; ++i) {
    const ave_fp4_kv_cache &c = caches[i], &c0 = caches[0];
    if (int rc = check_cache(&c)) return rc;
    if (c.pages != c0.pages || c.kv_heads != c0.kv_heads || c.page_size != c0.page_size || c.head_dim != c0.head_dim)
      return fail_inval("all caches must have one shape: layer %d differs from layer 0.", i);
    for (int j = 0; j < i; ++j)
      if (caches[j].k == c.k || caches[j].v == c.v) return fail_inval("layers %d and %d have the same cache.", j, i);
  }
  const ave_fp4_keep& k = *keep;
  if (k.tokens < 0 || k.batch < 0 || k.table_pages < 0 || k.max_q < 0)
    return fail_inval("tokens, batch, table_pages and max_q must be non-negative, got %d, %d, %d and %d.", k.tokens, k.batch, k.table_pages, k.max_q);
  if ((int64_t)k.table_pages * caches->page_size > INT32_MAX)
    return fail_inval("the page table must cover at most 2^31 - 1 tokens, got %d pages of %d.", k.table_pages, caches->page_size);
  if (k.batch == 0) return 0;
  if (!k.seq_lens || !k.cu_q || !k.accepted || (k.tokens > 0 && !k.path) || (k.table_pages > 0 && !k.page_table)) return fail_inval("null device pointer.");
  const Range in[] = {range(k.seq_lens, k.batch), range(k.cu_q, (int64_t)k.batch + 1), range(k.path, k.tokens), range(k.accepted, k.batch)};
  const Range out[] = {range(k.kept_lens, k.batch)};
  const Rows table[] = {{reinterpret_cast<uintptr_t>(k.page_table), k.batch, k.page_table_stride * 4, k.table_pages * (int64_t)4}};
  bool overlaps = overlap(in, out) || overlap(table, out);
  for (int i = 0; i < layers && !overlaps; ++i) {
    const ave_fp4_kv_cache& c = caches[i];
    const int64_t codes = (int64_t)c.kv_heads * c.page_size * (c.head_dim / 2);
    const Rows pages[] = {{reinterpret_cast<uintptr_t>(c.k), c.pages, c.k_page_stride, codes}, {reinterpret_cast<uintptr_t>(c.v), c.pages, c.v_page_stride, codes},
                          {reinterpret_cast<uintptr_t>(c.k_scale), c.pages, c.k_scale_page_stride, codes / 16},
                          {reinterpret_cast<uintptr_t>(c.v_scale), c.pages, c.v_scale_page_stride, codes / 16}};
    overlaps = overlap(pages, out);
  }
  if (overlaps) return fail_inval("kept_lens must not overlap an input, nor a cache.");
  return finish(ave::launch_keep_kv(caches, layers, k, static_cast<hipStream_t>(hip_stream)), "key/value keep kernel");
}

}  // extern "C"
