// Around a tree of drafted tokens: what its nodes see of each other, and the kept ones moved together in the caches of all layers.
#include <algorithm>

#include "fp4_common.hpp"
#include "kv_cache.hpp"

namespace ave {
namespace {

// ---- ancestors and positions ------------------------------------------------------------------------------------------------------
// A workgroup a sequence, a thread a node, which goes up from parent to parent: their indices fall, so that the bits come word by word, the
// last first.  Bound by latency: the parents lie in LDS, where a step takes about 100 cycles.
constexpr int kTreeThreads = 256, kTreeNodes = 8192;   // nodes whose parents LDS holds; the rest are looked up in memory

__global__ __launch_bounds__(kTreeThreads) void draft_tree_kernel(const int32_t* parents, const int32_t* cu_q, const int32_t* seq_lens, int tokens,
                                                                  uint64_t* seen, int words, int32_t* positions) {
  __shared__ int32_t up[kTreeNodes];
  const int b = blockIdx.x;
  int first = cu_q[b], end = cu_q[b + 1];
  first = first < 0 ? 0 : first > tokens ? tokens : first;
  end = end < first ? first : end > tokens ? tokens : end;
  const int n = end - first, base = positions ? seq_lens[b] - n : 0;
  for (int i = threadIdx.x; i < n && i < kTreeNodes; i += kTreeThreads) up[i] = parents[first + i];
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kTreeThreads) {
    int at = i, above = -1;
    uint64_t* row = seen + (int64_t)(first + i) * words;
    const auto next = [&] {
      const int p = at < kTreeNodes ? up[at] : parents[first + at];
      at = p >= 0 && p < at ? p : -1;
      ++above;
    };
    for (int w = words - 1; w >= 0; --w) {
      uint64_t bits = 0;
      while (at >= 0 && at >> 6 >= w) {
        if (at >> 6 == w) bits |= 1ull << (at & 63);
        next();
      }
      row[w] = bits;
    }
    while (at >= 0) next();   // (without bits)
    if (positions) positions[first + i] = base + above;
  }
}

// ---- kept tokens moved together -----------------------------------------------------------------------------------------------------
// A sequence's tokens of one head, keys or values, of one layer: 16 bytes of codes and a byte of scale a thread.  A token comes from no place below its own, so
// in rising order none is overwritten before it is read, if those of one step are all read before any is written: a step is a wave's (few tokens) or a
// workgroup's.
constexpr int kLayers = 48;   // of a launch: what its arguments hold
struct KeepArgs {
  ave_fp4_keep k;
  int pages, kv_heads, page_size, page_shift;
  struct {
    uint8_t* data[4];   // codes and scales of keys, of values
    int64_t stride[4];
  } layer[kLayers];
};

// PARTS: of D / 32 pieces a token; THREADS that share a step; EACH tokens a thread at once
template <int PIECES, int THREADS, int EACH>
__global__ __launch_bounds__(256) void keep_kv_kernel(KeepArgs p) {
  constexpr int kAtOnce = THREADS / PIECES;   // tokens
  const int unit = blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS, b = blockIdx.y, me = threadIdx.x % THREADS, piece = me % PIECES;
  const auto& layer = p.layer[blockIdx.z];
  const int values = unit & 1, head = unit >> 1;
  int first = p.k.cu_q[b], end = p.k.cu_q[b + 1], many = p.k.accepted[b];
  first = first < 0 ? 0 : first > p.k.tokens ? p.k.tokens : first;
  end = end < first ? first : end > p.k.tokens ? p.k.tokens : end;
  const int n = end - first, base = p.k.seq_lens[b] - n;
  many = many < 0 ? 0 : many > n ? n : many;
  if (unit == 0 && me == 0 && blockIdx.z == 0 && p.k.kept_lens) p.k.kept_lens[b] = base + many;
  const bool mine = head < p.kv_heads;
  if (THREADS < 256 && !mine) return;   // (a whole wave)
  const int32_t* table = p.k.page_table + (int64_t)b * p.k.page_table_stride;
  uint8_t* const codes = layer.data[2 * values];
  uint8_t* const scales = layer.data[2 * values + 1];
  const int64_t code_stride = layer.stride[2 * values], scale_stride = layer.stride[2 * values + 1];
  const int in_table = p.k.table_pages << p.page_shift;
  const auto place = [&](int position, int64_t& code, int64_t& scale) {   // byte offsets; false: no such place
    if (position < 0 || position >= in_table) return false;
    const int page = table[position >> p.page_shift];
    if (page < 0 || page >= p.pages) return false;
    const unsigned row = (unsigned)(head * p.page_size + (position & (p.page_size - 1))) * PIECES + piece;
    code = page * code_stride + (int64_t)row * 16;
    scale = page * scale_stride + row;
    return true;
  };
  for (int i0 = 0; i0 < many; i0 += kAtOnce * EACH) {
    v4i code[EACH];
    uint8_t scale[EACH];
    bool move[EACH];
    int64_t to_code[EACH], to_scale[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int i = i0 + e * kAtOnce + me / PIECES;
      move[e] = false;
      if (mine && i < many) {
        const int from = p.k.path[first + i];
        int64_t from_code, from_scale;
        if (from >= 0 && from < n && from != i && place(base + from, from_code, from_scale) && place(base + i, to_code[e], to_scale[e])) {
          move[e] = true;
          code[e] = *reinterpret_cast<const v4i*>(codes + from_code);
          scale[e] = scales[from_scale];
        }
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // read, before anybody writes (the barrier by itself waits for no load)
    if constexpr (THREADS > 64) __syncthreads();
#pragma unroll
    for (int e = 0; e < EACH; ++e)
      if (move[e]) {
        *reinterpret_cast<v4i*>(codes + to_code[e]) = code[e];
        scales[to_scale[e]] = scale[e];
      }
  }
}

template <int PIECES>
void launch_keep(const KeepArgs& p, int layers, hipStream_t s) {
  const int units = 2 * p.kv_heads;
  const bool few = p.k.max_q <= 4 * 64 / PIECES;
  for (int b = 0; b < p.k.batch; b += 65535) {
    KeepArgs part = p;
    part.k.page_table = p.k.page_table + (int64_t)b * p.k.page_table_stride;
    part.k.seq_lens += b, part.k.cu_q += b, part.k.accepted += b;
    if (part.k.kept_lens) part.k.kept_lens += b;
    const unsigned y = (unsigned)std::min(p.k.batch - b, 65535);
    if (few) hipLaunchKernelGGL((keep_kv_kernel<PIECES, 64, 2>), dim3((units + 3) / 4, y, layers), dim3(256), 0, s, part);
    else hipLaunchKernelGGL((keep_kv_kernel<PIECES, 256, 4>), dim3(units, y, layers), dim3(256), 0, s, part);
  }
}

}  // namespace

hipError_t launch_draft_tree(const int32_t* parents, const int32_t* cu_q, const int32_t* seq_lens, int tokens, int batch, uint64_t* seen, int words,
                             int32_t* positions, hipStream_t s) {
  hipLaunchKernelGGL(draft_tree_kernel, dim3((unsigned)batch), dim3(kTreeThreads), 0, s, parents, cu_q, seq_lens, tokens, seen, words, positions);
  return hipGetLastError();
}

hipError_t launch_keep_kv(const ave_fp4_kv_cache* caches, int layers, const ave_fp4_keep& k, hipStream_t s) {
  const ave_fp4_kv_cache& c0 = caches[0];
  for (int from = 0; from < layers; from += kLayers) {
    const int now = std::min(layers - from, kLayers);
    KeepArgs p{};
    p.k = k, p.pages = c0.pages, p.kv_heads = c0.kv_heads, p.page_size = c0.page_size, p.page_shift = log2_of(c0.page_size);
    if (from > 0) p.k.kept_lens = nullptr;
    for (int i = 0; i < now; ++i) {
      const ave_fp4_kv_cache& c = caches[from + i];
      p.layer[i] = {{c.k, c.k_scale, c.v, c.v_scale}, {c.k_page_stride, c.k_scale_page_stride, c.v_page_stride, c.v_scale_page_stride}};
    }
    if (c0.head_dim == 64) launch_keep<2>(p, now, s);
    else if (c0.head_dim == 128) launch_keep<4>(p, now, s);
    else launch_keep<8>(p, now, s);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace ave
