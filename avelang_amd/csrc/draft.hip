// Around a tree of drafted tokens: what its nodes see of each other, and the kept ones moved together in the caches of all layers.
#include <algorithm>

#include "fp4_common.hpp"
#include "kernels.hpp"
#include "kv_cache.hpp"

namespace ave {
namespace {

// ---- ancestors and positions ------------------------------------------------------------------------------------------------------
// A workgroup a sequence, a thread a node, which goes up from parent to parent: their indices fall, so that the bits come word by word, the
// last first.  Bound by latency: the parents lie in LDS, where a step takes about 100 cycles (8 nodes 2.1 us, 256 trees of 64 4.1).
constexpr int kTreeThreads = 256, kTreeNodes = 8192;   // nodes whose parents LDS holds; the rest are looked up in memory

__device__ inline void tree_of(const int32_t* parents, const int32_t* cu_q, const int32_t* seq_lens, int tokens, uint64_t* seen, int words,
                               int32_t* positions, int b) {
  __shared__ int32_t up[kTreeNodes];
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
__global__ __launch_bounds__(kTreeThreads) void draft_tree_kernel(const int32_t* parents, const int32_t* cu_q, const int32_t* seq_lens, int tokens, int batch,
                                                                  uint64_t* seen, int words, int32_t* positions) {
  for (int64_t b = blockIdx.x; b < batch; b += gridDim.x) {
    if (b >= gridDim.x) __syncthreads();   // the parents of the one before have been read
    tree_of(parents, cu_q, seq_lens, tokens, seen, words, positions, (int)b);
  }
}

// ---- kept tokens moved together -----------------------------------------------------------------------------------------------------
// A sequence's tokens of one head, keys or values, of one layer are a list; 16 bytes of codes and a byte of scale a thread.  A token comes from no place
// below its own, so in rising order none is overwritten before it is read, if those of one step are all read before any is written: a step is a wave's (few
// tokens) or a workgroup's.  Bound by latency where nodes of a draft move (64 sequences of up to 16 nodes, 32 layers, 8 heads of 128: 9.6 us, 9 MB), by HBM where a cache is
// thinned out (half of 16 x 4099 tokens: 17.2 us, 71 MB read and written at 4.1 TB/s, launch included).
constexpr int kLayers = 48;   // of a launch: what its arguments hold
struct KeepArgs {
  ave_fp4_keep k;
  int pages, kv_heads, page_size, page_shift;
  struct {
    uint8_t* data[4];   // codes and scales of keys, of values
    int64_t stride[4];
  } layer[kLayers];
};
struct KeepSpan {
  int first, n, many;   // first entry of `path`, nodes, kept ones
  int64_t base;         // place of the first node
};
__device__ inline KeepSpan keep_span(const KeepArgs& p, int b) {
  KeepSpan s;
  int end = p.k.cu_q[b + 1];
  s.first = p.k.cu_q[b], s.many = p.k.accepted[b], s.base = p.k.seq_lens[b];
  s.first = s.first < 0 ? 0 : s.first > p.k.tokens ? p.k.tokens : s.first;
  end = end < s.first ? s.first : end > p.k.tokens ? p.k.tokens : end;
  s.n = end - s.first;
  s.base -= s.n;
  s.many = s.many < 0 ? 0 : s.many > s.n ? s.n : s.many;
  return s;
}
// Where entry i goes and comes from: page and row of a head (token within the page); from.page < 0: nothing moves
struct Place {
  int page, row;
};
__device__ inline Place keep_place(const KeepArgs& p, int b, int64_t at) {
  if (at < 0 || at >= p.k.table_pages << p.page_shift) return {-1, 0};
  const int position = (int)at;
  const int page = p.k.page_table[(int64_t)b * p.k.page_table_stride + (position >> p.page_shift)];
  return {page < p.pages ? page : -1, position & (p.page_size - 1)};
}
__device__ inline void keep_places(const KeepArgs& p, int b, const KeepSpan& s, int i, Place& from, Place& to) {
  from = {-1, 0}, to = from;
  if (i >= s.many) return;
  const int at = p.k.path[s.first + i];
  if (at < 0 || at >= s.n || at == i) return;
  from = keep_place(p, b, s.base + at), to = keep_place(p, b, s.base + i);
  if (to.page < 0) from.page = -1;
}

// Few tokens: a workgroup takes a sequence's in `each` layers; places are looked up once.  A wave has 64 / PIECES entries of the list and one head,
// keys or values, at a time; entries beyond follow in the next round (a longer list than was expected).
template <int PIECES>
__global__ __launch_bounds__(256) void keep_few_kernel(KeepArgs p, int layers, int each) {
  constexpr int kAtOnce = 64 / PIECES, kUnits = 4;   // units (head, keys or values, layer) of a wave under way
  const int b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x / 64, piece = lane % PIECES;
  const KeepSpan s = keep_span(p, b);
  if (blockIdx.x == 0 && threadIdx.x == 0 && p.k.kept_lens) p.k.kept_lens[b] = (int32_t)(s.base + s.many);
  const int layer0 = blockIdx.x * each, now = min(each, layers - layer0), units = now * p.kv_heads * 2;
  for (int i0 = 0; i0 < s.many; i0 += kAtOnce) {
    Place from, to;
    keep_places(p, b, s, i0 + lane / PIECES, from, to);
    const bool move = from.page >= 0;
    if (!__any(move)) continue;
    for (int u0 = wave; u0 < units; u0 += 4 * kUnits) {
      v4i code[kUnits];
      uint8_t scale[kUnits];
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        const int u = u0 + 4 * k;
        if (u < units && move) {
          const auto& layer = p.layer[layer0 + (u >> 1) / p.kv_heads];
          const int kv = 2 * (u & 1);
          const unsigned row = (unsigned)((u >> 1) % p.kv_heads * p.page_size + from.row) * PIECES + piece;
          code[k] = *reinterpret_cast<const v4i*>(layer.data[kv] + from.page * layer.stride[kv] + (size_t)row * 16);
          scale[k] = layer.data[kv + 1][from.page * layer.stride[kv + 1] + row];
        }
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // read, before any is written
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        const int u = u0 + 4 * k;
        if (u < units && move) {
          const auto& layer = p.layer[layer0 + (u >> 1) / p.kv_heads];
          const int kv = 2 * (u & 1);
          const unsigned row = (unsigned)((u >> 1) % p.kv_heads * p.page_size + to.row) * PIECES + piece;
          *reinterpret_cast<v4i*>(layer.data[kv] + to.page * layer.stride[kv] + (size_t)row * 16) = code[k];
          layer.data[kv + 1][to.page * layer.stride[kv + 1] + row] = scale[k];
        }
      }
    }
  }
}

// Many tokens: a workgroup takes one list.  Places of 2048 entries are looked up at once and lie in LDS; then kEach entries a thread at a time, the next
// ones' bytes requested before the present ones' are waited for (every thread loads, so that how many loads are under way is known: what does not move
// reads the list's first place).
template <int PIECES>
__global__ __launch_bounds__(512) void keep_many_kernel(KeepArgs p) {
  constexpr int kAtOnce = 512 / PIECES, kEach = 4, kStep = kAtOnce * kEach, kChunk = 2048;
  __shared__ int from_slot[kChunk + kStep], to_slot[kChunk + kStep];   // -1: nothing moves
  const int b = blockIdx.y, piece = threadIdx.x % PIECES, mine = threadIdx.x / PIECES, kv = 2 * (blockIdx.x & 1), head = blockIdx.x >> 1;
  const auto& layer = p.layer[blockIdx.z];
  const KeepSpan s = keep_span(p, b);
  if (blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0 && p.k.kept_lens) p.k.kept_lens[b] = (int32_t)(s.base + s.many);
  uint8_t* const codes = layer.data[kv];
  uint8_t* const scales = layer.data[kv + 1];
  const int64_t code_stride = layer.stride[kv], scale_stride = layer.stride[kv + 1];
  const auto row_of = [&](int slot) { return (unsigned)(head * p.page_size + (slot & (p.page_size - 1))) * PIECES + piece; };
  struct Bytes {
    v4i code[kEach];
    int scale[kEach];
  };
  const auto request = [&](int i0, Bytes& x) {   // i0: within the chunk
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int slot = max(from_slot[i0 + e * kAtOnce + mine], 0), page = slot >> p.page_shift;
      const unsigned row = row_of(slot);
      x.code[e] = *reinterpret_cast<const v4i*>(codes + page * code_stride + (size_t)row * 16);
      x.scale[e] = scales[page * scale_stride + row];
    }
  };
  const auto store = [&](int i0, const Bytes& x) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int at = i0 + e * kAtOnce + mine;
      if (from_slot[at] < 0) continue;
      const int slot = to_slot[at], page = slot >> p.page_shift;
      const unsigned row = row_of(slot);
      *reinterpret_cast<v4i*>(codes + page * code_stride + (size_t)row * 16) = x.code[e];
      scales[page * scale_stride + row] = (uint8_t)x.scale[e];
    }
  };
  for (int c0 = 0; c0 < s.many; c0 += kChunk) {
    __syncthreads();
    for (int i = threadIdx.x; i < kChunk + kStep; i += 512) {
      Place from{-1, 0}, to{-1, 0};
      if (i < kChunk) keep_places(p, b, s, c0 + i, from, to);
      from_slot[i] = from.page < 0 ? -1 : from.page << p.page_shift | from.row;
      to_slot[i] = to.page << p.page_shift | to.row;
    }
    __syncthreads();
    const int here = min(s.many - c0, kChunk);
    Bytes now, next;
    request(0, now);
    for (int i0 = 0; i0 < here; i0 += kStep) {
      request(i0 + kStep, next);   // (from places that the present ones do not go to: those are all below them)
#pragma unroll
      for (int e = 0; e < kEach; ++e) asm volatile("" ::"v"(now.code[e]), "v"(now.scale[e]) : "memory");   // read, before anybody writes:
      __syncthreads();                                                                                    // the barrier by itself waits for no load
      store(i0, now);
      now = next;
    }
  }
}

template <int PIECES>
void launch_keep(const KeepArgs& p, int layers, int cus, hipStream_t s) {
  for (int b = 0; b < p.k.batch; b += 65535) {
    KeepArgs part = p;
    part.k.page_table = p.k.page_table + (int64_t)b * p.k.page_table_stride;
    part.k.seq_lens += b, part.k.cu_q += b, part.k.accepted += b;
    if (part.k.kept_lens) part.k.kept_lens += b;
    const unsigned y = (unsigned)std::min(p.k.batch - b, 65535);
    if (p.k.max_q <= 256) {
      const int each = std::max(1, std::min(layers, (int)((int64_t)layers * y / (8 * cus))));
      hipLaunchKernelGGL((keep_few_kernel<PIECES>), dim3((unsigned)((layers + each - 1) / each), y), dim3(256), 0, s, part, layers, each);
    } else {
      hipLaunchKernelGGL((keep_many_kernel<PIECES>), dim3(2 * (unsigned)p.kv_heads, y, (unsigned)layers), dim3(512), 0, s, part);
    }
  }
}

}  // namespace

hipError_t launch_draft_tree(const int32_t* parents, const int32_t* cu_q, const int32_t* seq_lens, int tokens, int batch, uint64_t* seen, int words,
                             int32_t* positions, hipStream_t s) {
  hipLaunchKernelGGL(draft_tree_kernel, dim3((unsigned)std::min(batch, 1 << 16)), dim3(kTreeThreads), 0, s, parents, cu_q, seq_lens, tokens, batch, seen, words,
                     positions);
  return hipGetLastError();
}

hipError_t launch_keep_kv(const ave_fp4_kv_cache* caches, int layers, const ave_fp4_keep& k, hipStream_t s) {
  const ave_fp4_kv_cache& c0 = caches[0];
  const int cus = compute_units();
  if (cus <= 0) return hipErrorInvalidDevice;
  for (int from = 0; from < layers; from += kLayers) {
    const int now = std::min(layers - from, kLayers);
    KeepArgs p{};
    p.k = k, p.pages = c0.pages, p.kv_heads = c0.kv_heads, p.page_size = c0.page_size, p.page_shift = log2_of(c0.page_size);
    if (from > 0) p.k.kept_lens = nullptr;
    for (int i = 0; i < now; ++i) {
      const ave_fp4_kv_cache& c = caches[from + i];
      p.layer[i] = {{c.k, c.k_scale, c.v, c.v_scale}, {c.k_page_stride, c.k_scale_page_stride, c.v_page_stride, c.v_scale_page_stride}};
    }
    if (c0.head_dim == 64) launch_keep<2>(p, now, cus, s);
    else if (c0.head_dim == 128) launch_keep<4>(p, now, cus, s);
    else launch_keep<8>(p, now, cus, s);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace ave
