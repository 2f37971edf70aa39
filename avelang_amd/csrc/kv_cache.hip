// What stands between the qkv projection and attention: norms of query and key heads, rotation by position, and the
// quantiser that appends keys and values to a paged MXFP4 cache; and the way back from the cache to bf16.
//
// Norm:      n = (x * r) * w,  r = 1 / sqrt(sum(x^2) / D + eps)
// Rotation:  a' = a cos - b sin,  b' = b cos + a sin   for the pairs (i, i + R/2) or (2i, 2i + 1), i < R/2
// Quantiser: per 32 channels, as quantize_mx.hip.
// Every product and sum is rounded by itself (no contraction) and the squares are added up neighbours first -- eight in a lane, then
// lanes 1, 2, 4, ... apart -- so that codes behind a norm and a rotation are the same bits wherever they are computed.
//
// Bound by HBM for a prompt (each input read once, each output written once), by latency for a decode batch: one launch for
// all roles of heads.  8192 tokens, 32 query and 8 key heads of 128, norm and rotation: 41 us, 4.2 TB/s; the append of 64 + 8 + 8 heads of 64:
// 32 us, 5.0 TB/s (a large copy reaches 5.2); the way back 4.3 TB/s.  64 tokens of 32 + 8 + 8 heads of 128: 3.8 us in a graph.  From fp32 54 us
// (4.8 TB/s) and 45 us (5.4).
#include "fp4_common.hpp"
#include "kv_cache.hpp"

#pragma clang fp contract(off)

namespace ave {
namespace {

// Eight consecutive elements, as they are: from any address of their type unless ALIGNED says 16 bytes
template <typename T>
struct Eight {
  v4i raw[sizeof(T) / 2];
};
template <bool ALIGNED, typename T>
__device__ inline Eight<T> load8(const T* p) {
  Eight<T> r;
  if (ALIGNED || (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
    for (int q = 0; q < (int)sizeof(T) / 2; ++q) r.raw[q] = ALIGNED ? __builtin_nontemporal_load(reinterpret_cast<const v4i*>(p) + q) : reinterpret_cast<const v4i*>(p)[q];
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j) r.raw[j / 4][j % 4] = reinterpret_cast<const int*>(p)[j];
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) r.raw[0][j] = (int)((unsigned)h[2 * j] | (unsigned)h[2 * j + 1] << 16);
  }
  return r;
}
template <typename T>
__device__ inline void unpack(const Eight<T>& r, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (sizeof(T) == 4) v[j] = __builtin_bit_cast(float, (int)r.raw[j / 4][j % 4]);
    else v[j] = __builtin_bit_cast(float, j % 2 ? (unsigned)r.raw[0][j / 2] & 0xFFFF0000u : (unsigned)r.raw[0][j / 2] << 16);
  }
}

__device__ inline void store8_bf16(uint16_t* p, const float (&v)[8], bool stream) {
  const v4i w = {(int)pack_bf16x2(v[0], v[1]), (int)pack_bf16x2(v[2], v[3]), (int)pack_bf16x2(v[4], v[5]), (int)pack_bf16x2(v[6], v[7])};
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    if (stream) __builtin_nontemporal_store(w, reinterpret_cast<v4i*>(p));
    else *reinterpret_cast<v4i*>(p) = w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = (uint16_t)((unsigned)w[j / 2] >> (16 * (j % 2)));
  }
}

// D / 8 lanes share a head, eight channels each; a workgroup has 2048 / D heads of one token side by side, and `each` (at most kEach) such
// groups -- queries, then keys, then values -- under way at once: what bounds a prompt is how many bytes are.  Neighbouring tokens go to
// one XCD, whose L2 puts their pieces of a cache line together.  A pair's other half comes from the lane that has it.  (One group after the other,
// the other half loaded again, tokens dealt out to the XCDs: 69 and 52 us where this came to 44 and 34.)
constexpr int kEach = 4;

template <typename T, int D, bool ALIGNED>
__global__ __launch_bounds__(256) void heads_kernel(HeadArgs p, int q_heads, int all_heads, int each, int page_shift) {
  constexpr int L = D / 8;
  const int token = blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8, lane = threadIdx.x % L, c0 = lane * 8;
  if (token >= p.tokens) return;
  const int h0 = blockIdx.y * each * (256 / L) + threadIdx.x / L;
  Eight<T> raw[kEach];
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    const int h = h0 + u * (256 / L);
    if (u >= each || h >= all_heads) continue;
    const bool is_q = h < q_heads, is_v = p.v.data && h >= q_heads + p.k.heads;
    const int head = is_q ? h : is_v ? h - q_heads - p.k.heads : h - q_heads;
    const void* data = is_q ? p.q.data : is_v ? p.v.data : p.k.data;
    const int64_t token_stride = is_q ? p.q.token_stride : is_v ? p.v.token_stride : p.k.token_stride;
    const int64_t head_stride = is_q ? p.q.head_stride : is_v ? p.v.head_stride : p.k.head_stride;
    raw[u] = load8<ALIGNED>(static_cast<const T*>(data) + token * token_stride + head * head_stride + c0);
  }
  // inputs are read once, outputs of prompts are larger than the caches on the way (8192 tokens: 45.7 us without the hints, 41.3 with; the append
  // and the way back 43.8 and 38.8)
  const bool stream = gridDim.x >= 1024;
  const int half = p.how.rotary_dim / 2;
  const bool turned = p.how.cos && c0 < 2 * half;
  const bool upper = !p.how.neighbours && c0 >= half;      // this lane's channels are the second ones of their pairs
  const int partner = (threadIdx.x & 63) + (upper ? -half / 8 : half / 8);   // the lane that has the others
  float cs[8], sn[8];
  if (turned) {
    const int pos = p.how.positions[token];
    if (pos >= 0 && pos < p.how.table_rows) {
      const size_t row = (size_t)pos * half;
      if (p.how.neighbours) {
#pragma unroll
        for (int j = 0; j < 8; ++j) cs[j] = p.how.cos[row + c0 / 2 + j / 2], sn[j] = p.how.sin[row + c0 / 2 + j / 2];
      } else {
        unpack(load8<false>(p.how.cos + row + (upper ? c0 - half : c0)), cs);
        unpack(load8<false>(p.how.sin + row + (upper ? c0 - half : c0)), sn);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) cs[j] = sn[j] = __builtin_nanf("");
    }
  }
  const int slot = p.slots ? p.slots[token] : -1, page = slot >> page_shift;
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    const int h = h0 + u * (256 / L);
    if (u >= each || h >= all_heads) continue;
    const bool is_q = h < q_heads, is_v = p.v.data && h >= q_heads + p.k.heads;
    const int head = is_q ? h : is_v ? h - q_heads - p.k.heads : h - q_heads;
    float x[8];
    unpack(raw[u], x);
    if (!is_v) {
      const void* weight = is_q ? p.how.q_weight : p.how.k_weight;
      if (weight) {
        float s[8], w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = x[j] * x[j];
        float sum = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
#pragma unroll
        for (int m = 1; m < L; m *= 2) sum += __shfl_xor(sum, m, 64);
        const float r = 1.0f / sqrtf(sum / (float)D + p.how.eps);
        if (p.how.weight_is_f32) unpack(load8<false>(static_cast<const float*>(weight) + c0), w);
        else unpack(load8<false>(static_cast<const __bf16*>(weight) + c0), w);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (x[j] * r) * w[j];
      }
      if (turned) {
        if (p.how.neighbours) {
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const float a = x[j], b = x[j + 1];
            x[j] = a * cs[j] - b * sn[j];
            x[j + 1] = b * cs[j] + a * sn[j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float y = __shfl(x[j], partner, 64);
            x[j] = upper ? x[j] * cs[j] + y * sn[j] : x[j] * cs[j] - y * sn[j];
          }
        }
      }
    }
    if (is_q || (!is_v && p.k_out.data)) {
      void* data = is_q ? p.q_out.data : p.k_out.data;
      const int64_t token_stride = is_q ? p.q_out.token_stride : p.k_out.token_stride, head_stride = is_q ? p.q_out.head_stride : p.k_out.head_stride;
      store8_bf16(static_cast<uint16_t*>(data) + token * token_stride + head * head_stride + c0, x, stream);
    } else {
      const unsigned amax = lane_xor_max_bits(lane_xor_max_bits(abs_max_bits(x), 1), 2);   // four lanes share a block
      const int byte = mx_scale_byte(amax);
      const float scale = mx_scale_value(byte);
      unsigned codes = 0;
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], scale, 0);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], scale, 1);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], scale, 2);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], scale, 3);
      if (byte == 0xFF) codes = 0u;
      if (slot >= 0 && page < p.cache.pages) {
        const size_t row = (size_t)head * p.cache.page_size + (slot & (p.cache.page_size - 1));   // within the page
        uint8_t* c = (is_v ? p.cache.v + page * p.cache.v_page_stride : p.cache.k + page * p.cache.k_page_stride) + row * (D / 2);
        uint8_t* f = (is_v ? p.cache.v_scale + page * p.cache.v_scale_page_stride : p.cache.k_scale + page * p.cache.k_scale_page_stride) + row * (D / 32);
        reinterpret_cast<unsigned*>(c)[lane] = codes;
        if (lane % 4 == 0) f[lane / 4] = (uint8_t)byte;
      }
    }
  }
}

template <typename T, int D>
hipError_t launch_some_heads(const HeadArgs& p, hipStream_t s) {
  const int q = p.q.data ? p.q.heads : 0, all = q + (p.k.data ? p.k.heads : 0) + (p.v.data ? p.v.heads : 0);
  const int groups = (all + 2048 / D - 1) / (2048 / D);
  if (all == 0) return hipSuccess;
  // few tokens: a workgroup for every group of heads; many: the fewest, which load their cosines once (32 + 8 + 8 heads of 128, 64 tokens 3.8 us
  // so, 5.7 otherwise; 512 5.8 and 6.7, 1024 9.1 and 8.7, 8192 50 and 43)
  const int want = (groups + kEach - 1) / kEach, each = p.tokens >= 1024 ? (groups + want - 1) / want : 1;
  const auto wide = [](const ave_fp4_heads& h) {
    return !h.data || ((reinterpret_cast<uintptr_t>(h.data) & 15) == 0 && h.token_stride * (int64_t)sizeof(T) % 16 == 0 && h.head_stride * (int64_t)sizeof(T) % 16 == 0);
  };
  const dim3 grid((unsigned)((p.tokens + 7) / 8 * 8), (unsigned)((groups + each - 1) / each));
  const int shift = log2_of(p.cache.page_size);
  if (wide(p.q) && wide(p.k) && wide(p.v)) hipLaunchKernelGGL((heads_kernel<T, D, true>), grid, dim3(256), 0, s, p, q, all, each, shift);
  else hipLaunchKernelGGL((heads_kernel<T, D, false>), grid, dim3(256), 0, s, p, q, all, each, shift);
  return hipGetLastError();
}

// A workgroup of 256 for every token: a launch has less than 2^32 threads (with more HIP starts some of them and reports nothing), so that 2^23
// tokens go at once.
template <typename T, int D>
hipError_t launch_heads_as(HeadArgs p, hipStream_t s) {
  constexpr int kMost = 1 << 23;
  for (int left = p.tokens; left > 0; left -= kMost) {
    p.tokens = left < kMost ? left : kMost;
    if (hipError_t e = launch_some_heads<T, D>(p, s); e != hipSuccess) return e;
    const auto on = [&](ave_fp4_heads& h, size_t element) {
      if (h.data) h.data = static_cast<char*>(h.data) + h.token_stride * kMost * (int64_t)element;
    };
    on(p.q, sizeof(T)), on(p.k, sizeof(T)), on(p.v, sizeof(T)), on(p.q_out, 2), on(p.k_out, 2);
    if (p.how.positions) p.how.positions += kMost;
    if (p.slots) p.slots += kMost;
  }
  return hipSuccess;
}

// A lane takes eight channels of one head of one token.
template <int D>
__global__ __launch_bounds__(256) void gather_kv_kernel(ave_fp4_kv_cache c, const int32_t* slots, size_t pieces, uint16_t* k, uint16_t* v,
                                                        int page_shift) {
  constexpr int L = D / 8;
  const size_t per_token = (size_t)c.kv_heads * L;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < 2 * pieces; i += (size_t)gridDim.x * 256) {
    const bool is_v = i >= pieces;
    const size_t at = is_v ? i - pieces : i;
    const size_t token = at / per_token;
    const unsigned rest = (unsigned)(at - token * per_token), head = rest / L, lane = rest % L;
    const int slot = slots[token], page = slot >> page_shift;
    v4i out = {0, 0, 0, 0};
    if (slot >= 0 && page < c.pages) {
      const size_t row = (size_t)head * c.page_size + (slot & (c.page_size - 1));
      const uint8_t* codes = (is_v ? c.v + page * c.v_page_stride : c.k + page * c.k_page_stride) + row * (D / 2);
      const uint8_t* scales = (is_v ? c.v_scale + page * c.v_scale_page_stride : c.k_scale + page * c.k_scale_page_stride) + row * (D / 32);
      const unsigned x = reinterpret_cast<const unsigned*>(codes)[lane];
      const int byte = scales[lane / 4];
      const float scale = byte == 0xFF ? __builtin_nanf("") : mx_scale_value(byte);
      const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, 1.0f, 1);
      const v2f d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, 1.0f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, 1.0f, 3);
      out = v4i{(int)pack_bf16x2(a[0] * scale, a[1] * scale), (int)pack_bf16x2(b[0] * scale, b[1] * scale),
                (int)pack_bf16x2(d[0] * scale, d[1] * scale), (int)pack_bf16x2(e[0] * scale, e[1] * scale)};
    }
    reinterpret_cast<v4i*>(is_v ? v : k)[at] = out;
  }
}

}  // namespace

hipError_t launch_heads(const HeadArgs& p, hipStream_t s) {
  const bool f32 = p.q.data ? p.q.is_f32 : p.k.is_f32;
  switch (p.head_dim) {
    case 64: return f32 ? launch_heads_as<float, 64>(p, s) : launch_heads_as<__bf16, 64>(p, s);
    case 128: return f32 ? launch_heads_as<float, 128>(p, s) : launch_heads_as<__bf16, 128>(p, s);
    default: return f32 ? launch_heads_as<float, 256>(p, s) : launch_heads_as<__bf16, 256>(p, s);
  }
}

hipError_t launch_gather_kv(const ave_fp4_kv_cache& c, const int32_t* slots, int tokens, uint16_t* k, uint16_t* v, hipStream_t s) {
  const size_t pieces = (size_t)tokens * c.kv_heads * (c.head_dim / 8);
  if (pieces == 0) return hipSuccess;
  size_t grid = (2 * pieces + 255) / 256;
  if (grid > 1u << 16) grid = 1u << 16;
  const int shift = log2_of(c.page_size);
#define AVE_GATHER(D) hipLaunchKernelGGL((gather_kv_kernel<D>), dim3((unsigned)grid), dim3(256), 0, s, c, slots, pieces, k, v, shift)
  if (c.head_dim == 64) AVE_GATHER(64);
  else if (c.head_dim == 128) AVE_GATHER(128);
  else AVE_GATHER(256);
#undef AVE_GATHER
  return hipGetLastError();
}

}  // namespace ave
