// Attention over a paged MXFP4 key/value cache: one wave per query row, all in fp32.
//   out = sum_j exp(s_j) v_j / (sum_j exp(s_j) + exp(sink)),  s_j = scale * q . k_j,  over the keys the row sees
// One pass over the keys, 64 at a time, with the running maximum and sum of the softmax.
#include "fp4_common.hpp"
#include "attn_common.hpp"
#include "kernels.hpp"

namespace ave {
namespace {

__device__ inline float wave_max(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m /= 2) v = fmaxf(v, __shfl_xor(v, m, 64));
  return v;
}
__device__ inline float wave_sum(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m /= 2) v += __shfl_xor(v, m, 64);
  return v;
}

template <int D>
__global__ __launch_bounds__(64) void attention_row_kernel(ave_fp4_attention a, ave_fp4_kv_cache c, int page_shift) {
  __shared__ float q[D];
  __shared__ float prob[64];
  const int token = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
  const int kv_head = head / (a.heads / c.kv_heads);
  int b = token, first = token, end = token + 1;
  if (a.cu_q) {   // the last sequence that starts at or before the token
    int lo = 0, hi = a.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (a.cu_q[mid] <= token) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    first = a.cu_q[b], end = a.cu_q[b + 1];
    if (token < first || token >= end) return;
  }
  int len = a.seq_lens[b];
  const int most = a.table_pages << page_shift;
  len = len < 0 ? 0 : len > most ? most : len;
  const int pos = len - (end - first) + (token - first);
  const int hi = a.causal ? (pos + 1 < len ? pos + 1 : len) : len;
  const int lo = a.window > 0 && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
  for (int i = lane; i < D; i += 64) {
    const unsigned bits = a.q[token * a.q_token_stride + head * a.q_head_stride + i];
    q[i] = __builtin_bit_cast(float, bits << 16);
  }
  __syncthreads();
  constexpr int C = D / 64;   // channels of the result per lane
  float acc[C] = {}, m = -INFINITY, l = 0.0f;
  const auto page_of = [&](int j) {
    const int page = a.page_table[b * a.page_table_stride + (j >> page_shift)];
    return page < 0 ? 0 : page >= c.pages ? c.pages - 1 : page;
  };
  const auto row_of = [&](int j) { return (size_t)kv_head * c.page_size + (j & (c.page_size - 1)); };
  for (int j0 = lo; j0 < hi; j0 += 64) {
    const int j = j0 + lane;
    float s = -INFINITY;
    if (j < hi) {
      const int page = page_of(j);
      const uint8_t* codes = c.k + page * c.k_page_stride + row_of(j) * (D / 2);
      const uint8_t* scales = c.k_scale + page * c.k_scale_page_stride + row_of(j) * (D / 32);
      s = 0.0f;
      for (int blk = 0; blk < D / 32; ++blk) {
        const v4i x = reinterpret_cast<const v4i*>(codes)[blk];
        const int byte = scales[blk];
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const v2f v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((unsigned)x[w], 1.0f, 0), v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((unsigned)x[w], 1.0f, 1);
          const v2f v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((unsigned)x[w], 1.0f, 2), v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((unsigned)x[w], 1.0f, 3);
          const float* qq = q + blk * 32 + w * 8;
          sum += v0[0] * qq[0] + v0[1] * qq[1] + v1[0] * qq[2] + v1[1] * qq[3] + v2[0] * qq[4] + v2[1] * qq[5] + v3[0] * qq[6] + v3[1] * qq[7];
        }
        s += sum * (byte == 0xFF ? __builtin_nanf("") : mx_scale_value(byte));
      }
      s *= a.scale;
    }
    const float m_new = fmaxf(m, wave_max(s));
    const float p = j < hi ? expf(s - m_new) : 0.0f, fade = m == -INFINITY ? 0.0f : expf(m - m_new);
    m = m_new;
    l = l * fade + wave_sum(p);
    prob[lane] = p;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] *= fade;
    const int n = hi - j0 < 64 ? hi - j0 : 64;
    for (int t = 0; t < n; ++t) {
      const int page = page_of(j0 + t);
      const uint8_t* codes = c.v + page * c.v_page_stride + row_of(j0 + t) * (D / 2);
      const int byte = c.v_scale[page * c.v_scale_page_stride + row_of(j0 + t) * (D / 32) + lane * C / 32];
      const float f = prob[t] * (byte == 0xFF ? __builtin_nanf("") : mx_scale_value(byte));
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int ch = lane * C + i;
        const unsigned code = (codes[ch / 2] >> (4 * (ch % 2))) & 15u;
        acc[i] += f * __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 0)[0];
      }
    }
    __syncthreads();
  }
  if (a.sinks && l > 0.0f) {
    const float sink = a.sinks[head], m_new = fmaxf(m, sink), fade = expf(m - m_new);
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] *= fade;
    l = l * fade + expf(sink - m_new);
    m = m_new;
  }
  const bool none = hi <= lo;
  uint16_t* out = a.out + ((size_t)token * a.heads + head) * D + lane * C;
#pragma unroll
  for (int i = 0; i < C; ++i) out[i] = none ? (uint16_t)0 : to_bf16(acc[i] / l);
  if (a.lse && lane == 0) a.lse[(size_t)token * a.heads + head] = none ? (a.sinks ? a.sinks[head] : -INFINITY) : m + logf(l);
}

}  // namespace

namespace {

AttnArgs args_of(const ave_fp4_attention& a, const ave_fp4_kv_cache& c) {
  AttnArgs p{};
  p.a = a, p.c = c;
  set_group(p, a.heads / c.kv_heads);
  p.page_shift = log2_of(c.page_size);
  return p;
}

// Row tiles of 16 of the kernel for few rows; 0: another kernel
int decode_row_tiles(const AttnArgs& p) {
  const int64_t rows = (int64_t)(p.a.cu_q ? p.a.max_q : 1) * p.group;
  const int most = p.c.head_dim == 256 ? 32 : 64;
  return rows > most ? 0 : rows > 32 ? 4 : rows > 16 ? 2 : 1;
}

}  // namespace

size_t attention_workspace_bytes(const ave_fp4_attention& a, const ave_fp4_kv_cache& c) {
  const AttnArgs p = args_of(a, c);
  if (const int tiles = decode_row_tiles(p)) return attn_decode_workspace(p, tiles);
  return 0;
}

hipError_t launch_attention(const ave_fp4_attention& a, const ave_fp4_kv_cache& c, void* workspace, hipStream_t s) {
  const AttnArgs args = args_of(a, c);
  if (const int tiles = decode_row_tiles(args)) return launch_attn_decode(args, tiles, workspace, s);
  const dim3 grid((unsigned)a.tokens, (unsigned)a.heads);
  const int shift = log2_of(c.page_size);
#define AVE_ROW(D) hipLaunchKernelGGL((attention_row_kernel<D>), grid, dim3(64), 0, s, a, c, shift)
  if (c.head_dim == 64) AVE_ROW(64);
  else if (c.head_dim == 128) AVE_ROW(128);
  else AVE_ROW(256);
#undef AVE_ROW
  return hipGetLastError();
}

}  // namespace ave
