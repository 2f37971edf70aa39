// Host-side launch interface of the kernels around the MXFP4 key/value cache, and the device-side view of it.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ave_fp4.h"

namespace ave {

inline int log2_of(int v) {
  int n = 0;
  while ((1 << n) < v) ++n;
  return n;
}

// Any of q, k, v may be absent (data null).  q and, without a cache, k leave as bf16; with a cache k and v are quantised into it.
struct HeadArgs {
  ave_fp4_heads q{}, k{}, v{}, q_out{}, k_out{};
  ave_fp4_norm_rope how{};
  ave_fp4_kv_cache cache{};
  const int32_t* slots = nullptr;
  int tokens = 0, head_dim = 0;
};
hipError_t launch_heads(const HeadArgs& p, hipStream_t s);
hipError_t launch_gather_kv(const ave_fp4_kv_cache& cache, const int32_t* slots, int tokens, uint16_t* k, uint16_t* v, hipStream_t s);

hipError_t launch_attention(const ave_fp4_attention& a, const ave_fp4_kv_cache& cache, void* workspace, hipStream_t s);
size_t attention_workspace_bytes(const ave_fp4_attention& a, const ave_fp4_kv_cache& cache);
hipError_t launch_tree_attention(const ave_fp4_attention& a, const ave_fp4_tree& t, const ave_fp4_kv_cache& cache, void* workspace, hipStream_t s);
size_t tree_attention_workspace_bytes(const ave_fp4_attention& a, const ave_fp4_tree& t, const ave_fp4_kv_cache& cache);

hipError_t launch_draft_tree(const int32_t* parents, const int32_t* cu_q, const int32_t* seq_lens, int tokens, int batch, uint64_t* seen, int words,
                             int32_t* positions, hipStream_t s);
hipError_t launch_verify_draft(const ave_fp4_draft& d, void* workspace, hipStream_t s);
size_t verify_draft_workspace_bytes(const ave_fp4_draft& d);
constexpr int kVocabPiece = 8192;   // of the vocabulary, of a workgroup
hipError_t launch_keep_kv(const ave_fp4_kv_cache* caches, int layers, const ave_fp4_keep& k, hipStream_t s);

}  // namespace ave
