/*
 * ave_fp4.h -- C ABI of libave_fp4.so: block-scaled FP4 GEMM for AMD MI355X (gfx950).
 *
 * Every entry point computes  C[M,N] (bf16) = A[M,K] . B[N,K]^T  with fp32
 * accumulation and a round-to-nearest-even bf16 store.  All data pointers are
 * DEVICE pointers to row-major contiguous arrays.  Calls enqueue work on the
 * given HIP stream and return immediately; they never synchronise and never
 * allocate, so they may be recorded into a HIP graph.
 *
 * Packed E2M1: two 4-bit codes per byte, LOW nibble = even k.
 *
 * Return value: 0 on success; AVE_FP4_EINVAL (-1) for a rejected argument;
 * otherwise the hipError_t of the failing HIP call.  ave_fp4_last_error()
 * returns the message for the calling thread.
 *
 * Reference interface each entry point stands in for (causalflow-ai/avelang):
 *   host wrapper  python/avelang_kernels/amdgpu_gemm.py:458-494
 *                 (gemm_pipeline_transposed_b: validate, allocate out, launch)
 *   launch path   python/avelang/runtime/jit.py:791-831 and
 *                 python/avelang/backends/amdgpu/driver.py:325-365
 *                 (current stream, raw data pointers, asynchronous, no sync)
 *   error text    python/avelang/backends/amdgpu/driver.py:125-138
 * The reference has only a bf16 kernel; the FP4 signatures below extend its
 * (A, B, out) convention with the block-scale tensors.
 */
#ifndef AVE_FP4_H_
#define AVE_FP4_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define AVE_FP4_EINVAL (-1)

/* Kernel selection for the *_ex entry points (testing and benchmarking). */
enum ave_fp4_variant {
  AVE_FP4_AUTO = 0,    /* shape-based dispatch, what the plain entry points use */
  AVE_FP4_GENERIC = 1, /* one wave per 32x32 tile, no LDS; any shape */
  AVE_FP4_TILE = 2,    /* 256x256 LDS-staged MFMA kernel; MXFP4: K % 256 == 0, or any multiple of 32 from 512 up with
                          16-byte aligned A and B (512 * n is fastest); NVFP4: K % 256 == 0 */
  AVE_FP4_DECODE = 3,  /* weight-streaming small-M kernel; MXFP4: M <= 64 and K a multiple of 32 from 512 up (16-byte
                          aligned operands), or M <= 16 and
                          K % 128 == 0 (K % 32 == 0 for up to 16 MB of weights);
                          NVFP4: M <= 64 and K % 128 == 0, or M <= 32 and K a multiple of 32 from 512 up, or
                          M <= 64 and K a multiple of 32 from 1024 up with an even number of whole 512-element units */
  AVE_FP4_NARROW = 4,  /* NVFP4: 64x128 (up to 64 rows) or 128x128 tiles, any K from 256 up (a multiple of 16; A and B 8-byte
                          aligned).  MXFP4: 256x128 tiles, three stage buffers; needs K a multiple of 32 from 512 up and 16-byte aligned scale
                          tensors; shape-based dispatch takes it for more than 64 rows when its tiles fit the compute units,
                          and for 33..64 rows against a nearly full round of 128-row tiles (N around 28672..32768 on 256
                          compute units) */
  AVE_FP4_TILE_F16 = 5, /* NVFP4 only: 256x256 tiles whose operands are dequantised to f16 once per workgroup on their way
                          into LDS, in steps of 64 elements of K; any K (a multiple of 16: a last step of 16, 32 or 48
                          elements is staged with zeros behind it).  Shape-based dispatch takes it for prefill shapes with
                          K % 64 == 0 and K % 256 != 0, where AVE_FP4_TILE cannot run, and below K = 1024 for K % 256 != 0
                          when C holds more than 1536 blocks of 32 x 32 */
  AVE_FP4_TILE_STREAMED = 6, /* MXFP4 plain GEMM only: AVE_FP4_TILE with look-ahead touches -- eight K stages before a
                          tile's end the workgroups request the weight panels of their next tiles, so that weights
                          which come from HBM (a model's layers, each with weights of its own) are in the last-level
                          cache when their stage loads ask for them; takes effect with K % 512 == 0, 16-byte aligned
                          scale tensors and more 256 x 256 tiles than compute units, and is AVE_FP4_TILE otherwise.
                          Requests go out for whole groups of 32 rows of tiles (8192 rows of A); with fewer the form runs
                          and requests nothing.
                          Same bits as AVE_FP4_TILE; on 8192 x 14336 x 4096 7 % faster on weights from HBM, 1 %
                          slower on cache-resident ones.  Also for the fused SwiGLU forms.  Shape-based dispatch keeps,
                          per device, the weight tensors of its latest MXFP4 GEMMs: weights found among the most
                          recent ones that add up to 192 MB at most are taken to be in the 256 MB last-level cache
                          (one GEMM replayed on the same operands) and run as AVE_FP4_TILE, all others from 32 rows of tiles
                          up as this form */
  AVE_FP4_SHORT = 7    /* MXFP4 plain GEMM only: 32x32 blocks of C, four waves each that share K (up to 2048), operands straight
                          into registers; for small calls */
};

/*
 * MXFP4: A [M, K/2] packed E2M1, A_scale [M, K/32] E8M0 bytes (2^(b-127), one per
 * 32 consecutive k); B [N, K/2], B_scale [N, K/32] likewise; C [M, N] bf16.
 * K must be a positive multiple of 32.  Replaces gemm_pipeline_transposed_b
 * (amdgpu_gemm.py:458-494) for MXFP4 operands; the reference's M % 128 / N % 128
 * restriction (amdgpu_gemm.py:471-474) is lifted.
 */
int ave_fp4_gemm_mxfp4(const uint8_t* A, const uint8_t* A_scale, const uint8_t* B, const uint8_t* B_scale,
                       uint16_t* C, int M, int N, int K, void* hip_stream);
int ave_fp4_gemm_mxfp4_ex(const uint8_t* A, const uint8_t* A_scale, const uint8_t* B, const uint8_t* B_scale,
                          uint16_t* C, int M, int N, int K, void* hip_stream, int variant);

/*
 * The same GEMM with a caller-provided device workspace, for shapes with far fewer 256 x 256 output tiles than
 * compute units and a long K (a few hundred rows of activations against a weight matrix with few rows, e.g.
 * 128..2048 x 4096 x 14336): K is cut into slices that run on different compute units, each slice's fp32 sums go
 * to the workspace, and a second kernel adds them in slice order and rounds to bf16 (deterministic; within the
 * same tolerance as the unsplit GEMM but not bit-identical to it, since the fp32 additions associate differently).
 * ave_fp4_gemm_mxfp4_workspace_bytes returns the bytes this takes for a shape on the current device, 0 when K
 * would not be split.  With a smaller (or null) workspace, or scale tensors that are not 16-byte aligned, the call
 * is ave_fp4_gemm_mxfp4.  The workspace must be 16-byte aligned; its contents need no initialisation and are
 * garbage afterwards; calls that may overlap on the device need workspaces of their own.  The library itself never
 * allocates.  No counterpart in the reference, whose gemm_pipeline_transposed_b (amdgpu_gemm.py:458-494) runs one
 * workgroup per output tile over the whole of K.
 */
size_t ave_fp4_gemm_mxfp4_workspace_bytes(int M, int N, int K);
int ave_fp4_gemm_mxfp4_ws(const uint8_t* A, const uint8_t* A_scale, const uint8_t* B, const uint8_t* B_scale,
                          uint16_t* C, int M, int N, int K, void* workspace, size_t workspace_bytes, void* hip_stream);
/*
 * The same GEMM for callers that cannot allocate: code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc.  No counterpart in the reference.  It is ave_fp4_gemm_mxfp4_ws with the partial sums of the K
 * split in a buffer that the library itself holds -- a static device array of AVE_FP4_NOALLOC_SCRATCH_BYTES, one
 * copy per GPU for the life of the process -- instead of a caller's workspace: same kernels and, wherever that split's
 * partial sums fit the scratch (e.g. 512 x 4096 x 14336, which takes exactly the 32 MiB), the same split and bit-identical
 * results.  The call allocates nothing and frees nothing.  The K split is planned under the scratch's size: where
 * ave_fp4_gemm_mxfp4_ws would want more partial sums than the scratch holds (on 256 compute units: a few hundred rows
 * against a K of about 30000 and more, e.g. 640 x 4096 x 32768 with 50 MiB) this call takes the best split that fits --
 * fewer, longer slices, or none -- so every shape the plain entry point accepts is accepted here, and the result then
 * differs from ave_fp4_gemm_mxfp4_ws's in the association of the fp32 sums only (same tolerance);
 * a shape that is not split runs as ave_fp4_gemm_mxfp4.  The scratch needs no initialisation (every partial sum
 * that is read was written by the same call) and keeps the last call's contents.  ALL calls on one GPU share the one
 * array: calls that may overlap on a GPU (different streams, or graphs replayed concurrently) race -- serialise
 * them, or give the others a workspace of their own through ave_fp4_gemm_mxfp4_ws.  The first call on a device looks
 * the array's address up; make it outside stream capture.
 */
#define AVE_FP4_NOALLOC_SCRATCH_BYTES (32u << 20)
int ave_fp4_gemm_mxfp4_noalloc(const uint8_t* A, const uint8_t* A_scale, const uint8_t* B, const uint8_t* B_scale,
                               uint16_t* C, int M, int N, int K, void* hip_stream);

/*
 * The GEMM as the library would run it when it may use a workspace: ave_fp4_gemm_mxfp4_ws's splits and those of the streaming kernel
 * (more than 64 rows, or 33 - 64 from K = 12288; any K % 32 == 0), whichever a model of the times puts first.
 * ave_fp4_gemm_mxfp4_planned_workspace_bytes gives the size, 0 where K is not split; the contract is that of
 * ave_fp4_gemm_mxfp4_ws.
 */
size_t ave_fp4_gemm_mxfp4_planned_workspace_bytes(int M, int N, int K);
int ave_fp4_gemm_mxfp4_planned(const uint8_t* A, const uint8_t* A_scale, const uint8_t* B, const uint8_t* B_scale,
                               uint16_t* C, int M, int N, int K, void* workspace, size_t workspace_bytes, void* hip_stream);

/*
 * MXFP4 gate+up GEMM with the SwiGLU activation fused into the epilogue:
 *   C[m, n] = silu(g) * u,  g = sum_k A[m,k] B[n,k],  u = sum_k A[m,k] B[N+n,k],  silu(x) = x / (1 + exp(-x)),
 * evaluated in fp32 on the fp32 accumulators, then rounded to bf16.  B [2N, K/2] and B_scale
 * [2N, K/32] hold the N gate rows followed by the N up rows; C is [M, N].  M <= 32 with N % 8 == 0
 * and K a multiple of 32 from 512 up runs on the weight-streaming kernel (AVE_FP4_DECODE); up to 64 rows on that or, where a model
 * of their times says so, on 32- to 128-row tiles by 128 weight rows; larger M with K % 512 == 0 and
 * 16-byte-aligned scale tensors -- or any K that is a multiple of 32 from 512 up with 16-byte aligned A and B --
 * on the LDS-staged kernel (AVE_FP4_TILE: a tile is 256 rows by 128 outputs,
 * its gate and up values meet in LDS as fp32); any other shape on the shape-agnostic kernel (AVE_FP4_GENERIC).  Extends gemm_pipeline_transposed_b
 * (amdgpu_gemm.py:458-494), which has no epilogue beyond the bf16 store (amdgpu_gemm.py:293-329).
 */
int ave_fp4_gemm_mxfp4_swiglu(const uint8_t* A, const uint8_t* A_scale, const uint8_t* B, const uint8_t* B_scale,
                              uint16_t* C, int M, int N, int K, void* hip_stream);
int ave_fp4_gemm_mxfp4_swiglu_ex(const uint8_t* A, const uint8_t* A_scale, const uint8_t* B, const uint8_t* B_scale,
                                 uint16_t* C, int M, int N, int K, void* hip_stream, int variant);

/*
 * The same gate+up GEMM and SwiGLU, with the MXFP4 quantiser of the next GEMM's activations fused behind it:
 * the fp32 result is rounded to bf16 and quantised per 32 consecutive n exactly as ave_fp4_quantize_mxfp4_bf16
 * would quantise the bf16 output of ave_fp4_gemm_mxfp4_swiglu, without that output ever being written: codes and scales
 * are bit-identical up to 32 rows and above 64; from 33 to 64 rows each call picks its own kernel, and a sum may round the other
 * way.  Q [M, N/2] packed E2M1 (16-byte aligned), Q_scale [M, N/32] E8M0; N % 32 == 0.
 * Up to 32 rows run on the weight-streaming kernel (K a multiple of 32 from 512 up, 16-byte aligned operands), everything
 * else on the LDS-staged kernels: K % 512 == 0 with 16-byte-aligned scale tensors, or any other multiple of
 * 32 from 512 up with 16-byte-aligned A and B; else AVE_FP4_EINVAL (use the two calls then).  No counterpart in the reference, whose kernel ends at the bf16 store
 * (amdgpu_gemm.py:293-329).
 */
int ave_fp4_gemm_mxfp4_swiglu_quant(const uint8_t* A, const uint8_t* A_scale, const uint8_t* B, const uint8_t* B_scale,
                                    uint8_t* Q, uint8_t* Q_scale, int M, int N, int K, void* hip_stream);

/*
 * Both fused forms with a caller-provided workspace (the contract of ave_fp4_gemm_mxfp4_ws): where few weight rows leave compute
 * units idle, K is cut into slices whose fp32 sums of gate and up values meet in a second launch, which applies the
 * activation and, in the quantising form, the quantiser.  Up to 32 rows the quantising form without row padding may also run as two
 * launches, the bf16 form into the workspace and the quantiser.  ave_fp4_gemm_mxfp4_swiglu_workspace_bytes gives the size for
 * either form (quant = 0 or 1), 0 where none is used.  Quantising the result of the one form is what the other gives, bit for bit, up to
 * 32 rows and above 64, both called with their workspace or both without.
 */
size_t ave_fp4_gemm_mxfp4_swiglu_workspace_bytes(int M, int N, int K, int quant);
int ave_fp4_gemm_mxfp4_swiglu_ws(const uint8_t* A, const uint8_t* A_scale, const uint8_t* B, const uint8_t* B_scale,
                                 uint16_t* C, int M, int N, int K, void* workspace, size_t workspace_bytes, void* hip_stream);
int ave_fp4_gemm_mxfp4_swiglu_quant_ws(const uint8_t* A, const uint8_t* A_scale, const uint8_t* B, const uint8_t* B_scale,
                                       uint8_t* Q, uint8_t* Q_scale, int M, int N, int N_padded, int K, void* workspace,
                                       size_t workspace_bytes, void* hip_stream);

/*
 * NVFP4: A_scale [M, K/16] and B_scale [N, K/16] are E4M3 bytes (one per 16
 * consecutive k); A_global / B_global point to ONE fp32 each in device memory
 * (per-tensor scale).  C = (A_global * B_global) * sum_k (a*sa)(b*sb).
 * K must be a positive multiple of 16.  Same reference counterpart as above.
 */
int ave_fp4_gemm_nvfp4(const uint8_t* A, const uint8_t* A_scale, const float* A_global, const uint8_t* B,
                       const uint8_t* B_scale, const float* B_global, uint16_t* C, int M, int N, int K,
                       void* hip_stream);
int ave_fp4_gemm_nvfp4_ex(const uint8_t* A, const uint8_t* A_scale, const float* A_global, const uint8_t* B,
                          const uint8_t* B_scale, const float* B_global, uint16_t* C, int M, int N, int K,
                          void* hip_stream, int variant);
/*
 * The NVFP4 GEMM with a caller-provided device workspace, the counterpart of ave_fp4_gemm_mxfp4_ws: where the output
 * tiles number at most half the compute units and a model of the times says that it pays, K is cut into slices that run
 * on different compute units (128 x 4096 x 14336: 25 us instead of 59).  Same contract as the MXFP4 form:
 * ave_fp4_gemm_nvfp4_workspace_bytes gives the size (0: no split), a smaller or null workspace makes the call
 * ave_fp4_gemm_nvfp4, the result is deterministic and within the GEMM's tolerance.
 */
size_t ave_fp4_gemm_nvfp4_workspace_bytes(int M, int N, int K);
int ave_fp4_gemm_nvfp4_ws(const uint8_t* A, const uint8_t* A_scale, const float* A_global, const uint8_t* B,
                          const uint8_t* B_scale, const float* B_global, uint16_t* C, int M, int N, int K, void* workspace,
                          size_t workspace_bytes, void* hip_stream);

/*
 * Grouped (MoE) MXFP4: rows row_offsets[e] .. row_offsets[e+1]-1 of A belong to
 * expert e and are multiplied by B[e] ([E, N, K/2], scales [E, N, K/32]).
 * row_offsets is a DEVICE array of E+1 non-decreasing int32 with
 * row_offsets[0] == 0 and row_offsets[E] == total_M; it is read by the kernel,
 * never by the host, so the call stays asynchronous.  One launch covers all
 * experts.  The reference has no grouped GEMM; the calling convention follows
 * amdgpu_gemm.py:458-494.
 */
int ave_fp4_grouped_gemm_mxfp4(const uint8_t* A, const uint8_t* A_scale, const uint8_t* B, const uint8_t* B_scale,
                               const int32_t* row_offsets, uint16_t* C, int total_M, int E, int N, int K,
                               void* hip_stream);
int ave_fp4_grouped_gemm_mxfp4_ex(const uint8_t* A, const uint8_t* A_scale, const uint8_t* B,
                                  const uint8_t* B_scale, const int32_t* row_offsets, uint16_t* C, int total_M,
                                  int E, int N, int K, void* hip_stream, int variant);

/*
 * Grouped gate+up GEMM with SwiGLU (and, in the _quant form, the MXFP4 quantiser of the result) for an MoE expert
 * layer in one launch: rows row_offsets[e] .. row_offsets[e+1]-1 of A use expert e's weights B[e], which hold the N
 * gate rows followed by the N up rows (B [E, 2N, K/2], B_scale [E, 2N, K/32]); C is [total_M, N] bf16, or
 * Q [total_M, N/2] + Q_scale [total_M, N/32] with N % 32 == 0.  Every expert's rows equal what
 * ave_fp4_gemm_mxfp4_swiglu (ave_fp4_gemm_mxfp4_swiglu_quant) gives for that expert alone, bit for bit where that call adds up K
 * in the same order: not where it cuts K into slices (its _ws form), nor up to 64 rows where it runs on the weight-streaming kernel.  K % 512 == 0 with 16-byte-aligned scale tensors, or another multiple of 32 from 512 up with
 * 16-byte-aligned A and B, takes the LDS-staged kernel; other K the shape-agnostic one (the _quant form then returns
 * AVE_FP4_EINVAL).  No counterpart in the reference.
 */
int ave_fp4_grouped_gemm_mxfp4_swiglu(const uint8_t* A, const uint8_t* A_scale, const uint8_t* B,
                                      const uint8_t* B_scale, const int32_t* row_offsets, uint16_t* C, int total_M,
                                      int E, int N, int K, void* hip_stream);
int ave_fp4_grouped_gemm_mxfp4_swiglu_quant(const uint8_t* A, const uint8_t* A_scale, const uint8_t* B,
                                            const uint8_t* B_scale, const int32_t* row_offsets, uint8_t* Q,
                                            uint8_t* Q_scale, int total_M, int E, int N, int K, void* hip_stream);

/*
 * MXFP4 quantiser: x [rows, K] row-major fp32 (ave_fp4_quantize_mxfp4_f32) or bf16 bit patterns
 * (..._bf16) -> packed [rows, K/2] E2M1 codes and scales [rows, K/32] E8M0 bytes, in the layout the
 * GEMM entry points take.  Per 32 consecutive k: scale 2^(floor(log2(amax)) - 2) (exponent clamped to
 * [-127, 127]; an all-zero block gets byte 127), elements divided by it and rounded to nearest-even
 * onto the E2M1 grid, saturating.  K % 32 == 0, x 16-byte aligned, packed 4-byte aligned.  Inputs
 * must be finite.  No counterpart in the reference (its benchmark feeds bf16 tensors directly,
 * benchmark/gemm/bench_amdgpu_gemm.py:27-29); this is the producer of the GEMM's operands.
 */
int ave_fp4_quantize_mxfp4_f32(const float* x, uint8_t* packed, uint8_t* scales, int rows, int K, void* hip_stream);
int ave_fp4_quantize_mxfp4_bf16(const uint16_t* x, uint8_t* packed, uint8_t* scales, int rows, int K,
                                void* hip_stream);

/*
 * Operands padded along K.  The LDS-staged kernels move whole 128-byte cache lines and whole 512-element units of K:
 * a K whose packed rows (K/2 bytes) are no multiple of 128 bytes costs their main loop about a quarter more per stage
 * (every 128-byte piece of a row then lies in two cache lines), and K % 512 != 0 adds a tail.  Operands whose rows are
 * padded with ZERO BLOCKS (zero codes, any finite scale byte) up to a multiple of 512 give the same sums -- a zero
 * code contributes exactly +0 whatever its scale -- at the speed of the padded length (measured: 8192 x 2880 x 2880
 * 66.7 us as it is, 57.5 us padded to 3072; 8192 x 14336 x 4128 305 us, 264 us padded to 4608).  Weights are padded once,
 * offline; these entry points produce padded activations without a copy:
 *   ave_fp4_quantize_mxfp4_{f32,bf16}_padded: x [rows, K] -> packed [rows, K_padded/2], scales [rows, K_padded/32];
 *     columns K .. K_padded-1 are written as zero codes under the scale byte 127.  K_padded >= K, both multiples of 32;
 *     K_padded == K is the plain quantiser.
 *   ave_fp4_gemm_mxfp4_swiglu_quant_padded / ave_fp4_grouped_gemm_mxfp4_swiglu_quant_padded (declared here, described
 *     with their unpadded forms above): Q [M, N_padded/2], Q_scale [M, N_padded/32]; columns N .. N_padded-1 of both are
 *     NOT written -- fill the two buffers with zero bytes once (code 0 under scale byte 0 = 2^-127 is a zero block).
 * The consumer is then called with K = K_padded (N_padded).  No counterpart in the reference, which takes K % 64 == 0
 * only (amdgpu_gemm.py:475-476).
 */
int ave_fp4_quantize_mxfp4_f32_padded(const float* x, uint8_t* packed, uint8_t* scales, int rows, int K, int K_padded,
                                      void* hip_stream);
int ave_fp4_quantize_mxfp4_bf16_padded(const uint16_t* x, uint8_t* packed, uint8_t* scales, int rows, int K, int K_padded,
                                       void* hip_stream);
int ave_fp4_gemm_mxfp4_swiglu_quant_padded(const uint8_t* A, const uint8_t* A_scale, const uint8_t* B,
                                           const uint8_t* B_scale, uint8_t* Q, uint8_t* Q_scale, int M, int N,
                                           int N_padded, int K, void* hip_stream);
int ave_fp4_grouped_gemm_mxfp4_swiglu_quant_padded(const uint8_t* A, const uint8_t* A_scale, const uint8_t* B,
                                                   const uint8_t* B_scale, const int32_t* row_offsets, uint8_t* Q,
                                                   uint8_t* Q_scale, int total_M, int E, int N, int N_padded, int K,
                                                   void* hip_stream);

/*
 * NVFP4 quantiser for a per-tensor scale the caller supplies: x [rows, K] row-major fp32 or bf16 bit patterns,
 * global_scale a device pointer to one positive fp32 g (calibrated ahead of time; amax / (448 * 6) uses the whole
 * range) -> packed [rows, K/2] E2M1 codes and scales [rows, K/16] E4M3 bytes, in the layout ave_fp4_gemm_nvfp4
 * takes together with the same g.  Per 16 consecutive k, each step one IEEE fp32 operation:
 * u = min((amax / 6) / g, 448); scale byte = E4M3(u), round to nearest even; d = decode(scale byte) * g;
 * codes = E2M1(x / d), round to nearest even, saturating (d == 0: zero codes).  K % 16 == 0, x 16-byte aligned,
 * packed 4-byte aligned.  Inputs must be finite.  No counterpart in the reference (see ave_fp4_quantize_mxfp4_f32).
 */
int ave_fp4_quantize_nvfp4_f32(const float* x, const float* global_scale, uint8_t* packed, uint8_t* scales, int rows,
                               int K, void* hip_stream);
int ave_fp4_quantize_nvfp4_bf16(const uint16_t* x, const float* global_scale, uint8_t* packed, uint8_t* scales, int rows,
                                int K, void* hip_stream);

/*
 * MoE routing in front of the grouped GEMM.  logits [tokens, E] fp32 router scores (finite).  Every
 * token is routed to its two highest-scoring experts (equal scores: the lower expert index ranks
 * first).  The 2*tokens routed rows are ordered by expert, inside an expert by token and then by rank
 * (a stable sort of the row-major [tokens, 2] choice table by expert):
 *   token_of_row [2*tokens] int32   token whose activations routed row i carries,
 *   row_offsets  [E+1]      int32   first routed row of every expert (the grouped GEMM's row_offsets),
 *   row_weight   [2*tokens] fp32    softmax(logits[token])[expert] of routed row i; may be NULL.
 * 2 <= E <= 256, tokens <= 2^29.  No counterpart in the reference, which has no MoE
 * code; it exists so that routing, gather and grouped GEMM can be recorded into one graph.
 */
int ave_fp4_moe_route_top2(const float* logits, int tokens, int E, int32_t* token_of_row, int32_t* row_offsets,
                           float* row_weight, void* hip_stream);

/*
 * The same routing, with one more output: rows_of_token [tokens, 2] int32, the routed row of every token's first
 * and second choice (the inverse of token_of_row; may be null), which ave_fp4_moe_combine_top2 reads.
 */
int ave_fp4_moe_route_top2_ex(const float* logits, int tokens, int E, int32_t* token_of_row, int32_t* row_offsets,
                              float* row_weight, int32_t* rows_of_token, void* hip_stream);

/*
 * The same routing with a caller-provided device workspace (16-byte aligned, no initialisation needed, garbage
 * afterwards): the tokens' choices and the counts of every chunk of tokens (32 and more, by E and the number of tokens) are passed
 * through it from one launch to a second, so that the logits are read once.  ave_fp4_moe_route_top2_workspace_bytes gives
 * its size, 0 where a single workgroup does all the work; with a smaller (or null) workspace the call is
 * ave_fp4_moe_route_top2_ex, every workgroup of which goes through all logits (16384 tokens: 21 us against 8.4 with 8 experts,
 * 280 against 13 with 128).  Same results; calls that may overlap need workspaces of their own.
 */
size_t ave_fp4_moe_route_top2_workspace_bytes(int tokens, int E);
int ave_fp4_moe_route_top2_ws(const float* logits, int tokens, int E, int32_t* token_of_row, int32_t* row_offsets,
                              float* row_weight, int32_t* rows_of_token, void* workspace, size_t workspace_bytes,
                              void* hip_stream);

/*
 * The step behind the expert GEMMs: out[t, :] = w0 * rows[r0, :] + w1 * rows[r1, :] with (r0, r1) =
 * rows_of_token[t], w = row_weight of those rows, divided by w0 + w1 when `renormalize` is non-zero.  rows
 * [2*tokens, H] bf16 (the down projection's output in routed order), out [tokens, H] bf16, both 16-byte aligned;
 * H % 8 == 0.  The two products and the sum are single IEEE fp32 operations, then one rounding to bf16; a row
 * index outside [0, 2*tokens) contributes zeros.  No counterpart in the reference.
 */
int ave_fp4_moe_combine_top2(const uint16_t* rows, const int32_t* rows_of_token, const float* row_weight, int tokens,
                             int H, int renormalize, uint16_t* out, void* hip_stream);

/*
 * Row gather of an MXFP4 operand: out[i] = A[index[i]], out_scale[i] = A_scale[index[i]] for
 * i < rows; A [src_rows, K/2], A_scale [src_rows, K/32], index [rows] int32.  An index outside
 * [0, src_rows) produces a row of zero bytes.  K % 32 == 0; A and out 16-byte aligned.  No
 * counterpart in the reference; it builds the grouped GEMM's A operand from token_of_row.
 */
int ave_fp4_gather_rows_mxfp4(const uint8_t* A, const uint8_t* A_scale, const int32_t* index, int rows, int src_rows,
                              int K, uint8_t* out, uint8_t* out_scale, void* hip_stream);

/*
 * Scale-layout adapters.  The GEMM entry points take block scales row-major, [rows, cols] bytes
 * (cols = K/32 for MXFP4, K/16 for NVFP4).  Other FP4 stacks keep them "blocked": padded to
 * multiples of 128 rows and 4 columns, cut into 128 x 4 tiles of 512 bytes stored in row-major tile
 * order, scale (r, c) of a tile at byte (r % 32) * 16 + (r / 32) * 4 + c.  The blocked tensor holds
 * ceil(rows/128)*128 * ceil(cols/4)*4 bytes and must be 4-byte aligned; to_blocked writes its
 * padding as zero, from_blocked ignores it.  No counterpart in the reference, whose kernel takes
 * no scales.
 */
int ave_fp4_scales_to_blocked(const uint8_t* scales, int rows, int cols, uint8_t* blocked, void* hip_stream);
int ave_fp4_scales_from_blocked(const uint8_t* blocked, int rows, int cols, uint8_t* scales, void* hip_stream);

/*
 * The MXFP4 GEMM on scale tensors that are ALREADY in the blocked layout above -- A_scale_blocked for [M, K/32],
 * B_scale_blocked for [N, K/32], each ceil(rows/128)*128 * K/32 bytes, 16-byte aligned -- read by the kernels as they
 * are: no conversion launch, no workspace.  K % 512 == 0 (then K/32 is a multiple of 4 and the tensors have no column
 * padding).  Up to 64 rows run on the weight-streaming kernel, which gathers a K step's four scale bytes per row as one
 * dword of a 512-byte tile; more rows on the 256 x 256 LDS-staged kernel, which copies the four column tiles of a pair of
 * K stages as whole kilobytes.  Same arithmetic in the same order as ave_fp4_gemm_mxfp4_ex with AVE_FP4_DECODE /
 * AVE_FP4_TILE on row-major scales: bit-identical results.  Other K: AVE_FP4_EINVAL (convert with
 * ave_fp4_scales_from_blocked).  The reference's entry takes its operands as its caller has them
 * (amdgpu_gemm.py:458-462); this is that for callers whose quantiser emits blocked scales.
 */
int ave_fp4_gemm_mxfp4_blocked_scales(const uint8_t* A, const uint8_t* A_scale_blocked, const uint8_t* B,
                                      const uint8_t* B_scale_blocked, uint16_t* C, int M, int N, int K, void* hip_stream);

/*
 * ---- Between the qkv projection and the output projection: a paged key/value cache held in MXFP4 ----
 *
 * No counterpart in the reference, whose only library kernel is a GEMM; with these a decoder layer's attention runs on the
 * library as its linear layers do.
 *
 * The cache of one layer is four device tensors: codes [pages, kv_heads, page_size, head_dim/2] (packed E2M1, low nibble =
 * even channel) and scales [pages, kv_heads, page_size, head_dim/32] (E8M0) of the keys, and the same of the values.  A
 * page may be followed by other data (the page strides, in bytes); inside a page all is contiguous.  head_dim is 64, 128
 * or 256, page_size a power of two from 16 to 4096.  Codes 16-byte aligned with page strides that are multiples of 16,
 * scales 4-byte aligned with multiples of 4.  A token's place is its slot: page * page_size + offset.
 */
typedef struct ave_fp4_kv_cache {
  uint8_t *k, *k_scale, *v, *v_scale;
  int64_t k_page_stride, k_scale_page_stride, v_page_stride, v_scale_page_stride; /* bytes */
  int32_t pages, kv_heads, page_size, head_dim;
} ave_fp4_kv_cache;

/* Heads of a batch of tokens, [tokens, heads, head_dim] with consecutive channels; strides in elements, any alignment. */
typedef struct ave_fp4_heads {
  void* data; /* bf16, or fp32 where is_f32 (inputs only) */
  int64_t token_stride, head_stride;
  int32_t heads, is_f32;
} ave_fp4_heads;

/*
 * What happens to query and key heads before they are stored.  Norm (weights set): n = (x * r) * w with
 * r = 1 / sqrt(sum(x^2) / head_dim + eps).  Rotation (cos set) of the first rotary_dim channels (a multiple of 16):
 * a' = a cos - b sin, b' = b cos + a sin for the pairs (i, i + rotary_dim/2), with `neighbours` (2i, 2i+1), cos and sin
 * [table_rows, rotary_dim/2] fp32 at row positions[token]; a position outside the table gives NaN.  All of it in fp32,
 * every product and sum rounded by itself and the squares added up neighbours first, so that the codes of normed and rotated
 * keys have the same bits wherever they are computed; one rounding at the end (to bf16, or by the quantiser).
 */
typedef struct ave_fp4_norm_rope {
  const void *q_weight, *k_weight; /* [head_dim], either may be null; bf16, or fp32 where weight_is_f32 */
  const float *cos, *sin;          /* null: no rotation */
  const int32_t* positions;        /* [tokens] */
  int32_t table_rows, rotary_dim, neighbours, weight_is_f32;
  float eps;
} ave_fp4_norm_rope;

/* Norm and rotation of query heads, key heads or both (a null pointer: none), bf16 out; an output may be its input. */
int ave_fp4_qk_norm_rope(const ave_fp4_heads* q, const ave_fp4_heads* k, int tokens, int head_dim, const ave_fp4_norm_rope* how,
                         const ave_fp4_heads* q_out, const ave_fp4_heads* k_out, void* hip_stream);

/*
 * Keys (normed and rotated as `how` says; null: as they are) and values of a batch of tokens into the cache at slots
 * [tokens]: the quantiser of ave_fp4_quantize_mxfp4_* per 32 channels, from fp32.  A slot outside the cache stores nothing (padding);
 * what a slot inside it holds that two tokens of a call share is undefined -- tokens are written by workgroups of their own, codes and scales apart,
 * so that it may be neither token -- and other slots are as they should be.  With q the same launch norms and rotates the queries into q_out (bf16).
 */
int ave_fp4_append_kv_mxfp4(const ave_fp4_heads* k, const ave_fp4_heads* v, int tokens, const int32_t* slots, const ave_fp4_norm_rope* how,
                            const ave_fp4_kv_cache* cache, const ave_fp4_heads* q, const ave_fp4_heads* q_out, void* hip_stream);

/* Cached tokens back as bf16 [tokens, kv_heads, head_dim] (exact: E2M1 times a power of two; a scale byte 0xFF gives NaN); a slot
 * outside the cache gives zeros. */
int ave_fp4_gather_kv_mxfp4(const ave_fp4_kv_cache* cache, const int32_t* slots, int tokens, uint16_t* k, uint16_t* v, void* hip_stream);

/*
 * Attention of the new tokens of `batch` sequences over their cached keys and values (the new tokens' own among them).
 * Sequence b holds seq_lens[b] tokens, token j in page page_table[b * page_table_stride + j / page_size]; its new tokens are rows
 * cu_q[b] .. cu_q[b+1]-1 of q (cu_q null: one each, tokens == batch) and its last ones: row i of n stands at position
 * p = seq_lens[b] - n + i.  It sees key j if j <= p (`causal`) and j > p - window (window > 0; causal only).  Query head h
 * reads key head h / (heads / kv_heads).
 *   out = sum_j exp(s_j) v_j / (sum_j exp(s_j) + exp(sink_h)),  s_j = scale * q . k_j      (sinks null: without the last term)
 *   lse = log of the denominator (optional; natural logarithm, the sink included; -inf where it is zero)
 * A row that sees no key gives zeros.  Scores, softmax and sums in fp32; queries enter the products with 19 bits and more below
 * their row's largest one, probabilities as bf16.  A NaN or infinity in a query, or a NaN scale (0xFF) of a key it sees, gives NaN; so does,
 * in its 32 channels, a scale of a value it sees from 253 on (beyond what bf16 holds; the quantiser writes 252 at most).
 * Rows of q behind cu_q[batch] are left alone.  Device data is never trusted with addresses: lengths are cut to the page
 * table's width, rows to q's, pages outside the cache are read as its nearest page.  Lengths, offsets and tables are read more than once: they must
 * not change before the call has run (if they do, results are anybody's, and no access leaves q, out, table or cache).
 * Limits: tokens * heads below 2^31 - 2^14, a table of at most 2^31 - 256 tokens, at most 1024 query heads on a key head.  In fp32 two scores beyond
 * 2^30 no longer differ by less than 64, and a row's numerator, which is summed before it is divided and at up to 2^8 times the probabilities, may
 * overflow for values beyond 2^100.
 * max_q: a bound on the new tokens of a sequence, by which the kernel is chosen (a wrong one costs time only).
 * The workspace (16-byte aligned, no initialisation, garbage afterwards; calls that may overlap need their own) takes the
 * partial results of sequences that several workgroups share; results do not depend on what it held.
 */
typedef struct ave_fp4_attention {
  const uint16_t* q;
  int64_t q_token_stride, q_head_stride; /* elements; consecutive channels, any alignment */
  uint16_t* out;                         /* [tokens, heads, head_dim] contiguous, 4-byte aligned */
  float* lse;                            /* [tokens, heads] or null */
  const int32_t* page_table;
  int64_t page_table_stride;             /* entries */
  const int32_t *seq_lens, *cu_q;
  const float* sinks;                    /* [heads] or null */
  int32_t tokens, batch, heads, table_pages, max_q, window, causal;
  float scale;
} ave_fp4_attention;
size_t ave_fp4_attention_mxfp4_workspace_bytes(const ave_fp4_attention* a, const ave_fp4_kv_cache* cache);
int ave_fp4_attention_mxfp4(const ave_fp4_attention* a, const ave_fp4_kv_cache* cache, void* workspace, size_t workspace_bytes,
                            void* hip_stream);

/*
 * ---- Checking a tree of drafted tokens ----
 *
 * A draft proposes several tokens behind the last decided one, possibly with alternatives: a tree.  Its nodes are appended to the cache as the
 * last tokens of their sequence (nodes cu_q[b] .. cu_q[b+1]-1 of all nodes, a parent before its children, node 0 the decided token), the
 * target model runs on all of them at once, and the nodes that it would have drawn itself are kept.  No counterpart in the reference.
 *
 * From the nodes' parents ([tokens], an index within the sequence; one that is not in [0, the node's own index) means none): `seen`, `words` 64-bit
 * words a node, bit j % 64 of word j / 64 is set where node j of the sequence is the node itself or one that it descends from (nodes from 64 * words on
 * have no bit), and the position of each node, seq_lens[b] less the number of nodes plus the number of nodes above it.  Either output may be null.
 * Rows behind cu_q[batch] are left alone.  No output may overlap an input.
 */
int ave_fp4_draft_tree(const int32_t* parents, const int32_t* cu_q, const int32_t* seq_lens, int tokens, int batch, uint64_t* seen, int words,
                       int32_t* positions, void* hip_stream);

/* What the new tokens of a sequence see of each other: bits as ave_fp4_draft_tree makes them, or any others. */
typedef struct ave_fp4_tree {
  const uint64_t* seen; /* [tokens, words], 8-byte aligned */
  int64_t stride;       /* words between rows; 0: one row for all */
  int32_t words;        /* new tokens from 64 * words on are seen by nobody */
} ave_fp4_tree;

/*
 * ave_fp4_attention_mxfp4 where the new tokens are not a chain: with n of them row i sees the keys before them, j < seq_lens[b] - n, and of the new ones
 * those whose bit is set in its row of `seen` (its own, too).  window > 0: the last `window` of what it sees -- of the keys before, those
 * from seq_lens[b] - n + (bits set) - window on; the new tokens are seen as their bits say.  `causal` is ignored.  Everything else, workspace
 * included, is as there.  With the bits of a chain (node i sees 0 .. i) the result is that of the causal call with the same window, up to the order
 * of sums.
 */
size_t ave_fp4_tree_attention_mxfp4_workspace_bytes(const ave_fp4_attention* a, const ave_fp4_tree* tree, const ave_fp4_kv_cache* cache);
int ave_fp4_tree_attention_mxfp4(const ave_fp4_attention* a, const ave_fp4_tree* tree, const ave_fp4_kv_cache* cache, void* workspace,
                                 size_t workspace_bytes, void* hip_stream);

/*
 * Which nodes of a draft are kept, so that the tokens are distributed as if the target model had drawn them one by one (temperature > 0), or are the ones
 * that it would choose (temperature 0, or not above it).  From node 0 on: p is the softmax of the node's logits over the temperature; its children c, in
 * the order of their indices, are tried one after the other until one is accepted; from that one on the same again.
 *   draft_probs null (children are given, not drawn): r is p without the tokens of rejected siblings, over its sum; c is accepted if uniform[c] < r(token)
 *   draft_probs (children of a node were drawn from its row q): r starts as p and becomes max(r - q, 0) over its sum with each rejection; c is accepted
 *   if uniform[c] q(token) < r(token)
 *   temperature 0: the child whose token has the largest logit (the lowest of equal ones) is accepted
 * Where no child is accepted, the next token is drawn from r: the first index where the running sum of r is above uniform[node 0] times the whole (temperature 0:
 * the token of the largest logit).  If rejections leave nothing of r, it is p (draft_probs: c is then rejected; tokens: r(token) is 0).
 * accepted[b]: nodes kept, node 0 among them (0 for a sequence without nodes); path[cu_q[b] + i], i < accepted[b]: their indices, rising; emitted: as many
 * tokens, those of the kept nodes from the second on, then the drawn one.  Both are -1 for the other nodes of the sequence.
 * Choices are those of softmax, sums and products in 64 bits (a choice lies between sums of very many probabilities), exponentials to 2^-42: what rejections leave of
 * draft_probs with a probability near that is not told from rounding.  Without draft_probs a node's acceptance is decided by a row sum in fp32 where that is exact enough
 * to say, else in 64, and a random number of 1 accepts none.  A probability below 2^-1020 of the row's largest is none: a logit 708 temperatures and more below the
 * largest one hides its token as -inf does.  A NaN among the logits counts as -inf, +inf as the largest finite number; a row without any number accepts no child and
 * draws -1.  uniform is taken into [0, 1], NaN as 0 (1 draws the last index that r has); a token that is no index of the vocabulary is never accepted; NaN and negative
 * numbers in draft_probs count as 0, as they are otherwise (no sum of 1 is asked for).
 * Rows behind cu_q[batch] are not written, and what they hold does not matter.  No output may overlap another output or an input.  Offsets are cut to the
 * rows; nothing in device memory leads out of the arrays.
 * The workspace (16-byte aligned, no initialisation) belongs to one call at a time.  Equal inputs give equal outputs.
 */
typedef struct ave_fp4_draft {
  const void* logits;        /* [rows, vocab] bf16, or fp32 where logits_f32: the target's, row t behind node t */
  int64_t logits_stride;     /* elements between rows */
  const int32_t *tokens, *parents; /* [rows] */
  const int32_t* cu_q;       /* [batch + 1] */
  const float* uniform;      /* [rows] */
  const float* temperature;  /* [batch] or null (1) */
  const float* draft_probs;  /* [rows, vocab] or null; rows of nodes without children are not read */
  int64_t draft_probs_stride;
  int32_t *accepted, *path, *emitted; /* [batch], [rows], [rows] */
  int32_t rows, batch, vocab, logits_f32;
} ave_fp4_draft;
size_t ave_fp4_verify_draft_workspace_bytes(const ave_fp4_draft* draft);
int ave_fp4_verify_draft(const ave_fp4_draft* draft, void* workspace, size_t workspace_bytes, void* hip_stream);

/*
 * Of the last n = cu_q[b+1] - cu_q[b] tokens of each sequence, those at path[cu_q[b] + i], i < accepted[b] (rising, each at least i), are moved together in the
 * caches of `layers` layers, codes and scales as they are: token seq_lens[b] - n + path[cu_q[b] + i] to place seq_lens[b] - n + i.  kept_lens[b] (null: not
 * asked for; must not overlap the inputs) = seq_lens[b] - n + accepted[b], the length that is left.  With the outputs of ave_fp4_verify_draft a checked
 * draft becomes part of its sequence; with n = seq_lens[b] tokens that a policy gives up leave a cache.
 * All caches have one shape (pages, kv_heads, page_size, head_dim) and the page table in common; pages that hold moved tokens belong to one sequence
 * only.  What stands behind the kept tokens is left as it was.  An index outside [0, n), a token outside the page table and a page outside the cache
 * move nothing; indices that do not rise leave a mix of the tokens that they name.
 * max_q: a bound on n, by which the kernel is chosen (a wrong one costs time only).
 */
typedef struct ave_fp4_keep {
  const int32_t* page_table;
  int64_t page_table_stride;
  const int32_t *seq_lens, *cu_q, *path, *accepted; /* [batch], [batch + 1], [tokens], [batch] */
  int32_t* kept_lens;
  int32_t tokens, batch, table_pages, max_q;
} ave_fp4_keep;
int ave_fp4_keep_kv_mxfp4(const ave_fp4_kv_cache* caches, int layers, const ave_fp4_keep* keep, void* hip_stream);

/* Message of the last failure on the calling thread ("" if none). */
const char* ave_fp4_last_error(void);

/* Library ABI version (bumped when a signature changes). */
int ave_fp4_abi_version(void);

#ifdef __cplusplus
}
#endif
#endif /* AVE_FP4_H_ */
