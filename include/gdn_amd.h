/*
 * gdn_amd.h — C ABI of the MI355X (gfx950) Gated DeltaNet hot-path library
 * (libgdn_amd.so).
 *
 * Plain pointers and sizes only.  All data pointers are DEVICE pointers unless
 * a parameter says otherwise; every call is asynchronous on `stream` (a
 * hipStream_t passed as void*, NULL = the null stream) and returns a status
 * code.  On failure nothing is launched and gdn_last_error() returns a message
 * for the calling thread.  bf16 tensors are passed as their 16-bit patterns.
 *
 * Reference interfaces replaced (paths into diacccc/GDN_18646):
 *   gdn_decode_hip            <- extern "C" gdn_decode_cuda, kernels/decode.cu:131-162
 *                                (and gdn_decode_forward, kernels/decode.cu:172-214)
 *   gdn_prefill_hip           <- gdn_prefill, kernels/prefill_chunked.cu:422-504
 *   gdn_prefill_noalloc_hip   <- no reference counterpart (gdn_prefill_hip with a static
 *                                scratch buffer, for callers that cannot allocate)
 *   gdn_prefill_varlen_hip    <- no reference counterpart (packed cu_seqlens prefill);
 *                                semantics = gdn_prefill per sequence
 *   gdn_rmsnorm_hip           <- rmsnorm_forward_impl / launch_rmsnorm,
 *                                kernels/rmsnorm.cu:112-131,251-276
 *   gdn_proj_conv_silu_hip    <- fused_proj_conv_silu, kernels/fused_proj_conv_silu.cu:298-355
 *   gdn_in_proj_hip           <- GDNLayerCustom.forward's projections, gdn_layer.py:240-252
 *   gdn_in_proj_varlen_hip,   <- no reference counterpart (packed sequences through the layer;
 *   gdn_prefill_varlen_tm_hip    the reference layer has no cu_seqlens path, gdn_layer.py:222-263)
 *   gdn_packed_history_hip,   <- no reference counterpart (packed sequences)
 *   gdn_store_offsets_hip
 *   gdn_decode_conv_step_hip  <- _decode_conv_step / _decode_fused_proj_step, gdn_layer.py:43-69
 *   gdn_decode_in_proj_hip    <- GDNLayerCustom.decode's RMSNorm, projections and conv step,
 *                                gdn_layer.py:280-299 (with 43-69)
 *   gdn_decode_out_proj_hip   <- GDNLayerCustom.decode's output projection, gdn_layer.py:309
 *   gdn_out_proj_hip, _fits   <- GDNLayerCustom.forward's output projection, gdn_layer.py:263
 *   gdn_layer_decode_step_hip <- GDNLayerCustom.decode as a whole, gdn_layer.py:265-316
 *   gdn_block_norm_hip, _bwd  <- no reference counterpart (the reference layer has no residual,
 *                                gate or norm after the block, and no backward pass)
 *   gdn_fp8_quantize_hip,     <- no reference counterpart (8-bit projections)
 *   gdn_fp8_matmul_hip
 *   gdn_fp4_quantize_hip,     <- no reference counterpart (4-bit weights)
 *   gdn_fp4_fp8_quantize_hip,
 *   gdn_fp4_dequantize_hip,
 *   gdn_fp4_matmul_hip
 *   gdn_grad_norm_hip,        <- no reference counterpart (the reference does not train)
 *   gdn_clip_grad_norm_hip
 */
#ifndef GDN_AMD_H
#define GDN_AMD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef uint16_t gdn_bf16_t; /* bfloat16 bit pattern */

enum {
    GDN_OK = 0,
    GDN_ERR_INVALID_ARGUMENT = 1, /* null pointer, bad size, misaligned buffer */
    GDN_ERR_UNSUPPORTED = 2,      /* shape outside what the kernels are built for */
    GDN_ERR_WORKSPACE = 3,        /* workspace missing or smaller than required */
    GDN_ERR_HIP = 4               /* a HIP runtime call or launch failed */
};

/* Library version, e.g. 1 for this interface revision. */
int gdn_abi_version(void);

/* Human-readable text for a status code, and the last error of this thread. */
const char* gdn_status_string(int status);
const char* gdn_last_error(void);

/*
 * Decode: one token per sequence, state updated as
 *   S <- g S ; r = k^T S ; S <- S + k (beta (v - r))^T ; o = scale q^T S
 * with g = exp(-exp(A_log[h]) softplus(a + dt_bias[h])), beta = sigmoid(b).
 *   q, k     [B, H, dk]   bf16        v        [B, H, dv] bf16
 *   a, b     [B, H]       bf16        A_log, dt_bias [H] fp32
 *   S_in     [B, H, dk, dv] fp32      o        [B, H, dv] fp32
 *   S_out    [B, H, dk, dv] fp32 — may be the same buffer as S_in (in place)
 * Supported: dk == 128, dv % 32 == 0, 32 <= dv <= 1024.  Buffers 16-byte aligned.
 * Replaces gdn_decode_cuda (kernels/decode.cu:131-162), which took no stream,
 * returned nothing and silently did nothing for an unsupported dv.
 */
int gdn_decode_hip(const gdn_bf16_t* q, const gdn_bf16_t* k, const gdn_bf16_t* v,
                   const gdn_bf16_t* a, const gdn_bf16_t* b,
                   const float* A_log, const float* dt_bias,
                   const float* S_in, float scale,
                   float* o, float* S_out,
                   int B, int H, int dk, int dv, void* stream);

/*
 * Chunked prefill (chunk size 64) of B equal-length sequences.
 *   q, k [B, H, T, dk] bf16; v [B, H, T, dv] bf16; a, b_logits [B, H, T] bf16
 *   A_log [H] fp32; dt_bias scalar; mask [B, T] fp32 or NULL (all ones)
 *   state_in [B, H, dk, dv] fp32 or NULL (zero state)
 *   out [B, H, T, dv] bf16; state_out [B, H, dk, dv] fp32
 * scale == 0 means dk^-0.5.  Any T >= 1.  Supported: dk == 128, dv % 16 == 0,
 * 16 <= dv <= 512.  Masked tokens decay the state but write nothing, and their
 * outputs are zero (reference/prefill_ref.py:79-80,130).
 * workspace: device buffer of at least gdn_prefill_workspace_bytes(B, H, T,
 * dk, dv) bytes, 256-byte aligned; it holds per-chunk intermediates.
 * Replaces gdn_prefill (kernels/prefill_chunked.cu:422-504), which required
 * H == 16, dv == 256 and T % 64 == 0 and allocated its outputs itself.
 */
size_t gdn_prefill_workspace_bytes(int B, int H, int T, int dk, int dv);

int gdn_prefill_hip(const gdn_bf16_t* q, const gdn_bf16_t* k, const gdn_bf16_t* v,
                    const float* A_log, const gdn_bf16_t* a, float dt_bias,
                    const gdn_bf16_t* b_logits, const float* mask,
                    const float* state_in, float scale,
                    gdn_bf16_t* out, float* state_out,
                    int B, int H, int T, int dk, int dv,
                    void* workspace, size_t workspace_bytes, void* stream);

/*
 * gdn_prefill_hip with the output written token-major: out [B, T, H, dv]
 * (the layout the output projection consumes, so the caller's
 * transpose(1, 2).contiguous() copy disappears); all else identical.
 * Replaces the transposes around the prefill call in the reference layer
 * (gdn_layer.py:256-263), which has no kernel-level counterpart.
 */
int gdn_prefill_tm_hip(const gdn_bf16_t* q, const gdn_bf16_t* k, const gdn_bf16_t* v,
                       const float* A_log, const gdn_bf16_t* a, float dt_bias,
                       const gdn_bf16_t* b_logits, const float* mask,
                       const float* state_in, float scale,
                       gdn_bf16_t* out, float* state_out,
                       int B, int H, int T, int dk, int dv,
                       void* workspace, size_t workspace_bytes, void* stream);

/*
 * gdn_prefill_hip without a workspace argument, for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc).  No reference counterpart.
 * The per-chunk intermediates go to a static device buffer of
 * GDN_PREFILL_NOALLOC_MAX_BYTES that the library holds per GPU until the
 * process ends; the call allocates nothing.  A shape whose
 * gdn_prefill_workspace_bytes() exceeds that size is refused with
 * GDN_ERR_WORKSPACE before any HIP call (e.g. B=1, H=16, T=8192, dk=dv=128
 * needs 40 MiB and B=4, H=16, T=4096 56 MiB, which fit; B=4, H=16, T=8192
 * needs 88 MiB and does not).
 * The buffer used is the current device's, so `stream` (when not null) must
 * belong to the current device (else GDN_ERR_INVALID_ARGUMENT).
 * All calls on one GPU share the buffer: calls that overlap on one GPU (two
 * streams, two threads) race, so serialise them.  Nothing in it needs to
 * start zeroed.  Outputs are bit-identical to gdn_prefill_hip's.
 */
#define GDN_PREFILL_NOALLOC_MAX_BYTES (64u << 20)

int gdn_prefill_noalloc_hip(const gdn_bf16_t* q, const gdn_bf16_t* k, const gdn_bf16_t* v,
                            const float* A_log, const gdn_bf16_t* a, float dt_bias,
                            const gdn_bf16_t* b_logits, const float* mask,
                            const float* state_in, float scale,
                            gdn_bf16_t* out, float* state_out,
                            int B, int H, int T, int dk, int dv, void* stream);

/*
 * The two phases of gdn_prefill_hip, same arguments, for callers that overlap
 * them with other work (and for per-phase timing):
 *   intra — every chunk in parallel: reads q, k, a, b_logits, mask, A_log,
 *           dt_bias, scale; fills `workspace` (out/state pointers unused);
 *   state — chunks in order per (sequence, head): reads the workspace, q, k,
 *           v, state_in; writes out and state_out.
 * gdn_prefill_hip is intra followed by state on the same stream.  No
 * reference counterpart (the reference runs one fused kernel).
 */
int gdn_prefill_intra_hip(const gdn_bf16_t* q, const gdn_bf16_t* k, const gdn_bf16_t* v,
                          const float* A_log, const gdn_bf16_t* a, float dt_bias,
                          const gdn_bf16_t* b_logits, const float* mask,
                          const float* state_in, float scale,
                          gdn_bf16_t* out, float* state_out,
                          int B, int H, int T, int dk, int dv,
                          void* workspace, size_t workspace_bytes, void* stream);

int gdn_prefill_state_hip(const gdn_bf16_t* q, const gdn_bf16_t* k, const gdn_bf16_t* v,
                          const float* A_log, const gdn_bf16_t* a, float dt_bias,
                          const gdn_bf16_t* b_logits, const float* mask,
                          const float* state_in, float scale,
                          gdn_bf16_t* out, float* state_out,
                          int B, int H, int T, int dk, int dv,
                          void* workspace, size_t workspace_bytes, void* stream);

/*
 * Packed variable-length prefill: num_seqs sequences concatenated along T.
 *   q, k [H, T_total, dk]; v [H, T_total, dv]; a, b_logits [H, T_total]
 *   cu_seqlens: DEVICE int32 [num_seqs + 1], non-decreasing, cu[0] = 0,
 *               cu[num_seqs] = T_total
 *   max_seqlen: upper bound on any sequence length (<= 0: T_total is used)
 *   mask [T_total] fp32 or NULL; state_in [num_seqs, H, dk, dv] or NULL
 *   out [H, T_total, dv] bf16; state_out [num_seqs, H, dk, dv] fp32
 * Each sequence is an independent prefill (state does not cross sequences).
 */
size_t gdn_prefill_varlen_workspace_bytes(int num_seqs, int H, int T_total, int dk, int dv);

int gdn_prefill_varlen_hip(const gdn_bf16_t* q, const gdn_bf16_t* k, const gdn_bf16_t* v,
                           const float* A_log, const gdn_bf16_t* a, float dt_bias,
                           const gdn_bf16_t* b_logits, const float* mask,
                           const int32_t* cu_seqlens, int num_seqs, int max_seqlen,
                           const float* state_in, float scale,
                           gdn_bf16_t* out, float* state_out,
                           int H, int T_total, int dk, int dv,
                           void* workspace, size_t workspace_bytes, void* stream);

/*
 * gdn_prefill_varlen_hip with the output written token-major: out
 * [T_total, H, dv] (the layout the output projection consumes); all else
 * identical.  No reference counterpart (the layer's packed-sequence forward).
 */
int gdn_prefill_varlen_tm_hip(const gdn_bf16_t* q, const gdn_bf16_t* k, const gdn_bf16_t* v,
                              const float* A_log, const gdn_bf16_t* a, float dt_bias,
                              const gdn_bf16_t* b_logits, const float* mask,
                              const int32_t* cu_seqlens, int num_seqs, int max_seqlen,
                              const float* state_in, float scale,
                              gdn_bf16_t* out, float* state_out,
                              int H, int T_total, int dk, int dv,
                              void* workspace, size_t workspace_bytes, void* stream);

/*
 * RMSNorm: y[r, :] = bf16(x[r, :] * rsqrt(mean(x[r, :]^2) + eps) * gamma).
 *   x, y [R, D] bf16 (may not alias); gamma [D] bf16.  D % 8 == 0, D <= 16384.
 */
int gdn_rmsnorm_hip(const gdn_bf16_t* x, const gdn_bf16_t* gamma, gdn_bf16_t* y,
                    int R, int D, float eps, void* stream);

/*
 * Projection + causal depthwise conv (taps conv_k) + SiLU, fp32 accumulation:
 *   out[b, t, c] = bf16(SiLU(sum_j conv_w[c, j] * P[b, t - conv_k + 1 + j, c]))
 *   P = x W^T with P[b, t<0, :] = 0.
 *   x [B, T, D] bf16; W [D_out, D] bf16; conv_w [D_out, conv_k] bf16;
 *   out [B, T, D_out] bf16.  D % 64 == 0, D_out % 16 == 0, conv_k in 1..4.
 */
int gdn_proj_conv_silu_hip(const gdn_bf16_t* x, const gdn_bf16_t* W,
                           const gdn_bf16_t* conv_w, gdn_bf16_t* out,
                           int B, int T, int D, int D_out, int conv_k, void* stream);

/*
 * Layer in-projection for a prefill: P = xn [B, T, D] x W^T with
 * W = [W_q; W_k; W_v; W_a; W_b] ([2 H dk + H dv + 2 H, D] bf16), causal
 * depthwise conv (conv_w_qkv [2 H dk + H dv, conv_k]) + SiLU on the q/k/v
 * columns, written head-major: q, k [B, H, T, dk]; v [B, H, T, dv];
 * a, b [B, H, T] (no conv).  Optional conv caches [B, H d, conv_k - 1] bf16
 * of projected tokens (oldest first): *_in (NULL = zeros) precede t = 0,
 * *_out (NULL = not written, must not alias *_in) receive the last conv_k - 1
 * projected tokens.  D % 64 == 0, conv_k in 1..4.
 * Replaces the three fused_proj_conv_silu launches, the a/b GEMMs and the
 * transposes of GDNLayerCustom.forward (gdn_layer.py:240-252).
 */
int gdn_in_proj_hip(const gdn_bf16_t* xn, const gdn_bf16_t* W_qkvab, const gdn_bf16_t* conv_w_qkv,
                    const gdn_bf16_t* cache_q_in, const gdn_bf16_t* cache_k_in, const gdn_bf16_t* cache_v_in,
                    gdn_bf16_t* cache_q_out, gdn_bf16_t* cache_k_out, gdn_bf16_t* cache_v_out,
                    gdn_bf16_t* q, gdn_bf16_t* k, gdn_bf16_t* v, gdn_bf16_t* a, gdn_bf16_t* b,
                    int B, int T, int D, int H, int dk, int dv, int conv_k, void* stream);

/*
 * gdn_in_proj_hip for num_seqs packed sequences: xn [T_total, D];
 * cu_seqlens is a HOST int32 array [num_seqs + 1] (0 = cu[0] <= cu[1] <= ...
 * <= cu[num_seqs] = T_total).  Each sequence's causal conv starts from its
 * own cache (cache_*_in [num_seqs, H d, conv_k - 1], NULL = zeros) and
 * cache_*_out [num_seqs, H d, conv_k - 1] (NULL = not written) receives its
 * last conv_k - 1 projected tokens; outputs are packed head-major:
 * q, k [H, T_total, dk]; v [H, T_total, dv]; a, b [H, T_total], as
 * gdn_prefill_varlen_hip reads them.  One launch per non-empty sequence.
 * No reference counterpart (the layer's packed-sequence forward; the
 * reference layer has no cu_seqlens path, gdn_layer.py:222-263).
 */
int gdn_in_proj_varlen_hip(const gdn_bf16_t* xn, const gdn_bf16_t* W_qkvab, const gdn_bf16_t* conv_w_qkv,
                           const int32_t* cu_seqlens, int num_seqs,
                           const gdn_bf16_t* cache_q_in, const gdn_bf16_t* cache_k_in, const gdn_bf16_t* cache_v_in,
                           gdn_bf16_t* cache_q_out, gdn_bf16_t* cache_k_out, gdn_bf16_t* cache_v_out,
                           gdn_bf16_t* q, gdn_bf16_t* k, gdn_bf16_t* v, gdn_bf16_t* a, gdn_bf16_t* b,
                           int T_total, int D, int H, int dk, int dv, int conv_k, void* stream);

/*
 * The layer's x_n history after num_seqs packed sequences (HOST cu_seqlens as
 * above): hist [num_seqs, nc, D] receives the last nc rows of each sequence of
 * xn [T_total, D], preceded by those of prev [num_seqs, nc, D] (NULL = zeros)
 * where a sequence is shorter.  D % 8 == 0, 16-byte aligned buffers.
 * No reference counterpart (the decode-state `xn` of packed sequences).
 */
int gdn_packed_history_hip(const gdn_bf16_t* xn, const int32_t* cu_seqlens, int num_seqs, const gdn_bf16_t* prev,
                           gdn_bf16_t* hist, int nc, int D, void* stream);

/*
 * Stores n offsets held on the HOST to dst on the GPU, in stream order and
 * without a copy from host memory (they travel with the launch), e.g. the
 * cu_seqlens of gdn_prefill_varlen_hip.  No reference counterpart.
 */
int gdn_store_offsets_hip(const int32_t* host, int32_t* dst, int n, void* stream);

/*
 * Decode-step conv: P [B, 2 H dk + H dv + 2 H] bf16 holds xn W^T of the new
 * token (columns q|k|v|a|b).  q/k/v columns go through the causal conv over
 * the cached previous conv_k - 1 projections (cache_* [B, H d, conv_k - 1],
 * updated in place) and SiLU; a/b pass through.  Outputs in the decode
 * kernel's layouts: q, k [B, H, dk]; v [B, H, dv]; a, b [B, H].  With
 * xn_hist [B, conv_k - 1, D] (nullable) the same launch also moves the x_n
 * history one token older and appends xn [B, D] (the layer's decode-state
 * `xn`).  B <= 65535.
 * Replaces _decode_conv_step / _decode_fused_proj_step (gdn_layer.py:43-69).
 */
int gdn_decode_conv_step_hip(const gdn_bf16_t* P, const gdn_bf16_t* conv_w_qkv,
                             gdn_bf16_t* cache_q, gdn_bf16_t* cache_k, gdn_bf16_t* cache_v,
                             const gdn_bf16_t* xn, gdn_bf16_t* xn_hist,
                             gdn_bf16_t* q, gdn_bf16_t* k, gdn_bf16_t* v, gdn_bf16_t* a, gdn_bf16_t* b,
                             int B, int D, int H, int dk, int dv, int conv_k, void* stream);

/*
 * One decode step's input side for B <= 16 sequences: x_n = RMSNorm(x)
 * (x [B, D] bf16, gamma [D], eps; the same numbers as gdn_rmsnorm_hip),
 * P = x_n W_qkvab^T kept in fp32, then the conv step of
 * gdn_decode_conv_step_hip on P (conv caches updated in place; they receive
 * bf16(P)) and SiLU.  Outputs q, k [B, H, dk]; v [B, H, dv]; a, b [B, H].
 * xn_hist [B, conv_k - 1, D] (NULL = skipped) is shifted one token and x_n
 * appended, in place.  D % 32 == 0, D <= 4096, conv_k in 1..4.  Caches and
 * xn_hist must not alias the outputs.
 * Replaces GDNLayerCustom.decode's rmsnorm, projection GEMM and conv step
 * (gdn_layer.py:280-299 and 43-69).
 */
int gdn_decode_in_proj_hip(const gdn_bf16_t* x, const gdn_bf16_t* gamma, float eps, const gdn_bf16_t* W_qkvab,
                           const gdn_bf16_t* conv_w_qkv, gdn_bf16_t* cache_q, gdn_bf16_t* cache_k,
                           gdn_bf16_t* cache_v, gdn_bf16_t* xn_hist, gdn_bf16_t* q, gdn_bf16_t* k, gdn_bf16_t* v,
                           gdn_bf16_t* a, gdn_bf16_t* b, int B, int D, int H, int dk, int dv, int conv_k,
                           void* stream);

/*
 * y [B, N] bf16 = bf16(o) W^T for o [B, K] fp32 (the decode kernel's output,
 * rounded to bf16 as the reference's o.to(bf16)), W [N, K] bf16, fp32
 * accumulation.  B <= 16, K % 32 == 0, K <= 4096.
 * Replaces GDNLayerCustom.decode's output projection (gdn_layer.py:309).
 */
int gdn_decode_out_proj_hip(const float* o, const gdn_bf16_t* W, gdn_bf16_t* y, int B, int K, int N,
                            void* stream);

/*
 * The layer's output projection over M tokens: y [M, N] = o [M, K] W^T, W
 * [N, K], bf16 with fp32 sums.  K % 128 == 0, K <= 2^20, N % 8 == 0, 16-byte
 * aligned buffers.  Made for up to one round of its tiles; larger calls work,
 * at less than a library GEMM's rate.  The order of a row's sums follows M, K
 * and N.  gdn_out_proj_fits: 1 where M > 0 rows of these K and N are taken and
 * are one round, else 0 (no error is set).
 * Replaces `o @ W_o.T` of GDNLayerCustom.forward (gdn_layer.py:263).
 */
int gdn_out_proj_fits(int64_t M, int64_t K, int64_t N);
int gdn_out_proj_hip(const gdn_bf16_t* o, const gdn_bf16_t* W, gdn_bf16_t* y, int M, int K, int N, void* stream);

/*
 * One whole decode step of the layer, on `stream`: gdn_decode_in_proj_hip
 * (RMSNorm, projections, conv step, x_n history), gdn_decode_hip (state S,
 * in place when S_out == S_in) and gdn_decode_out_proj_hip, so a serving loop
 * pays one host call per step.  q, k, v, a, b ([B, H dk] x2, [B, H dv],
 * [B, H] x2 bf16) and o ([B, H dv] fp32) are caller-owned scratch; y is
 * [B, D] bf16.  B <= 16: gdn_decode_in_proj_hip, the recurrence and
 * gdn_decode_out_proj_hip, whose constraints and errors apply.
 * 16 < B <= 65535: RMSNorm (x_n written to y, which
 * is then scratch until the out-projection overwrites it, and the x_n
 * history shifted), a tiled in-projection with the conv step in its
 * epilogue, the recurrence, a tiled out-projection; D % 64 == 0, D <= 16384,
 * H dk and H dv multiples of 64, conv_k in 1..4, x/gamma/W/W_o/y/q/k/v/o/
 * caches/xn_hist 16-byte aligned.  Every argument is checked before the first
 * launch, so a refused call leaves the caches and state untouched.
 * Replaces GDNLayerCustom.decode (gdn_layer.py:265-316) as a whole.
 */
int gdn_layer_decode_step_hip(const gdn_bf16_t* x, const gdn_bf16_t* gamma, float eps, const gdn_bf16_t* W_qkvab,
                              const gdn_bf16_t* conv_w_qkv, gdn_bf16_t* cache_q, gdn_bf16_t* cache_k,
                              gdn_bf16_t* cache_v, gdn_bf16_t* xn_hist, const float* A_log, const float* dt_bias,
                              const float* S_in, float* S_out, float scale, const gdn_bf16_t* W_o, gdn_bf16_t* q,
                              gdn_bf16_t* k, gdn_bf16_t* v, gdn_bf16_t* a, gdn_bf16_t* b, float* o, gdn_bf16_t* y,
                              int B, int D, int H, int dk, int dv, int conv_k, void* stream);

/* Element types, 8-bit (e4m3: largest 448; e5m2: largest 57344) and 4-bit (e2m1: largest 6) formats, and gate activations. */
enum { GDN_BF16 = 0, GDN_F32 = 1, GDN_E8M0 = 2 };
enum { GDN_E4M3 = 0, GDN_E5M2 = 1, GDN_E2M1 = 2 };
enum { GDN_ACT_NONE = 0, GDN_ACT_SIGMOID = 1, GDN_ACT_SILU = 2, GDN_ACT_TANH = 3 };

/*
 * The norms before and after a block, fused with its gate and residual:
 *   u = RMSNorm(y) post_gamma                       (u = y without post_gamma)
 *   h = residual + residual_scale scale act(gate) u (absent: 0 and 1)
 *   n = RMSNorm(h) gamma
 * in fp32, rounded once where written; n follows from the unrounded h.
 *   y [R, D], gate [ceil(R / rows_per_gate), D] (row r takes gate row
 *   r / rows_per_gate: 1 = a gate row a token, T = one a sequence of T, R =
 *   one for all), n [R, D]: type_y; residual, h [R, D]: type_r;
 *   post_gamma, gamma, scale [D]: type_p.  Inputs but y may be NULL, outputs
 *   too.  Types (y, r, p): bf16 bf16 bf16, bf16 bf16 fp32, bf16 fp32 fp32,
 *   fp32 fp32 fp32.  ld*: elements from a row to the next.  h may be written
 *   over the rows of residual, y or a gate a token (same address, type and
 *   stride); a call whose h is not apart from an input otherwise, by its range
 *   of memory or by columns within a common stride, is refused, and so are rows
 *   of h or n that overlap.  The other outputs have to lie apart from the inputs.
 *   codes [R, ldc >= D padded to 128] and scales [ceil(D / 128), lds >= R]: n
 *   (h without gamma), unrounded, as e4m3 codes in blocks of 128 columns (see
 *   gdn_fp8_quantize_hip); codes 16-byte aligned, ldc % 16 == 0.
 *   rstd_y, rstd_h [R]: 1 / rms of y (with post_gamma) and of h (with gamma),
 *   which gdn_block_norm_bwd_hip takes.
 * D <= 16384, any D and alignment (16-byte ones and D % 8 == 0 are faster).
 */
int gdn_block_norm_hip(const void* y, int64_t ldy, const void* residual, int64_t ldr, const void* gate, int64_t ldg,
                       int64_t rows_per_gate, const void* post_gamma, const void* gamma, const void* scale,
                       float residual_scale, int act, float eps, void* h, int64_t ldh, void* n, int64_t ldn,
                       uint8_t* codes, int64_t ldc, uint8_t* scales, int64_t lds, float* rstd_y, float* rstd_h,
                       int64_t R, int64_t D, int type_y, int type_r, int type_p, void* stream);

/*
 * Gradients of gdn_block_norm_hip.  dh [R, D] (type_r) and dn [R, D] (type_y)
 * are those of h and n, either may be NULL (0; dn, gamma and rstd_h go
 * together, as do post_gamma and rstd_y); the other inputs and the rstd are the
 * forward pass's.  Outputs, contiguous, of their inputs' types, NULL = not
 * wanted (dy is): dresidual, dy [R, D], dgate [gate rows, D], dpost_gamma,
 * dgamma, dscale [D].  A gate row that rows share, and the parameters, get
 * fp32 sums in a fixed order.  workspace: gdn_block_norm_bwd_workspace_bytes
 * (R, D, rows_per_gate, or 1 without a gate) bytes, 16-byte aligned, where a
 * parameter's or a shared gate's gradient is wanted.  R == 0: the parameters'
 * gradients are zeros, dgate is not written.  At most 65535 shared gate rows.
 */
size_t gdn_block_norm_bwd_workspace_bytes(int64_t R, int64_t D, int64_t rows_per_gate);

int gdn_block_norm_bwd_hip(const void* dh, int64_t lddh, const void* dn, int64_t lddn, const void* y, int64_t ldy,
                           const void* residual, int64_t ldr, const void* gate, int64_t ldg, int64_t rows_per_gate,
                           const void* post_gamma, const void* gamma, const void* scale, float residual_scale, int act,
                           const float* rstd_y, const float* rstd_h, void* dresidual, void* dy, void* dgate,
                           void* dpost_gamma, void* dgamma, void* dscale, int64_t R, int64_t D, int type_y, int type_r,
                           int type_p, void* workspace, size_t workspace_bytes, void* stream);

/*
 * x [M, K] (bf16 or fp32, rows ldx elements apart) to 8-bit floating point
 * (GDN_E4M3 or GDN_E5M2), one power-of-two scale a block of block_rows (1 or
 * 128) x 128 values: 2^e with the least e >= -127 for which the block's largest
 * magnitude over 2^e is no larger than the format's largest number (e = 0 for
 * zeros), kept as the byte e + 127 (e8m0); a code is value / 2^e to the nearest,
 * ties to even.  A block with an infinity or NaN gets scale NaN (0xff), codes
 * NaN.  Along the rows: codes [M, ldc], columns K up to the next multiple of 128
 * zero; scales [ceil(K / 128), lds >= M] (block_rows 1; lds % 16 == 0) or
 * [ceil(M / 128), lds >= ceil(K / 128)] (128).  Along the columns, the same of
 * x^T: codes_t [K, ldt], columns M up to the next multiple of 128 zero; scales_t
 * [ceil(M / 128), ldst >= K] or [ceil(K / 128), ldst >= ceil(M / 128)].  Either
 * pair may be NULL.  Code rows 16-byte aligned.  What lies behind these in
 * wider buffers is left as it is.
 */
int gdn_fp8_quantize_hip(const void* x, int64_t ldx, int type_x, int64_t M, int64_t K, int block_rows, int format,
                         uint8_t* codes, int64_t ldc, uint8_t* scales, int64_t lds, uint8_t* codes_t, int64_t ldt,
                         uint8_t* scales_t, int64_t ldst, void* stream);

/*
 * Product of fp8 codes with a scale for each block of 128:
 *   out[m, n] = sum_kb a_scale[m, kb] b_scale[n, kb] sum_{k in kb} a[m, k] b[n, k]
 * out [M, ldo] bf16 or fp32 (type_out), rounded once from fp32 sums.  fp32 results
 * sum every product in full.  bf16 results leave a block's 128 products to one
 * instruction, which lines them up with the largest and drops what lies below 2^-17
 * of it: up to 2^-10 of the product of the row's and the column's largest code in
 * the block (times both scales), less than the result's rounding unless large
 * products of a block cancel; ask for fp32 results where they may.
 *   a [M, lda], b [N, ldb] codes (16-byte aligned rows, lda and ldb <= 2^22);
 *   a_scale e8m0 [K / 128, lda_s >= M], 16-byte aligned, lda_s % 16 == 0;
 *   b_scale e8m0 or fp32 (type_b_scale), a 128 x 128 block each
 *   [ceil(N / 128), ldb_s >= K / 128] (b_block_rows 128) or a row and block
 *   each [K / 128, ldb_s >= N], 16-byte aligned, ldb_s % 16 == 0 (1).
 * K % 128 == 0 (zero codes pad), any M, any N (up to 2^30 with an fp32 scale a
 * row and block).  Scales may be anything that the types hold; only the product of
 * the two has to be in fp32's range.  A row's sums do not depend on other rows'
 * values; their order follows M, N, K and the column.
 */
int gdn_fp8_matmul_hip(const uint8_t* a, int64_t lda, int format_a, const uint8_t* a_scale, int64_t lda_s,
                       const uint8_t* b, int64_t ldb, int format_b, const void* b_scale, int64_t ldb_s, int b_block_rows,
                       int type_b_scale, void* out, int64_t ldo, int type_out, int64_t M, int64_t N, int64_t K,
                       void* stream);

/*
 * x [M, K] (bf16 or fp32, rows ldx elements apart) to 4-bit floating point (e2m1),
 * one power-of-two scale a block of block_rows (1 or 32) x 32 values: 2^e with the
 * least e >= -127 for which the block's largest magnitude over 2^e is no larger than
 * 6 (e = 0 for zeros), kept as the byte e + 127 (e8m0); a code is value / 2^e to the
 * nearest, ties to even.  (Encoders that take 2^(floor(log2 max) - 2) and cut off at 6 give
 * other codes; they are decoded and multiplied alike.)  A block with an infinity or NaN gets scale NaN (0xff), codes
 * 0.  Along the rows: codes [M, ldc bytes], two a byte, the earlier one low, columns K
 * up to the next multiple of 256 zero; scales [K / 128, lds >= M, 4], blocks of 128
 * columns first (as many as the codes have), a row's four bytes adjacent.  Along the
 * columns, the same of x^T: codes_t [K, ldt bytes], columns M up to the next multiple
 * of 256 zero; scales_t [M / 128, ldst >= K, 4].  Either pair may be NULL.  Code rows
 * 16-byte aligned.  What lies behind these in wider buffers is left as it is.
 */
int gdn_fp4_quantize_hip(const void* x, int64_t ldx, int type_x, int64_t M, int64_t K, int block_rows, uint8_t* codes,
                         int64_t ldc, uint8_t* scales, int64_t lds, uint8_t* codes_t, int64_t ldt, uint8_t* scales_t,
                         int64_t ldst, void* stream);

/*
 * Both from one read of x: e2m1 codes along its rows, in blocks of 1 x 32 (codes and
 * scales as gdn_fp4_quantize_hip writes them), and e4m3 codes along its columns, in
 * blocks of 128 (codes_t [K, ldt >= M up to the next multiple of 128] and scales_t [M /
 * 128, ldst >= K] as gdn_fp8_quantize_hip writes them).
 */
int gdn_fp4_fp8_quantize_hip(const void* x, int64_t ldx, int type_x, int64_t M, int64_t K, uint8_t* codes, int64_t ldc,
                             uint8_t* scales, int64_t lds, uint8_t* codes_t, int64_t ldt, uint8_t* scales_t, int64_t ldst,
                             void* stream);

/*
 * What e2m1 codes [M, ldc bytes] with scales [K / 128, lds >= M, 4] stand for: out [M,
 * ldo] bf16 or fp32 (type_out), exactly; what lies beyond bf16's range is infinite,
 * a scale of 0xff NaN.  Any K, codes at 4 bytes.
 */
int gdn_fp4_dequantize_hip(const uint8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds, void* out, int64_t ldo,
                           int type_out, int64_t M, int64_t K, void* stream);

/*
 * Product with 4-bit weights:
 *   out[m, n] = sum_k a[m, k] a_scale[m, block of k] b[n, k] b_scale[n, block of k]
 * out [M, ldo] bf16 or fp32 (type_out), rounded once from fp32 sums.
 *   b [N, ldb bytes] e2m1 codes in rows of whole 256 values (zero codes behind K),
 *   b_scale e8m0 [K / 128 (an even number), ldb_s >= N, 4]: a scale a row and 32;
 *   a (format_a): GDN_E2M1, the same with a_scale [K / 128, lda_s >= M, 4], K % 256 ==
 *   0; or GDN_E4M3, GDN_E5M2 codes [M, lda] with a scale a row and 128, a_scale e8m0
 *   [K / 128, lda_s >= M], K % 128 == 0 (as gdn_block_norm_hip and
 *   gdn_fp8_quantize_hip write them).
 * Code rows are 16-byte aligned and at most 2^22 bytes apart.  Scales: 16-byte aligned
 * rows of K's blocks, ld % 4 == 0 (of 8-bit codes % 16), readable in whole.  M, N up to
 * 2^28, M N / 256 up to 2^31 and as far as a launch of 2^32 threads reaches (else
 * GDN_ERR_UNSUPPORTED).  With 8-bit codes, bf16 results leave 128 products to one instruction, which
 * drops what lies below 2^-17 of the largest; fp32 results sum every product in full.
 * With 4-bit ones, results of either type are sums of which each 128 products are added
 * with an error of at most 2^-21 of the largest among them, their sums of 32, the sum so
 * far and the new one.
 * Scales may be anything that the type holds; only the product of the two (of a row and
 * a column, in each block) has to be in fp32's range (fp32 results of 8-bit codes: where
 * the four scales of 128 values of b lie more than 2^110 apart, the smallest ones'
 * products lose bits).  A row's sums do not depend on
 * other rows' values; their order follows M, N, K and the column.
 */
int gdn_fp4_matmul_hip(const uint8_t* a, int64_t lda, int format_a, const uint8_t* a_scale, int64_t lda_s,
                       const uint8_t* b, int64_t ldb, const uint8_t* b_scale, int64_t ldb_s, void* out, int64_t ldo,
                       int type_out, int64_t M, int64_t N, int64_t K, void* stream);

/*
 * The 2-norm of `count` tensors together (a HOST array of device pointers; each n
 * adjacent elements, bf16 or fp32), norm [1] = sqrt(sum of squares), with sums in 64
 * bits in a fixed order.  Elements count as often as they are given.  type_out and out
 * are not read.  No tensors: 0.  workspace: gdn_grad_norm_workspace_bytes(count), 8-byte
 * aligned.
 */
typedef struct {
    const void* grad;
    void* out;
    int64_t n;
    int type, type_out;
} gdn_grad_t;

size_t gdn_grad_norm_workspace_bytes(int64_t count);

int gdn_grad_norm_hip(const gdn_grad_t* grads, int64_t count, float* norm, void* workspace, size_t workspace_bytes,
                      void* stream);

/*
 * The same, and out = grad min(1, max_norm / (norm + 1e-6)) for each tensor: the factor
 * from the 64-bit sums and the product each rounded to 24 bits of mantissa (a factor below
 * fp32's normal numbers keeps them), then to type_out; out may be grad itself (then of its
 * type; not written where the factor is 1) and lies apart from the other tensors, or the
 * call is refused.  norm and workspace lie apart from all of them.  A norm that is NaN makes
 * every result NaN.  An infinity among the gradients makes the factor 0: zeros, and NaN
 * where it stands; with an infinite max_norm, of which the factor is NaN, NaN everywhere.
 * (A norm that is infinite in 32 bits alone is not meant: its factor is as any other.)
 * max_norm >= 0.
 */
int gdn_clip_grad_norm_hip(const gdn_grad_t* grads, int64_t count, double max_norm, float* norm, void* workspace,
                           size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* GDN_AMD_H */
