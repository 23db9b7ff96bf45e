/*
 * fgs_moe.h -- C ABI of the MI355X (gfx950) fused-MoE library `libfgs_moe.so`.
 *
 * The library replaces the fused-MoE operator path of FlagGems-sglang
 * (reference: src/flaggems_sglang/ops/fused_moe.py). The reference has no
 * native FFI of its own -- its Python entry points launch Triton JIT kernels
 * and call `triton_kernels.matmul_ogs`. Each entry point below names the
 * reference function (file:line) whose work it takes over; the Python host
 * layer (flaggems_sglang.ops.fused_moe) binds them with ctypes.
 *
 * Conventions
 *   - Plain pointers to device memory and plain integer sizes. bf16 tensors
 *     are passed as `void*` (IEEE bfloat16, little endian); fp8 tensors are
 *     OCP e4m3fn bytes (max 448); int8 tensors are two's complement.
 *   - `stream` is a `hipStream_t` passed as `void*` (NULL = legacy stream).
 *   - Every launching entry point is asynchronous and stream ordered. The
 *     library never allocates or frees device memory and never synchronises;
 *     scratch memory comes in through the caller's `workspace` argument,
 *     sized with fgs_moe_workspace_bytes().
 *   - All arguments are validated on the host before any launch. Return
 *     codes: FGS_OK (0); FGS_EINVAL (-1) invalid argument; FGS_EUNSUPPORTED
 *     (-2) valid but unsupported combination; FGS_ELAUNCH (-3) HIP error.
 *     fgs_moe_last_error() returns the message of the calling thread's last
 *     failure.
 *   - Thread-safe and re-entrant: no mutable globals besides the
 *     thread-local error string and device properties cached once.
 */
#ifndef FGS_MOE_H_
#define FGS_MOE_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FGS_OK 0
#define FGS_EINVAL (-1)
#define FGS_EUNSUPPORTED (-2)
#define FGS_ELAUNCH (-3)

/* Quantisation modes (`qmode` arguments). */
#define FGS_QMODE_BF16 0        /* bf16 weights and activations               */
#define FGS_QMODE_FP8_BLOCK 1   /* e4m3fn w8a8, 128x128 weight blocks, 1x128  */
#define FGS_QMODE_INT8_CHANNEL 2 /* int8 w8a8, per-channel w, per-token a     */

/* `flags` bits of the fused entry points. */
#define FGS_FLAG_ROUTER_WEIGHT_ON_INPUT 0x1 /* gammas on GEMM1 output rows */
/* GEMM1 activation gelu(gate) * up (exact erf gelu, sgl_kernel's
 * gelu_and_mul, ops/fused_moe.py:219-220) instead of silu(gate) * up */
#define FGS_FLAG_ACT_GELU 0x2
#define FGS_FLAG_FORCE_DECODE 0x100         /* schedule: streaming kernels  */
#define FGS_FLAG_FORCE_PREFILL 0x200        /* schedule: LDS-tiled kernels  */
/* schedule: the weighted top-k sum runs as its own kernel (moe_sum); a
 * one-token call otherwise folds it into GEMM2 when that is faster */
#define FGS_FLAG_SEPARATE_SUM 0x400
/* schedule: a one-token call folds the weighted top-k sum into GEMM2 */
#define FGS_FLAG_FOLD_SUM 0x800
/* schedule: a one-token fp8 / int8 call quantises its activations with the
 * separate quantiser kernels; by default (top-k <= 64) its GEMMs quantise
 * their bf16 activation rows themselves (fp8: x and the GEMM1 output; int8:
 * the GEMM1 output, per-token scales), with the quantisers' arithmetic, so
 * both give the same bytes and scales */
#define FGS_FLAG_SEPARATE_QUANT 0x8
/* schedule: LDS-tiled kernels with row-block configuration c (0: 256 rows,
 * 1: 128, 2: 64, 3: 32, 4: 160) instead of the rows-per-expert choice */
#define FGS_FLAG_TILE(c) ((((c) + 1) & 0x7) << 12)
#define FGS_FLAG_TILE_MASK 0x7000

/* Library version string, e.g. "fgs_moe 0.1.0 gfx950". */
const char* fgs_moe_version(void);

/* Message of the calling thread's most recent failed call ("" if none). */
const char* fgs_moe_last_error(void);

/* Size of the padded sorted-id buffer the alignment writes:
 * numel + num_experts * (block_size - 1). Returns -1 on invalid input. */
int64_t fgs_moe_align_max_padded(int64_t numel, int32_t num_experts,
                                 int32_t block_size);

/* moe_align_block_size: expert-grouped, block-padded routing order.
 * Replaces the routing conversion of _standard_topk_to_triton_kernels
 * (ops/fused_moe.py:119-146: stable argsort :134, histogram :137-139).
 *   topk_ids     int32 [numel] (numel = M * topk), expert id per slot.
 *   sorted_ids   int32 [max_padded]: for each expert e in ascending order,
 *                the flat slot indices i with topk_ids[i] == e in ascending
 *                i (stable), then pad entries = numel up to a multiple of
 *                block_size; entries past the padded total are numel too.
 *   expert_ids   int32 [max_padded / block_size]: expert of each block,
 *                -1 past the padded total.
 *   num_post_pad int32 [1]: padded total.
 * Slots whose id is outside [0, num_experts) are dropped (not routed).
 * Bit-exact and deterministic (no atomics decide any order).
 * scratch: device memory of fgs_moe_align_scratch_bytes() bytes (or null /
 * too small: the computation then runs on one workgroup, slower for large
 * numel); the result is identical either way. */
int32_t fgs_moe_align_block_size(const int32_t* topk_ids, int64_t numel,
                                 int32_t num_experts, int32_t block_size,
                                 int32_t* sorted_ids, int32_t* expert_ids,
                                 int32_t* num_post_pad, int64_t max_padded,
                                 void* scratch, int64_t scratch_bytes,
                                 void* stream);

/* Scratch bytes fgs_moe_align_block_size uses for numel slots (0: none
 * needed), or -1 for invalid arguments. No reference counterpart (the
 * reference's conversion runs as torch ops, ops/fused_moe.py:130-139). */
int64_t fgs_moe_align_scratch_bytes(int64_t numel, int32_t num_experts);

/* Routing-format conversion: (topk_weights, topk_ids) -> the routing tuple
 * of triton_kernels that _standard_topk_to_triton_kernels builds
 * (ops/fused_moe.py:119-146), computed on the GPU:
 *   gate_scal  f32 [numel], topk_indx int32 [numel], gate_indx int32 [numel]:
 *              the reference's per-token ascending id sort (:130-131), the
 *              stable argsort of the flattened ids (:134), its inverse
 *              (:135) and the gathered weights (:136);
 *   hist       int32 [E] (:137-139, ids outside [0, E) not counted);
 *   token_offs_raw int32 [E + 1], token_offs_pad int32 [4][E + 1] and
 *   block_pid_map int32 [4][max_tiles]: the tables of triton_kernels'
 *              compute_expt_data_torch (:140) for block_m = 16, 32, 64, 128
 *              (row i of the [4][...] arrays): exclusive sums of hist and of
 *              ceil(hist / block_m) (the latter in tiles), and per tile
 *              (b << 16) | e for expert e's b-th tile, -1 past the last.
 * numel = m * topk; num_experts <= 1022; max_tiles >=
 * fgs_moe_routing_max_tiles(numel, E) (compute_expt_data_torch's bound);
 * workspace: fgs_moe_routing_workspace_bytes(numel, E) bytes, 256-aligned.
 * Slots whose id is outside [0, E) (not routed here) sort behind expert
 * E-1, in slot order, where no expert's token_offs_raw range reaches them
 * (the reference's argsort would put negative ids ahead of expert 0; its
 * callers never pass any). Deterministic (no atomics). */
int64_t fgs_moe_routing_max_tiles(int64_t numel, int32_t num_experts);
int64_t fgs_moe_routing_workspace_bytes(int64_t numel, int32_t num_experts);
int32_t fgs_moe_topk_to_routing(const float* topk_weights, const int32_t* topk_ids,
                                int64_t m, int32_t topk, int32_t num_experts,
                                float* gate_scal, int32_t* topk_indx, int32_t* gate_indx,
                                int32_t* hist, int32_t* token_offs_raw,
                                int32_t* token_offs_pad, int32_t* block_pid_map,
                                int64_t max_tiles, void* workspace, int64_t ws_bytes,
                                void* stream);

/* The inverse conversion: the routing tuple -> per-slot (topk_weights,
 * topk_ids) in the row-sorted slot order of the tuple's flat indices (each
 * token's slots by ascending expert id, ops/fused_moe.py:130). Expert e owns
 * the gathered positions [token_offs_raw[e], token_offs_raw[e + 1]) of
 * gather_src, with token_offs_raw the exclusive sums of expt_hist -- the
 * ranges matmul_ogs reads (ops/fused_moe.py:205-231); slots at positions
 * past the histogram's total get id -1 (dropped). For v = gather_src[p]:
 * topk_ids[v] = that expert, topk_weights[v] = gate_scal[p].
 *   gate_scal f32 [m*topk], gather_src int32 [m*topk] (gather_indx.src_indx,
 *   a permutation of [0, m*topk)), expt_hist int32 [num_experts];
 *   num_experts <= 1024. Counts are clamped to the slots that exist;
 *   gather_src entries outside [0, m*topk) are skipped. */
int32_t fgs_moe_routing_to_topk(const float* gate_scal, const int32_t* gather_src,
                                const int32_t* expt_hist, int64_t m, int32_t topk,
                                int32_t num_experts, float* topk_weights, int32_t* topk_ids,
                                void* stream);

/* silu_and_mul: out[r, c] = bf16(silu(f32(in[r, c])) * f32(in[r, n + c])).
 * in bf16 [rows, 2n], out bf16 [rows, n].
 * Replaces _silu_and_mul_triton / _silu_and_mul_kernel
 * (ops/fused_moe.py:44-63, 88-116). */
int32_t fgs_moe_silu_and_mul(const void* in, void* out, int64_t rows,
                             int64_t n, void* stream);

/* moe_sum: out[t, c] = bf16(sum_j f32(in[t, j, c])), in bf16 [m, topk, k],
 * out bf16 [m, k]. Replaces the top-k reduction that matmul_ogs performs
 * with `scatter_indx` (ops/fused_moe.py:224-231). */
int32_t fgs_moe_sum(const void* in, void* out, int64_t m, int32_t topk,
                    int64_t k, void* stream);

/* Router gating: scores -> top-k -> optional renormalisation, producing
 * the (topk_weights, topk_ids) the fused entry points consume. Replaces the
 * torch routing of the reference's tests (tests/test_fused_moe.py:37-41:
 * softmax, topk, renormalise) that feeds _standard_topk_to_triton_kernels
 * (ops/fused_moe.py:119-146); sigmoid scoring for DeepSeek-style routers.
 *   logits  f32 or bf16 (logits_bf16 != 0) [m, num_experts], num_experts <= 1024
 *   topk_weights f32 [m, topk], topk_ids int32 [m, topk], topk <= 64
 * Experts are ranked by logit (descending; equal logits: lower id first) and
 * written in rank order; weights are the scores, divided by their top-k sum
 * when renormalize != 0. */
#define FGS_SCORING_SOFTMAX 0
#define FGS_SCORING_SIGMOID 1
int32_t fgs_moe_topk_gating(const void* logits, int32_t logits_bf16, int64_t m,
                            int32_t num_experts, int32_t topk, int32_t scoring,
                            int32_t renormalize, float* topk_weights,
                            int32_t* topk_ids, void* stream);

/* Dynamic per-(row, group) fp8 quantisation: x bf16 [rows, cols],
 * q e4m3fn [rows, cols], scales f32 [rows, cols / group] with
 * scale = max(amax, 1e-10) / 448 and q = e4m3fn(clamp(x / scale, +-448)).
 * group: a power of two in [8, 512] dividing cols.
 * No reference counterpart (the reference asserts fp8 off,
 * ops/fused_moe.py:170-172); needed by the fp8 w8a8 path. */
int32_t fgs_moe_quant_fp8_group(const void* x, void* q, float* scales,
                                int64_t rows, int64_t cols, int32_t group,
                                void* stream);

/* Dynamic per-row int8 quantisation: scale = max(amax, 1e-10) / 127,
 * q = clamp(rne(x / scale), -127, 127). x bf16 [rows, cols], q int8,
 * scales f32 [rows]; cols a multiple of 8.
 * No reference counterpart (ops/fused_moe.py:173-175 asserts per-channel
 * quant off); needed by the int8 w8a8 path. */
int32_t fgs_moe_quant_int8_token(const void* x, int8_t* q, float* scales,
                                 int64_t rows, int64_t cols, void* stream);

/* Workspace bytes one fused call needs for the given problem.
 * m tokens, hidden K, inter N (per-expert intermediate), num_experts E,
 * topk, qmode, flags (schedule bits matter). Returns -1 on invalid input. */
int64_t fgs_moe_workspace_bytes(int64_t m, int64_t hidden, int64_t inter,
                                int32_t num_experts, int32_t topk,
                                int32_t qmode, int32_t flags);

/* The schedule a fused call of this problem runs, as a short text into
 * buf (NUL-terminated, truncated to len - 1 bytes):
 * "direct" / "direct_sum" (one token, two streaming GEMMs, the top-k sum
 * separate / folded into GEMM2), "stream mt=T" (streaming GEMMs over the
 * aligned rows) or "tiled cfg=A cfg2=B [ksplit2=S] [tail2]" (LDS-tiled
 * GEMMs). Host-only. No counterpart in the reference (a diagnostic for
 * benchmarks and tests). */
int32_t fgs_moe_schedule(int64_t m, int64_t hidden, int64_t inter, int32_t num_experts,
                         int32_t topk, int32_t qmode, int32_t flags, char* buf,
                         int32_t len);

/* Host-only validation of a problem (no device access). Returns FGS_OK or
 * the status and message the fused entry point would return. */
int32_t fgs_moe_validate(int64_t m, int64_t hidden, int64_t inter,
                         int32_t num_experts, int32_t topk, int32_t qmode,
                         int32_t flags, int64_t ws_bytes);

/* Fused MoE, bf16. Replaces triton_kernel_fused_experts
 * (ops/fused_moe.py:149-232): routing conversion, GEMM1 (matmul_ogs with
 * gather, :205-212), silu_and_mul (:214-218), GEMM2 with top-k gammas and
 * scatter-reduce (:224-231).
 *   x            bf16 [m, hidden]
 *   w13          bf16 [E, 2*inter, hidden]  (gate rows 0..inter-1, then up)
 *   w2           bf16 [E, hidden, inter]
 *   topk_weights f32  [m, topk]
 *   topk_ids     int32 [m, topk]
 *   out          bf16 [m, hidden]
 *   out = sum_j w[t,j] * (silu(x W13g^T) * (x W13u^T)) W2^T  per token.
 * With FGS_FLAG_ROUTER_WEIGHT_ON_INPUT the gamma scales the GEMM1 output
 * rows (before the activation) and GEMM2 is unweighted
 * (ops/fused_moe.py:202-203). */
int32_t fgs_moe_fused_bf16(const void* x, const void* w13, const void* w2,
                           const float* topk_weights, const int32_t* topk_ids,
                           int64_t m, int64_t hidden, int64_t inter,
                           int32_t num_experts, int32_t topk, int32_t flags,
                           void* workspace, int64_t ws_bytes, void* out,
                           void* stream);

/* Allocation-free variant of fgs_moe_fused_bf16. No counterpart in the
 * reference: it is for callers that cannot allocate device memory -- code
 * under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc. Same arguments, kernels and results as fgs_moe_fused_bf16,
 * without the workspace: the library's own device scratch array of
 * FGS_NOALLOC_SCRATCH_BYTES per GPU (held from library load until the
 * process ends) stands in for it, and the call makes no hipMalloc / hipFree
 * or other allocating runtime call (stage profiling is off for it).
 * Problems whose workspace (fgs_moe_workspace_bytes) exceeds the scratch
 * return FGS_EUNSUPPORTED with a message naming the size, before any
 * launch. Every call on a GPU shares that GPU's scratch, which keeps the
 * last call's contents (no part of it needs to start at zero): calls that
 * overlap on one GPU -- on different streams, or from different threads
 * without ordering -- race. The scratch is the current device's: a stream
 * of another device is refused (FGS_EINVAL). Under HIP graph capture, make
 * one eager call on the device first: the first call on a device takes the
 * scratch address and sets kernel attributes, which must not happen inside
 * a capture; the captured launches use no memset and allocate nothing. */
#define FGS_NOALLOC_SCRATCH_BYTES (64ll << 20)
int32_t fgs_moe_fused_bf16_noalloc(const void* x, const void* w13, const void* w2,
                                   const float* topk_weights, const int32_t* topk_ids,
                                   int64_t m, int64_t hidden, int64_t inter,
                                   int32_t num_experts, int32_t topk, int32_t flags,
                                   void* out, void* stream);

/* Fused MoE with biases and the swiglu activation, bf16. Replaces
 * triton_kernel_fused_experts_with_bias (ops/fused_moe.py:235-325):
 * GEMM1 with bias b1 and swiglu fused (matmul_ogs(..., bias=b1,
 * fused_activation=swiglu, :303-313)), GEMM2 with bias b2 (:315-323), top-k
 * gammas and sum.
 *   w13 bf16 [E, 2*inter, hidden] (gate rows 0..inter-1, then linear rows:
 *       the reference's interleaved columns de-interleaved once by the caller)
 *   b13 f32 [E, 2*inter] (same row order), b2 f32 [E, hidden]
 *   a = bf16(g * sigmoid(alpha*g) * (u + 1)) with g = x W13g^T + b13g,
 *   u = x W13u^T + b13u and, for limit > 0, g = min(g, limit),
 *   u = clamp(u, -limit, limit); y = bf16(a W2^T + b2); out = bf16(sum_j w_j y_j).
 *   With FGS_FLAG_ROUTER_WEIGHT_ON_INPUT: a = bf16(w_j * swiglu) and
 *   out = bf16(sum_j y_j) (matmul_ogs scales its fused activation's output).
 * FGS_FLAG_ACT_GELU is rejected (the reference raises for non-silu,
 * :280-283). */
int32_t fgs_moe_fused_bf16_bias(const void* x, const void* w13, const float* b13,
                                const void* w2, const float* b2,
                                const float* topk_weights, const int32_t* topk_ids,
                                int64_t m, int64_t hidden, int64_t inter,
                                int32_t num_experts, int32_t topk, int32_t flags,
                                float alpha, float limit, void* workspace,
                                int64_t ws_bytes, void* out, void* stream);

/* The same with quantised weights: the precision configs the reference
 * threads into its two matmul_ogs calls (w1_pcg / w2_pcg,
 * ops/fused_moe.py:296-301, 303-324) carrying this build's w8a8 formats.
 *   qmode FGS_QMODE_FP8_BLOCK: w13 / w2 e4m3fn with the 128x128 block
 *       scales of fgs_moe_fused_fp8_block (activations quantised per 1x128
 *       group inside the call);
 *   qmode FGS_QMODE_INT8_CHANNEL: w13 / w2 int8 with the per-output-row
 *       scales of fgs_moe_fused_int8_channel (activations per token).
 * Biases, swiglu, gammas and the sum as fgs_moe_fused_bf16_bias; the
 * biases add to the dequantised GEMM outputs. */
int32_t fgs_moe_fused_quant_bias(int32_t qmode, const void* x, const void* w13,
                                 const float* b13, const void* w2, const float* b2,
                                 const float* w13_scale, const float* w2_scale,
                                 const float* topk_weights, const int32_t* topk_ids,
                                 int64_t m, int64_t hidden, int64_t inter,
                                 int32_t num_experts, int32_t topk, int32_t flags,
                                 float alpha, float limit, void* workspace,
                                 int64_t ws_bytes, void* out, void* stream);

/* The fused entry points above in one, with the layer output scaled: out =
 * bf16(out_scale * bf16(layer output)), the values of an in-place
 * multiplication of the output (the adapter's routed scaling factor,
 * ops/fused_moe.py:415-420) without its launch and its pass over the output.
 * qmode and scales as fgs_moe_fused_bf16 / _fp8_block / _int8_channel; b13
 * and b2 both null or both set as in fgs_moe_fused_routed below. */
int32_t fgs_moe_fused_scaled(int32_t qmode, const void* x, const void* w13, const void* w2,
                             const float* w13_scale, const float* w2_scale, const float* b13,
                             const float* b2, float alpha, float limit,
                             const float* topk_weights, const int32_t* topk_ids, int64_t m,
                             int64_t hidden, int64_t inter, int32_t num_experts, int32_t topk,
                             int32_t flags, float out_scale, void* workspace, int64_t ws_bytes,
                             void* out, void* stream);

/* Fused MoE on the reference's routing tuple instead of (topk_weights,
 * topk_ids): the inputs triton_kernel_fused_experts
 * (ops/fused_moe.py:149-232) and triton_kernel_fused_experts_with_bias
 * (:235-325) hand to matmul_ogs -- routing_data.gate_scal, gather_indx.src_indx
 * and routing_data.expt_hist. The tuple's gathered order is used as the
 * GEMMs' expert-sorted order directly (one kernel builds the block-padded
 * rows and each slot's expert id and gate scale; no top-k reconstruction, no
 * second alignment), with the slot conventions of fgs_moe_routing_to_topk.
 * qmode and scales as fgs_moe_fused_bf16 / _fp8_block / _int8_channel; b13
 * and b2 both null (silu, or gelu with FGS_FLAG_ACT_GELU) or both set (the
 * bias variant: swiglu(alpha, limit) as fgs_moe_fused_bf16_bias). Same
 * workspace (fgs_moe_workspace_bytes) and output as those entry points on
 * the equivalent (topk_weights, topk_ids). src is a permutation of the slots:
 * entries outside [0, m * topk) are skipped, a slot named twice takes either
 * entry's result, and the output row of a token with a slot that src never
 * names is unspecified. */
int32_t fgs_moe_fused_routed(int32_t qmode, const void* x, const void* w13, const void* w2,
                             const float* w13_scale, const float* w2_scale, const float* b13,
                             const float* b2, float alpha, float limit,
                             const float* gate_scal, const int32_t* gather_src,
                             const int32_t* expt_hist, int64_t m, int64_t hidden,
                             int64_t inter, int32_t num_experts, int32_t topk, int32_t flags,
                             void* workspace, int64_t ws_bytes, void* out, void* stream);

/* Fused MoE, fp8 w8a8 with block scales (block_n = block_k = 128).
 *   w13 e4m3fn [E, 2*inter, hidden], w13_scale f32 [E, 2*inter/128, hidden/128]
 *   w2  e4m3fn [E, hidden, inter],   w2_scale  f32 [E, hidden/128, inter/128]
 * Activations (x and the GEMM1 output) are quantised dynamically per 1x128
 * group inside the call. No reference counterpart: the reference rejects
 * use_fp8_w8a8 / w*_scale / block_shape (ops/fused_moe.py:170-185). */
int32_t fgs_moe_fused_fp8_block(const void* x, const void* w13,
                                const void* w2, const float* w13_scale,
                                const float* w2_scale, int32_t block_n,
                                int32_t block_k, const float* topk_weights,
                                const int32_t* topk_ids, int64_t m,
                                int64_t hidden, int64_t inter,
                                int32_t num_experts, int32_t topk,
                                int32_t flags, void* workspace,
                                int64_t ws_bytes, void* out, void* stream);

/* Fused MoE, int8 w8a8 with per-output-channel weight scales.
 *   w13 int8 [E, 2*inter, hidden], w13_scale f32 [E, 2*inter]
 *   w2  int8 [E, hidden, inter],   w2_scale  f32 [E, hidden]
 * Activations are quantised dynamically per token (row) inside the call.
 * No reference counterpart (per_channel_quant asserted off,
 * ops/fused_moe.py:173-175). */
int32_t fgs_moe_fused_int8_channel(const void* x, const void* w13,
                                   const void* w2, const float* w13_scale,
                                   const float* w2_scale,
                                   const float* topk_weights,
                                   const int32_t* topk_ids, int64_t m,
                                   int64_t hidden, int64_t inter,
                                   int32_t num_experts, int32_t topk,
                                   int32_t flags, void* workspace,
                                   int64_t ws_bytes, void* out, void* stream);

/* ---- dense operators around the routed experts -------------------------
 * No counterparts on the reference's path (its layer takes its input
 * normalised and has no 8-bit mode, ops/fused_moe.py:170-185): the norm before the
 * layer, the dense e4m3 products of the shared expert and the projections,
 * and the shared expert's activation. Element types of these entries: */
#define FGS_DTYPE_BF16 0
#define FGS_DTYPE_FP16 1
#define FGS_DTYPE_FP32 2
/* and their 8-bit outputs: e4m3fn with a scale per 128 columns of a row (the
 * last group may be shorter), int8 with a scale per row. The scale of a group
 * with a NaN is NaN, of one with an infinity infinite (its finite values then
 * have code 0). */
#define FGS_QUANT_NONE 0
#define FGS_QUANT_FP8_GROUP 1
#define FGS_QUANT_INT8_TOKEN 2

/* Root-mean-square norm, with the residual's addition and an 8-bit output:
 *   h = f32(x) + f32(residual);  residual_out = h in x's type
 *   n = h / sqrt(mean(h^2) + eps) * (f32(weight) + weight_offset)
 *   norm_out = n in x's type;  q, scales from the unrounded n
 * (scale = max(amax, 1e-10) / 448, q = e4m3fn(n / scale), or / 127, rne).
 *   x [rows, cols] with row stride x_stride (elements), residual likewise or
 *   null (then residual_out is unused); residual_out [rows, cols] may be
 *   residual or x itself; weight [cols] in x's type or fp32
 *   norm_out [rows, cols] contiguous, or null
 *   q [rows, cols] contiguous, scales f32 at scales[r * scale_row_stride +
 *   g * scale_col_stride] (g = column / 128; int8: g = 0), both null for
 *   FGS_QUANT_NONE
 * Any cols in [1, 65536] and any alignment to the element size; multiples of
 * 8 columns and 16-byte aligned rows take whole vectors. */
int32_t fgs_moe_rms_norm(const void* x, int64_t x_stride, const void* residual,
                         int64_t residual_stride, const void* weight, int32_t dtype,
                         int32_t weight_dtype, float eps, float weight_offset, int64_t rows,
                         int64_t cols, void* norm_out, void* residual_out,
                         int64_t residual_out_stride, int32_t quant, void* q, float* scales,
                         int64_t scale_row_stride, int64_t scale_col_stride, void* stream);

/* Gated activation with an 8-bit output: v = act(f32(x[r, c])) *
 * f32(x[r, n + c]) with act silu, or the exact gelu (gelu != 0), and q,
 * scales from the unrounded v as above (quant: FP8_GROUP or INT8_TOKEN).
 *   x [rows, 2n] with row stride x_stride; q [rows, n] contiguous; n in
 *   [1, 65536] */
int32_t fgs_moe_silu_and_mul_quant(const void* x, int64_t x_stride, int32_t dtype, int64_t rows,
                                   int64_t n, int32_t gelu, int32_t quant, void* q,
                                   float* scales, int64_t scale_row_stride,
                                   int64_t scale_col_stride, void* stream);

/* Dense e4m3 product with block scales (128x128 of the weights, 1x128 of the
 * activations), sums in fp32:
 *   out[i, j] = sum_kb a_scale[i, kb] * w_scale[j / 128, kb] *
 *               sum_{l in kb} a[i, l] * w[j, l]   (+ bias[j])
 *   a e4m3fn [m, k] with row stride lda; a_scale f32 at a_scale[i *
 *   as_row_stride + kb * as_col_stride]; w e4m3fn [n, k] with row stride ldw;
 *   w_scale f32 [ceil(n / 128), ceil(k / 128)] contiguous; bias [n] of
 *   bias_dtype, or null; out [m, n] of out_dtype (bf16 or fp16) with row
 *   stride ldo
 * The matrix instruction cuts each of eight neighbouring products 13 bits
 * below the largest one: about 1.5e-5 of a result from normal data, at most
 * 7 * 2^-13 of each eight's largest product (also where these cancel).
 * k a positive multiple of 16, m, n and k up to 2^22; a and w rows 16-byte
 * aligned and at most 2^22 apart, a_scale rows at most 2^20. `flags`: 0, or
 * FGS_BLOCK_FORM(f), the kernel form f whatever the sizes (for measurement
 * and tests). No workspace. */
#define FGS_BLOCK_FORM(f) ((f) + 1)
int32_t fgs_moe_fp8_block_matmul(const void* a, int64_t lda, const float* a_scale,
                                 int64_t as_row_stride, int64_t as_col_stride, const void* w,
                                 int64_t ldw, const float* w_scale, const void* bias,
                                 int32_t bias_dtype, int64_t m, int64_t n, int64_t k,
                                 int32_t out_dtype, int32_t flags, void* out, int64_t ldo,
                                 void* stream);
/* The schedule such a call runs, as text (as fgs_moe_schedule). */
int32_t fgs_moe_fp8_block_matmul_schedule(int64_t m, int64_t n, int64_t k, int32_t flags,
                                          char* buf, int32_t len);

/* ---- the routed layer's steps, with gradients ---------------------------
 * The reference runs the layer as one call without gradients
 * (ops/fused_moe.py:149-232); these are its steps for a program that trains it or
 * sends tokens to other GPUs between them. Activations of the products: */
#define FGS_ACT_NONE 0
#define FGS_ACT_RELU 1
#define FGS_ACT_SILU 2
#define FGS_ACT_GELU 3 /* exact (erf) */

/* Gradient of fgs_moe_topk_gating's weights: dlogits [m, num_experts] (of
 * logits' type) from the weights and ids that it returned for these logits and
 * dweights f32 [m, topk]. (Ids outside [0, num_experts) have no gradient.) logits may
 * be null where they are not read: softmax renormalised, sigmoid not. */
int32_t fgs_moe_topk_gating_grad(const void* logits, int32_t logits_bf16, int64_t m,
                                 int32_t num_experts, int32_t topk, int32_t scoring,
                                 int32_t renormalize, const float* topk_weights,
                                 const int32_t* topk_ids, const float* dweights, void* dlogits,
                                 void* stream);

/* Tokens sorted by expert: rows[p] = x[s / topk] for the slot s in place p of the
 * slots sorted by expert, then by slot.
 *   x: m rows of row_bytes (any element type), x_stride bytes apart
 *   topk_ids int32 [m, topk]; ids outside [0, num_experts) (slots of other GPUs'
 *   experts) come behind the last expert's, as rows of zeros
 *   rows [m * topk] of row_bytes, contiguous; counts int32 [num_experts]
 *   row_of_slot int32 [m, topk]: the slot's row, -1 for slots of no expert here
 *   slot_of_row int32 [m * topk]: its inverse, -1 for the rows behind
 * No result depends on the order of atomics. num_experts <= 1022; m * topk <= 2^30,
 * and fewer than 2^23 tokens with fewer than 2^27 slots fit the grids of all entries
 * here (others are refused where they do not). Workspace: fgs_moe_permute_workspace_bytes, 256-byte aligned, this call's
 * alone until it has run. */
int64_t fgs_moe_permute_workspace_bytes(int64_t numel, int32_t num_experts);
int32_t fgs_moe_permute(const void* x, int64_t x_stride, int64_t m, int64_t row_bytes,
                        const int32_t* topk_ids, int32_t topk, int32_t num_experts, void* rows,
                        int32_t* counts, int32_t* row_of_slot, int32_t* slot_of_row,
                        void* workspace, int64_t ws_bytes, void* stream);
/* The same rows by an order that fgs_moe_permute has made. */
int32_t fgs_moe_permute_rows(const void* x, int64_t x_stride, int64_t m, int64_t row_bytes,
                             const int32_t* row_of_slot, int32_t topk, const int32_t* slot_of_row,
                             void* rows, void* stream);

/* Rows back to tokens: out[t] = sum_k w[t, k] rows[row_of_slot[t, k]], in fp32 from
 * k = 0 on. Slots whose row lies outside [0, n_rows) add nothing, whatever their
 * weight. topk_weights f32 [m, topk] or null (ones); rows [n_rows, cols] of dtype
 * with row stride ld; out [m, cols] contiguous. */
int32_t fgs_moe_unpermute(const void* rows, int64_t ld, int64_t n_rows,
                          const int32_t* row_of_slot, const float* topk_weights, int64_t m,
                          int32_t topk, int64_t cols, int32_t dtype, void* out, void* stream);
/* Its gradients: drows[row_of_slot[t, k]] = w[t, k] dout[t], 0 for rows whose
 * slot_of_row is negative ([n_rows, cols] contiguous, or null), and dweights[t, k] =
 * <dout[t], rows[row_of_slot[t, k]]>, 0 for slots without a row (f32 [m, topk], or
 * null). The order is one that fgs_moe_permute has made: a row that two slots name
 * has either's gradient. */
int32_t fgs_moe_unpermute_grad(const void* dout, int64_t ldd, const void* rows, int64_t ld,
                               int64_t n_rows, const int32_t* row_of_slot,
                               const int32_t* slot_of_row, const float* topk_weights, int64_t m,
                               int32_t topk, int64_t cols, int32_t dtype, void* drows,
                               float* dweights, void* stream);

/* Products of bf16 or fp16 matrices with fp32 sums, dense or by group of rows:
 *   v = x[i] . w[e][j] + bias[e][j]
 *   out[i, j] = act(v_j) + residual[i, j]                      (wide = n)
 *   out[i, j] = act(v_j) * v_{n + j} + residual[i, j]          (gated: wide = 2 n)
 * rounded once to dtype; z (or null) f32 [rows, wide] gets v.
 *   x [rows, k] with row stride ldx; w [groups][wide, k] with row stride ldw and
 *   w_group_stride elements between the groups' matrices; bias [groups, wide] or
 *   null; residual [rows, n] with row stride ldr, or null; out [rows, n] contiguous
 *   counts int32 [groups] on the device: the rows of each group, which follow each
 *   other from row 0 on (negative ones count as 0, and what passes the last row is
 *   cut); rows behind the last group's have no product (out = residual, or 0; their
 *   z is not defined). Null: one matrix for all rows.
 * n and k multiples of 8, n (gated: 2 n) and k up to 2^20; fewer than 2^30 rows, up to 4096 groups; rows of x, w,
 * residual 16-byte aligned and at most 2^21 elements apart. No workspace. `flags`:
 * 0, or FGS_LINEAR_FORM(f), the kernel form f whatever the sizes (for measurement
 * and tests). */
#define FGS_LINEAR_FORM(f) ((f) + 1)
int32_t fgs_moe_linear(const void* x, int64_t ldx, const void* w, int64_t ldw,
                       int64_t w_group_stride, const void* bias, const void* residual,
                       int64_t ldr, const int32_t* counts, int32_t groups, int64_t rows,
                       int64_t n, int64_t k, int32_t dtype, int32_t act, int32_t gated,
                       int32_t flags, float* z, void* out, void* stream);
/* Its gradients. dz [rows, wide] contiguous, of v, in dtype (rows behind the last group's: of
 * whatever z holds there; the entries below leave them out). With dtype | FGS_DZ_REST a
 * second matrix follows it, bf16 [rows, wide], of what its rounding left (0 where dz is not
 * finite), for the bias's gradient: */
#define FGS_DZ_REST 0x100
int32_t fgs_moe_linear_act_grad(const void* dout, int64_t ldd, const float* z, int64_t rows,
                                int64_t n, int32_t dtype, int32_t act, int32_t gated, void* dz,
                                void* stream);
/* dx [rows, k] = dz[i] w[e], contiguous (rows behind the last group's: 0); rows of w at
 * least k elements apart, */
int32_t fgs_moe_linear_input_grad(const void* dz, int64_t ldz, const void* w, int64_t ldw,
                                  int64_t w_group_stride, const int32_t* counts, int32_t groups,
                                  int64_t rows, int64_t wide, int64_t k, int32_t dtype,
                                  int32_t flags, void* dx, void* stream);
/* dw [groups][wide, k] = sum over the group's rows of dz[i]^T x[i], contiguous; rows of
 * dz at least wide, rows of x at least k elements apart, */
int32_t fgs_moe_linear_weight_grad(const void* dz, int64_t ldz, const void* x, int64_t ldx,
                                   const int32_t* counts, int32_t groups, int64_t rows,
                                   int64_t wide, int64_t k, int32_t dtype, int32_t flags,
                                   void* dw, void* stream);
/* dbias [groups, wide] = sum over the group's rows of dz[i] (dtype | FGS_DZ_REST: of both
 * matrices, contiguous); workspace fgs_moe_linear_bias_grad_workspace_bytes (0: none),
 * 16-byte aligned. */
int64_t fgs_moe_linear_bias_grad_workspace_bytes(int32_t groups, int64_t rows, int64_t wide);
int32_t fgs_moe_linear_bias_grad(const void* dz, int64_t ldz, const int32_t* counts,
                                 int32_t groups, int64_t rows, int64_t wide, int32_t dtype,
                                 void* workspace, int64_t ws_bytes, void* dbias, void* stream);
/* The schedule of a product, as text (as fgs_moe_schedule): `pass` 0 the forward
 * one, 1 the input's gradient, 2 the weights'. */
int32_t fgs_moe_linear_schedule(int32_t pass, int32_t groups, int64_t rows, int64_t n, int64_t k,
                                int32_t gated, int32_t flags, char* buf, int32_t len);

/* Stage timing for benchmarks. No reference counterpart (the reference
 * times the whole op with triton.testing.do_bench,
 * benchmark/performance_utils.py:365-377). While enabled on the calling
 * thread, every fused call records HIP events on its stream between its
 * stages: 0 alignment, 1 activation quantisation, 2 GEMM1 (+activation),
 * 3 GEMM2-input quantisation, 4 GEMM2, 5 top-k sum. Stages a mode does not
 * run read ~0. on = 1 records every stage boundary; on = 2 only those of
 * stages 2..4 (GEMM1 through GEMM2), so a timed run carries three fewer
 * events per call; on = 3 only GEMM1's two (the other stages then read
 * 0); on = 0 stops. */
#define FGS_PROFILE_STAGES 6
int32_t fgs_moe_profile_enable(int32_t on);

/* Waits for the recorded events, writes the mean milliseconds of each stage
 * over the calls recorded since the last read into stage_ms[0..n_stages),
 * clears the record and returns the number of calls averaged (or < 0). */
int32_t fgs_moe_profile_read(float* stage_ms, int32_t n_stages);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* FGS_MOE_H_ */
