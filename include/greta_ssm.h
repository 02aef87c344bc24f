/*
 * greta_ssm.h -- C ABI of the state-space operators in libgreta_dynconv.so:
 * the selective state-space scan, its short causal convolution, and the
 * metadata of a packed serving batch. B200 (sm_100a). No counterpart in the
 * reference, whose only recurrent mixer is the dynamic convolution of
 * greta_dynconv.h; these take the same packed streams, cache slots and
 * request metadata.
 *
 * Conventions are those of greta_dynconv.h (device pointers on the current
 * device, GRETA_DT_* element types, a cudaStream_t, status codes; calls only
 * enqueue kernels and can be captured into a CUDA graph). Besides:
 *   - Token counts are below 2^31.
 *   - Offsets: cu_seqlens / starts hold num_seqs + 1 token offsets; sequence s
 *     is tokens [starts[s], starts[s+1]). A sequence may be empty. Rows that no
 *     sequence holds (ahead of the first, behind the last): the training calls
 *     write zeros to their outputs and gradients, the packed calls leave
 *     the output as it was, or write zeros when zero_rest != 0.
 *   - Workspaces are device memory of at least the size that the matching
 *     *_workspace function returns, 16-byte aligned, and hold nothing between
 *     calls. Two calls that may run at the same time need two of them.
 *   - The same call on the same inputs gives the same bits.
 */
#ifndef GRETA_SSM_H
#define GRETA_SSM_H

#include "greta_dynconv.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Short causal depthwise convolution with static filters:
 *   pre[t, d] = bias[d] + sum_k w[k, d] x[t + k - W + 1, d]  (tap W-1 = current token)
 *   y[t, d]   = silu ? SiLU(pre) : pre
 *
 *   x     : [T, D], rows ldx elements apart (contiguous channels)
 *   w     : element (k, d) at w[k * sw_k + d * sw_d]; 1 <= W <= 16
 *   bias  : [D] or NULL
 *   y     : [T, D] contiguous
 *   cu_seqlens: NULL = one sequence of T tokens; int64 when cu_int64 != 0
 * History ahead of a sequence is zero.
 */
GRETA_API int greta_ssm_conv_fwd(int dtype, const void* x, int64_t ldx, const void* w, int64_t sw_k, int64_t sw_d,
                                 const void* bias, void* y, const void* cu_seqlens, int cu_int64, int64_t num_seqs,
                                 int64_t T, int64_t D, int64_t W, int silu, void* stream);

/* Gradients of greta_ssm_conv_fwd: dx [T, D], dw [W, D] (both contiguous, of
 * the element type) and dbias [D] (NULL when bias is NULL); dout [T, D]
 * contiguous. dw and dbias are summed in fp32; with GRETA_SSM_GRADS_F32 added to
 * `silu` they are fp32 arrays, which take the sums as they are (for parameters
 * that are kept in fp32 beside 16-bit activations). */
#define GRETA_SSM_GRADS_F32 0x100
GRETA_API int greta_ssm_conv_bwd(int dtype, const void* x, int64_t ldx, const void* w, int64_t sw_k, int64_t sw_d,
                                 const void* bias, const void* dout, void* dx, void* dw, void* dbias,
                                 const void* cu_seqlens, int cu_int64, int64_t num_seqs, int64_t T, int64_t D,
                                 int64_t W, int silu, void* workspace, int64_t workspace_bytes, void* stream);
GRETA_API int64_t greta_ssm_conv_bwd_workspace(int64_t T, int64_t D, int64_t W);

/*
 * The same convolution over a packed serving batch: history from each
 * request's cache slot, and the slot's last W-1 inputs written back (bit-exact
 * copies), in one launch. state, slots, has_initial, starts (int32) and
 * error_flags as in greta_dynconv_packed_state; a request without tokens
 * leaves its slot as it was. Requests of one batch have different slots.
 *
 * A batch of few rows more than requests is taken for a decode step, whose
 * requests are walked token by token. A table of mostly empty requests may hide a
 * long one in as many rows: GRETA_SSM_LONGEST(n) added to `zero_rest` tells that
 * no request has more than n tokens (below 2^22; 0: not known), and the choice
 * goes by that. Results do not depend on it.
 */
#define GRETA_SSM_LONGEST(n) ((n) << 8)
GRETA_API int greta_ssm_conv_packed(int dtype, const void* x, int64_t ldx, const void* w, int64_t sw_k, int64_t sw_d,
                                    const void* bias, void* y, void* state, int64_t num_slots, int64_t s_slot,
                                    int64_t s_d, int64_t s_h, const int32_t* starts, const int32_t* slots,
                                    const int8_t* has_initial, int64_t num_reqs, int64_t T, int64_t D, int64_t W,
                                    int silu, int zero_rest, int32_t* error_flags, void* stream);

/*
 * Selective state-space scan. Per token, with f = d / (D / F):
 *   dt     = delta[t, d] + delta_bias[d], through softplus when `softplus`
 *   h[n]   = exp(dt A[d, n]) h[n] + dt u[t, d] B[t, f, n]
 *   y      = sum_n C[t, f, n] h[n] + skip[d] u[t, d]
 *   out    = gate ? y SiLU(gate[t, d]) : y
 *
 *   u, delta, gate : [T, D] of the element type, rows ldu / ldd / ldg apart
 *   B, C           : [T, F, N] of the element type, token rows ldb / ldc apart
 *                    (each token's F x N block contiguous)
 *   A              : fp32 [D, N] contiguous; skip, delta_bias: fp32 [D] or NULL
 *   out            : [T, D] contiguous
 *   F divides D; 1 <= N <= 128. States are fp32.
 *   saved          : NULL, or fp32 [T / 8 + 1, D, N]: the states ahead of every
 *                    8th token of the stream, for the backward
 *   ranges         : 0, or the number of token ranges to cut the stream into
 *                    (tests and tuning; results differ by rounding only)
 */
GRETA_API int greta_ssm_scan_fwd(int dtype, const void* u, int64_t ldu, const void* delta, int64_t ldd,
                                 const void* gate, int64_t ldg, const void* B, int64_t ldb, const void* C,
                                 int64_t ldc, const float* A, const float* skip, const float* delta_bias, void* out,
                                 float* saved, const void* cu_seqlens, int cu_int64, int64_t num_seqs, int64_t T,
                                 int64_t D, int64_t N, int64_t F, int softplus, int ranges, void* workspace,
                                 int64_t workspace_bytes, void* stream);

/*
 * The scan over a packed serving batch, prompts and single tokens in any mix:
 * each request starts from its cache slot's state (zeros without
 * has_initial or slot) and leaves its last state there. state: fp32
 * [num_slots, D, N] through element strides; starts (int32), slots,
 * has_initial, error_flags as in greta_dynconv_packed_state. A request without
 * tokens leaves its slot as it was. Requests of one batch have different
 * slots. zero_rest with GRETA_SSM_LONGEST as in greta_ssm_conv_packed.
 */
GRETA_API int greta_ssm_scan_packed(int dtype, const void* u, int64_t ldu, const void* delta, int64_t ldd,
                                    const void* gate, int64_t ldg, const void* B, int64_t ldb, const void* C,
                                    int64_t ldc, const float* A, const float* skip, const float* delta_bias,
                                    void* out, float* state, int64_t num_slots, int64_t s_slot, int64_t s_d,
                                    int64_t s_n, const int32_t* starts, const int32_t* slots,
                                    const int8_t* has_initial, int64_t num_reqs, int64_t T, int64_t D, int64_t N,
                                    int64_t F, int softplus, int zero_rest, int ranges, int32_t* error_flags,
                                    void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Gradients of greta_ssm_scan_fwd, from its inputs, `saved` and dout [T, D]
 * (contiguous): du, ddelta, dgate [T, D], dB, dC [T, F, N] contiguous of the
 * element type; dA [D, N], dskip, ddelta_bias [D] fp32. dgate, dskip and
 * ddelta_bias may be NULL where their input is.
 */
GRETA_API int greta_ssm_scan_bwd(int dtype, const void* u, int64_t ldu, const void* delta, int64_t ldd,
                                 const void* gate, int64_t ldg, const void* B, int64_t ldb, const void* C,
                                 int64_t ldc, const float* A, const float* skip, const float* delta_bias,
                                 const float* saved, const void* dout, void* du, void* ddelta, void* dgate, void* dB,
                                 void* dC, float* dA, float* dskip, float* ddelta_bias, const void* cu_seqlens,
                                 int cu_int64, int64_t num_seqs, int64_t T, int64_t D, int64_t N, int64_t F,
                                 int softplus, int ranges, void* workspace, int64_t workspace_bytes, void* stream);
GRETA_API int64_t greta_ssm_scan_bwd_workspace(int64_t num_seqs, int64_t T, int64_t D, int64_t N, int64_t F,
                                               int ranges);

/* Bytes of workspace of greta_ssm_scan_fwd and greta_ssm_scan_packed (the same `ranges`;
 * packed: 0 for greta_ssm_scan_fwd, 1 for greta_ssm_scan_packed, which needs
 * none for a batch of single tokens; with the GRETA_SSM_LONGEST of that call). */
GRETA_API int64_t greta_ssm_scan_workspace(int packed, int64_t num_seqs, int64_t T, int64_t D, int64_t N, int64_t F,
                                           int ranges);

/*
 * Metadata of a packed serving batch in one launch, from the lengths of the
 * requests on the device: request i adds query_lens[i] tokens to
 * context_lens[i] cached ones (negative lengths count as 0).
 *
 *   starts      [num_reqs + 1] token offsets, none above T (the rows of the
 *               packed tensors: tokens past them are dropped)
 *   has_initial [num_reqs] 1 where context_lens > 0
 *   seq_idx     [T] request of each token, -1 behind the last
 *   positions   [T] position of each token in its request, 0 behind the last
 * With block_tables (int32 [num_reqs, width], rows s_row apart; NULL: none of
 * the following), each request's table grows by the blocks that its new tokens
 * begin, taken in request order from the front of free_blocks [num_free]:
 *   slot_map    [T] block * block_size + position % block_size, -1 where there
 *               is no block (behind the last token, past the table's width, or
 *               the list ran out; such table entries become -1)
 *   blocks_used [1] blocks asked for (above num_free: the list ran out), for all
 *               of query_lens: blocks that only tokens past T would begin, or that
 *               lie past the table's width, are counted and stand in no table
 * At most 16384 requests.
 */
GRETA_API int greta_ssm_batch_metadata(const int32_t* query_lens, const int32_t* context_lens, int64_t num_reqs,
                                       int64_t T, int32_t* starts, int8_t* has_initial, int32_t* seq_idx,
                                       int64_t* positions, int32_t* block_tables, int64_t s_row, int64_t width,
                                       int64_t block_size, const int32_t* free_blocks, int64_t num_free,
                                       int64_t* slot_map, int32_t* blocks_used, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* GRETA_SSM_H */
