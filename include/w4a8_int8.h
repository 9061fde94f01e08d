/*
 * w4a8_int8.h - C ABI of the int8 (W8A8) operators for MI355X (gfx950), in libw4a8int8.so.
 *
 * The conventions are those of w4a8_moe.h (device pointers, sizes and a hipStream_t passed as void*; status codes;
 * caller-owned workspaces; nothing synchronises or allocates), whose status codes and types these entry points
 * share. The library is one of its own: a host without int8 checkpoints does not load it, and its error text is read
 * with w4a8_int8_last_error().
 *
 * Rows are int8 with one fp32 scale each, weights (N, K) or (E, N, K) int8 with one fp32 scale per output channel:
 *   out[m, n] = xs[m] * ws[n] * sum_k x[m, k] w[n, k],
 * the sum in whole numbers, the rest in fp32 (xs * ws first). Quantisation: a = max(absmax, 127 * 2^-100), q = the whole number nearest
 * to 127 v / a (ties to even), scale = a / 127; a row that holds an infinity or a NaN gets the scale NaN. No reference
 * counterpart (the reference serves int4 and E2M1 weights).
 */
#ifndef W4A8_INT8_H_
#define W4A8_INT8_H_

#include "w4a8_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define W4A8_DTYPE_INT8 3

W4A8_API int w4a8_int8_abi_version(void);

/* Message of the calling thread's last failed call into this library ("" if none). */
W4A8_API const char* w4a8_int8_last_error(void);

/* int8 rows q (rows, K) and scales (rows,) of x (rows, K) fp16 / bf16, or with silu_gate_up != 0 of silu(gate) * up of
 * x = [gate | up] (rows, 2 K), formed in fp32. x_stride: elements between rows. */
W4A8_API int w4a8_act_quant_int8(const void* x, int x_dtype, int64_t rows, int64_t K, int64_t x_stride, int silu_gate_up,
                                 int8_t* q, float* scales, void* stream);

/* Dense layer: out (M, N) fp16 / bf16 = x (M, K) times w (N, K) transposed + bias. x int8 with x_scales (M,), or fp16 /
 * bf16 (x_scales unused): quantised in the call, as w4a8_act_quant_int8 does. K a multiple of 16 up to 131071; rows of x
 * start at multiples of 16 bytes; x and w aligned to 16 bytes. bias (N,): null, fp32 (bias_is_f32 != 0) or of out's
 * type. */
W4A8_API size_t w4a8_int8_gemm_workspace_size(int x_dtype, int64_t M, int64_t K, int64_t N);
W4A8_API int w4a8_int8_gemm(const void* x, int x_dtype, const float* x_scales, int64_t M, int64_t K, int64_t x_stride,
                            const int8_t* w, const float* w_scales, int64_t N, const void* bias, int bias_is_f32, void* out,
                            int out_dtype, void* workspace, size_t workspace_bytes, void* stream);

/* The gated expert layer: out (T, H) = sum over a token's slots of topk_weights * (silu(gate) * up, quantised) times w2
 * transposed. x as above, rows contiguous; w13 (E, 2 inter, H) = [gate | up], w2 (E, H, inter); H and inter multiples of
 * 64. topk_ids (T, top_k) are global expert ids; with expert_map (num_global_experts entries, -1 = not local) they are
 * mapped to the E local experts. Slots without one contribute nothing. The slots' rows are summed in fp32, in the slots'
 * order: a token's output has the same bits in any batch. */
W4A8_API size_t w4a8_moe_int8_workspace_size(int64_t T, int64_t H, int64_t inter, int64_t E, int64_t top_k);
W4A8_API int w4a8_moe_int8_apply(const void* x, int x_dtype, const float* x_scales, int64_t T, int64_t H, int64_t inter,
                                 int64_t E, int64_t top_k, const int8_t* w13, const float* w13_scales, const int8_t* w2,
                                 const float* w2_scales, const float* topk_weights, const int32_t* topk_ids,
                                 const int32_t* expert_map, int64_t num_global_experts, void* out, int out_dtype,
                                 void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* W4A8_INT8_H_ */
