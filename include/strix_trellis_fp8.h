/*
 * Layers in 8-bit floating point (e4m3: 4 exponent bits, 3 mantissa bits,
 * largest value 448, no infinities) with a scale for each block of 128 x 128
 * weights: a linear layer, and the gated half of a feed-forward block.  MI355X
 * extensions of the strix_trellis C ABI beside strix_trellis_ops.h, whose
 * conventions they follow: contexts, streams, views, buffers, plans
 * (strix_amd_op_plan_submit and _destroy), workspaces, what has to outlive what,
 * and which calls the caller has to order.
 */
#ifndef STRIX_TRELLIS_FP8_H
#define STRIX_TRELLIS_FP8_H

#include "strix_trellis_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element type of a view beside those of strix_trellis_ops.h. */
#define STRIX_AMD_DTYPE_E4M3 UINT32_C(17)

/* ---- weights ----
 * w[n][i] t[n / 128][i / 128]: e4m3 [N][I] with F32 scales [ceil(N / 128)][ceil(I / 128)], or F32, F16
 * or BF16 weights, which preparation rounds:
 *   t = max(RN32(max |w| / 448), 2^-126) over the block     q = e4m3(RN32(w * RN32(1 / t))), ties to even
 * (a block with an infinity or a NaN gives NaN outputs in its channels).  With `up`, a second matrix of
 * the same shape and type, the handle is a pair: the gate (`weights`) and up projections of one
 * feed-forward block.  Preparation copies into one private allocation, padded to 32 channels and
 * 128 inputs, and synchronises the stream.  1 <= N <= 2^24, 1 <= I <= 2^17. */
#define STRIX_AMD_FP8_MAX_INPUT UINT32_C(131072)
#define STRIX_AMD_FP8_MAX_OUTPUT UINT32_C(16777216)
typedef struct strix_amd_fp8_weights_impl *strix_amd_fp8_weights;
typedef struct strix_amd_fp8_weights_desc {
    uint32_t struct_size;
    uint32_t abi_version;
    strix_amd_view weights;        /* [N][I] */
    strix_amd_buffer scales;       /* with E4M3 weights, else absent */
    strix_amd_buffer bias;         /* F32 [N] or absent */
    strix_amd_view up;             /* [N][I] or absent */
    strix_amd_buffer up_scales;
    strix_amd_buffer up_bias;      /* present as `bias` is */
    uint64_t reserved[4];
} strix_amd_fp8_weights_desc;
strix_status strix_amd_fp8_weights_prepare(strix_context context, const strix_amd_fp8_weights_desc *desc,
    const strix_stream *stream, strix_amd_fp8_weights *out);
strix_status strix_amd_fp8_weights_destroy(strix_amd_fp8_weights weights);

/* ---- linear layer ----
 *   z[m][n] = sum over blocks b of (s[m][b] t[n / 128][b]) sum of q[m][i] w[n][i] over i in b
 *   y[m][n] = alpha * (z[m][n] + bias[n]) + beta * y_old[m][n]
 * Input rows are E4M3 with input_scales F32 [rows][ceil(I / 128)] (s), or F32, F16 or BF16, rounded in the
 * call by the rule above with a scale per row and block of 128 inputs.  A row with an infinity or a
 * NaN gives NaN outputs in that row alone.  Sums are FP32: a block's, then over the blocks with the
 * FP32 product s t; the result is rounded once to the output's type.  For F16 and BF16 outputs a block's
 * products may lose, of each eight neighbouring ones, what lies below 2^-13 of the largest (about 1e-5
 * of the block's sum).  A row's results do not depend on the other rows; the last bits may depend on
 * their number (the order of the sums does).
 * rows 0..INT_MAX; output F32, F16 or BF16.  beta == 0 never reads the old output.  The workspace is
 * 256-byte aligned.  Output and workspace overlap nothing. */
typedef struct strix_amd_fp8_linear_desc {
    uint32_t struct_size;
    uint32_t abi_version;
    strix_amd_fp8_weights weights;   /* not a pair */
    strix_amd_view input;            /* [rows][I] */
    strix_amd_buffer input_scales;
    strix_amd_view output;           /* [rows][N] */
    float alpha;
    float beta;
    strix_amd_buffer workspace;
    uint64_t reserved[4];
} strix_amd_fp8_linear_desc;
strix_status strix_amd_fp8_linear_workspace_bytes(strix_context context, const strix_amd_fp8_linear_desc *desc,
    uint64_t *out_bytes);
strix_status strix_amd_fp8_linear(strix_context context, const strix_amd_fp8_linear_desc *desc,
    const strix_stream *stream);
strix_status strix_amd_fp8_linear_plan_create(strix_context context, const strix_amd_fp8_linear_desc *desc,
    const strix_stream *stream, strix_amd_op_plan *out);

/* ---- gated half of a feed-forward block ----
 *   h[m][n] = act(z_gate[m][n] + bias[n]) * (z_up[m][n] + up_bias[n])
 * with z as above, SILU g / (1 + e^-g) and GELU g / 2 (1 + tanh(sqrt(2 / pi) (g + 0.044715 g^3))), in FP32.
 * Output F32, F16 or BF16, or E4M3 with output_scales F32 [rows][ceil(N / 128)]: h rounded by the rule
 * above, as the linear layer takes its input.  Otherwise as the linear layer. */
#define STRIX_AMD_GATED_SILU UINT32_C(0)
#define STRIX_AMD_GATED_GELU UINT32_C(1)
typedef struct strix_amd_fp8_gated_desc {
    uint32_t struct_size;
    uint32_t abi_version;
    strix_amd_fp8_weights weights;   /* a pair */
    strix_amd_view input;            /* [rows][I] */
    strix_amd_buffer input_scales;
    strix_amd_view output;           /* [rows][N] */
    strix_amd_buffer output_scales;  /* with an E4M3 output, else absent */
    uint32_t activation;             /* STRIX_AMD_GATED_* */
    uint32_t flags;                  /* 0 */
    strix_amd_buffer workspace;
    uint64_t reserved[4];
} strix_amd_fp8_gated_desc;
strix_status strix_amd_fp8_gated_workspace_bytes(strix_context context, const strix_amd_fp8_gated_desc *desc,
    uint64_t *out_bytes);
strix_status strix_amd_fp8_gated(strix_context context, const strix_amd_fp8_gated_desc *desc,
    const strix_stream *stream);
strix_status strix_amd_fp8_gated_plan_create(strix_context context, const strix_amd_fp8_gated_desc *desc,
    const strix_stream *stream, strix_amd_op_plan *out);

#ifdef __cplusplus
}
#endif
#endif /* STRIX_TRELLIS_FP8_H */
