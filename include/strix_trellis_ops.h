/*
 * Operators around the trellis linear layers: an 8-bit integer linear layer,
 * the norms and the residual sum between two blocks, and the log
 * probabilities of tokens behind the output head.  MI355X extensions of the
 * strix_trellis C ABI with no counterpart in the reference header; contexts,
 * streams, status codes and the descriptor conventions are that ABI's.
 *
 * Every call runs on the calling thread's current device, which has to be the
 * context's, and only enqueues work on the given stream.  Nothing here
 * allocates device memory except strix_amd_int8_weights_prepare.  An operator
 * is called directly, or prepared once as a plan (validated at creation;
 * submission allocates, copies, synchronises and queries nothing, so it can
 * be captured into a graph).  Calls and submissions that share a workspace or
 * an output must be ordered by the caller.  Weights and plans hold their context
 * (it is not destroyed before them), plans their weights; every buffer is the
 * caller's and has to outlive the work on it, captured graphs included.
 */
#ifndef STRIX_TRELLIS_OPS_H
#define STRIX_TRELLIS_OPS_H

#include "strix_trellis.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of the views below: STRIX_DTYPE_F16, _BF16, _F32, and: */
#define STRIX_AMD_DTYPE_I8 UINT32_C(16)

/* Rows of device memory: element [r][c] at data + (r * row_stride + c) * size.
 * row_stride >= width where rows > 1; data aligned to the element size;
 * buffer_bytes counts from data.  An optional view that is absent is all
 * zeros (struct_size included). */
typedef struct strix_amd_view {
    uint32_t struct_size;
    uint32_t abi_version;
    void *data;
    uint64_t buffer_bytes;
    uint32_t dtype;
    uint32_t flags;          /* 0 */
    uint64_t rows;
    uint64_t width;
    uint64_t row_stride;
    uint64_t reserved[2];
} strix_amd_view;

/* Contiguous device memory; absent: NULL and 0 bytes. */
typedef struct strix_amd_buffer {
    void *data;
    uint64_t bytes;
} strix_amd_buffer;

/* A prepared operator. */
typedef struct strix_amd_op_plan_impl *strix_amd_op_plan;
strix_status strix_amd_op_plan_submit(strix_amd_op_plan plan);
strix_status strix_amd_op_plan_destroy(strix_amd_op_plan plan);

/* ---- 8-bit integer linear layer ----
 *   y[m][n] = alpha * (s[m] * t[n] * sum_i q[m][i] * w[n][i] + bias[n]) + beta * y_old[m][n]
 * w int8 [N][I] with the scale t[n] of each output channel, q int8 with the
 * scale s[m] of each token.  Activations in F32, F16 or BF16 are rounded in
 * the call:
 *   s[m] = max(RN32(max_i |x[m][i]| / 127), 2^-126)   q[m][i] = x[m][i] / s[m] to the nearest integer, ties to even
 * (exactly: the quotient itself is rounded once).  A row with an infinity or
 * a NaN gives NaN outputs in that row alone.  The integer sum is exact; the
 * rest is FP32, rounded once to the output's type, so a row's bits do not
 * depend on the other rows or on their number.  s t sum is infinite only where
 * that product is past FP32's range itself, whatever s and t are.
 *
 * Weights are prepared from device memory: I8 with their scales, or F32, F16
 * or BF16 rounded per channel by the rule above (a channel with an infinity
 * or a NaN gives NaN outputs).  Preparation copies into one private
 * allocation, padded to 32 channels and 128 inputs, and synchronises the
 * stream.  1 <= N <= 2^24, 1 <= I <= 131071 (the exact sum fits 32 bits). */
#define STRIX_AMD_INT8_MAX_INPUT UINT32_C(131071)
#define STRIX_AMD_INT8_MAX_OUTPUT UINT32_C(16777216)
typedef struct strix_amd_int8_weights_impl *strix_amd_int8_weights;
typedef struct strix_amd_int8_weights_desc {
    uint32_t struct_size;
    uint32_t abi_version;
    strix_amd_view weights;      /* [N][I] */
    strix_amd_buffer scales;     /* F32 [N] with I8 weights, else absent */
    strix_amd_buffer bias;       /* F32 [N] or absent */
    uint64_t reserved[4];
} strix_amd_int8_weights_desc;
strix_status strix_amd_int8_weights_prepare(strix_context context, const strix_amd_int8_weights_desc *desc,
    const strix_stream *stream, strix_amd_int8_weights *out);
strix_status strix_amd_int8_weights_destroy(strix_amd_int8_weights weights);

/* rows 0..INT_MAX.  input: I8 with input_scales F32 [rows], or F32 / F16 /
 * BF16 without; output F32 / F16 / BF16.  beta == 0 never reads the old
 * output.  The workspace (256-byte aligned) holds the rounded activations.
 * Input, output, workspace and weights must not overlap. */
typedef struct strix_amd_int8_linear_desc {
    uint32_t struct_size;
    uint32_t abi_version;
    strix_amd_int8_weights weights;
    strix_amd_view input;            /* [rows][I] */
    strix_amd_buffer input_scales;
    strix_amd_view output;           /* [rows][N] */
    float alpha;
    float beta;
    strix_amd_buffer workspace;
    uint64_t reserved[4];
} strix_amd_int8_linear_desc;
strix_status strix_amd_int8_linear_workspace_bytes(strix_context context,
    const strix_amd_int8_linear_desc *desc, uint64_t *out_bytes);
strix_status strix_amd_int8_linear(strix_context context, const strix_amd_int8_linear_desc *desc,
    const strix_stream *stream);
strix_status strix_amd_int8_linear_plan_create(strix_context context, const strix_amd_int8_linear_desc *desc,
    const strix_stream *stream, strix_amd_op_plan *out);

/* ---- norms and residual sum between two blocks ----
 *   t = post_weight ? norm(block) * (weight_offset + post_weight) + post_bias : block
 *   u = residual_scale * residual + block_scale * channel_scale * act(gate) * t        -> hidden
 *   n = norm(u) * (weight_offset + pre_weight) + pre_bias                              -> normed
 * per row of `width` channels, with norm(v) = v / sqrt(mean(v^2) + eps) (RMS)
 * or (v - mean(v)) / sqrt(mean((v - mean(v))^2) + eps) (LAYER).  A part that
 * is absent drops out: no block or no residual: that term is 0 (one of the
 * two is needed); no gate or channel_scale: 1; no bias: 0.  hidden and normed
 * are each optional, one is needed; normed needs pre_weight and the reverse.
 * n is computed from u in FP32, before u is rounded to the views' type; sums are
 * FP32, and those past its range are taken of the row times a power of two.
 * All views have one type (F32, F16 or BF16) and one width, 1..32768; the
 * gate is [rows][width], [1][width], [rows][1] or [1][1].  Vectors are F32
 * [width].  hidden and normed may each be exactly the memory of block or of
 * residual (same data and row stride), which is then overwritten; any other
 * overlap of an output with a view or a vector is refused. */
#define STRIX_AMD_NORM_RMS UINT32_C(0)
#define STRIX_AMD_NORM_LAYER UINT32_C(1)
#define STRIX_AMD_GATE_LINEAR UINT32_C(0)
#define STRIX_AMD_GATE_SIGMOID UINT32_C(1)
#define STRIX_AMD_NORM_MAX_WIDTH UINT32_C(32768)
typedef struct strix_amd_block_norm_desc {
    uint32_t struct_size;
    uint32_t abi_version;
    strix_amd_view block;
    strix_amd_view residual;
    strix_amd_view gate;
    strix_amd_view hidden;
    strix_amd_view normed;
    strix_amd_buffer post_weight;
    strix_amd_buffer post_bias;
    strix_amd_buffer pre_weight;
    strix_amd_buffer pre_bias;
    strix_amd_buffer channel_scale;
    uint32_t norm;               /* STRIX_AMD_NORM_* */
    uint32_t gate_activation;    /* STRIX_AMD_GATE_* */
    float eps;                   /* > 0, finite */
    float weight_offset;
    float residual_scale;
    float block_scale;
    uint64_t reserved[4];
} strix_amd_block_norm_desc;
strix_status strix_amd_block_norm(strix_context context, const strix_amd_block_norm_desc *desc,
    const strix_stream *stream);
strix_status strix_amd_block_norm_plan_create(strix_context context, const strix_amd_block_norm_desc *desc,
    const strix_stream *stream, strix_amd_op_plan *out);

/* ---- log probabilities of tokens ----
 * Per row of `vocab` logits, l = scale * logits, p = softmax(l), in nats:
 *   logprobs[r]     log p of tokens[r]
 *   ranks[r]        tokens ahead of tokens[r]: a larger logit, or the same one at a lower id
 *   entropy[r]      -sum p log p
 *   top_ids[r][j], top_logprobs[r][j]   the `top` first tokens in that order
 * Logits of -inf (masked tokens) have p = 0: log probability -inf, last in
 * the order, by id.  A row with no logit above -inf, with a NaN or with a
 * +inf has no distribution: its floats are NaN and its integers -1.  A token
 * outside 0..vocab-1 gives NaN and -1 for that row's logprobs and ranks alone.
 * Sums and logarithms are FP32.  A row's results do not depend on the other rows;
 * the last bits of its floats may depend on their number (the order of the sums
 * does).
 * Each output is optional, at least one is needed; logprobs and ranks need
 * tokens.  0 <= top <= min(vocab, STRIX_AMD_MAX_TOP); top_ids and
 * top_logprobs need top > 0.  The workspace is 256-byte aligned. */
#define STRIX_AMD_MAX_TOP UINT32_C(64)
typedef struct strix_amd_token_logprobs_desc {
    uint32_t struct_size;
    uint32_t abi_version;
    strix_amd_view logits;           /* [rows][vocab], F32 / F16 / BF16 */
    strix_amd_buffer tokens;         /* int32 [rows] */
    strix_amd_buffer logprobs;       /* F32 [rows] */
    strix_amd_buffer ranks;          /* int32 [rows] */
    strix_amd_buffer entropy;        /* F32 [rows] */
    strix_amd_buffer top_ids;        /* int32 [rows][top] */
    strix_amd_buffer top_logprobs;   /* F32 [rows][top] */
    uint32_t top;
    float scale;                     /* 2^-16 .. 2^16: 1 / temperature */
    strix_amd_buffer workspace;
    uint64_t reserved[4];
} strix_amd_token_logprobs_desc;
strix_status strix_amd_token_logprobs_workspace_bytes(strix_context context,
    const strix_amd_token_logprobs_desc *desc, uint64_t *out_bytes);
strix_status strix_amd_token_logprobs(strix_context context, const strix_amd_token_logprobs_desc *desc,
    const strix_stream *stream);
strix_status strix_amd_token_logprobs_plan_create(strix_context context,
    const strix_amd_token_logprobs_desc *desc, const strix_stream *stream, strix_amd_op_plan *out);

#ifdef __cplusplus
}
#endif
#endif /* STRIX_TRELLIS_OPS_H */
