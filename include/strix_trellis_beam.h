/*
 * Decoding with several beams: the selection of their continuations behind the
 * output head, and the reordering of their states.  MI355X extensions of the
 * strix_trellis C ABI beside strix_trellis_ops.h, whose conventions they follow:
 * contexts, streams, views, buffers, plans (strix_amd_op_plan_submit and
 * _destroy), workspaces, what has to outlive what, and which calls the caller has
 * to order.
 */
#ifndef STRIX_TRELLIS_BEAM_H
#define STRIX_TRELLIS_BEAM_H

#include "strix_trellis_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

#define STRIX_AMD_MAX_BEAMS UINT32_C(64)

/* ---- selection ----
 * Rows of logits belong to prompts of `beams` consecutive rows.  A beam b with a finite score offers
 * every token v at
 *   c(b, v) = scores[b] + log p(v),   p = softmax(scale * logits[b])
 * (logits of -inf have p = 0), or, where `finished` is not 0, the token `pad` alone at its score.  A
 * beam whose score is not finite offers nothing; nor does one that is not finished and whose logits
 * hold a NaN, a +inf, or none above -inf.  Per prompt, the `keep` largest of these, equal ones by the lower
 * beam, then the lower token:
 *   next_scores[p][j] = c    parents[p][j] = b (0..beams-1)    tokens[p][j] = v
 * Candidates of -inf are none, nor are those whose c is -inf in FP32 (masks of a type's lowest value with
 * a scale above 1); places that are left have -inf, -1 and -1.  Values are compared as FP64
 * sums of FP32 statistics: tokens of two beams whose values differ by less than about 1e-6, or by less
 * than FP64 holds at their size, may change places.  1 <= beams <= 64, 1 <= keep <= 64; rows a multiple
 * of beams.  The workspace is 256-byte aligned.  Outputs and workspace overlap nothing. */
typedef struct strix_amd_beam_select_desc {
    uint32_t struct_size;
    uint32_t abi_version;
    strix_amd_view logits;           /* [prompts * beams][vocab], F32 / F16 / BF16 */
    strix_amd_buffer scores;         /* F32 [prompts * beams] */
    strix_amd_buffer finished;       /* int32 [prompts * beams] or absent */
    strix_amd_buffer next_scores;    /* F32 [prompts][keep] */
    strix_amd_buffer parents;        /* int32 [prompts][keep] */
    strix_amd_buffer tokens;         /* int32 [prompts][keep] */
    uint32_t beams;
    uint32_t keep;
    int32_t pad;
    float scale;                     /* 2^-16 .. 2^16: 1 / temperature */
    strix_amd_buffer workspace;
    uint64_t reserved[4];
} strix_amd_beam_select_desc;
strix_status strix_amd_beam_select_workspace_bytes(strix_context context, const strix_amd_beam_select_desc *desc,
    uint64_t *out_bytes);
strix_status strix_amd_beam_select(strix_context context, const strix_amd_beam_select_desc *desc,
    const strix_stream *stream);
strix_status strix_amd_beam_select_plan_create(strix_context context, const strix_amd_beam_select_desc *desc,
    const strix_stream *stream, strix_amd_op_plan *out);

/* ---- reordering ----
 *   target[o][p * beams + b][i] = source[o][p * beams + parents[p][b]][i]
 * for pieces of `bytes` bytes, piece [o][r][i] at data + o * strides[0] + r * strides[1] + i * strides[2]
 * (a cache [layers][rows][heads][length * size], of any capacity, is moved up to its length).  A parent
 * outside 0..beams-1 is the row itself.  `target` is `source` itself, with the same strides: rows that
 * are their own parents are then not touched; or memory that shares no byte with it.  Pieces
 * of the target do not overlap each other, and its dimensions lie within one another: with the strides in
 * ascending order each is at least what the piece and the dimensions before it span (another layout is an
 * unsupported format).  Strides of a dimension of one do not count.
 * 1 <= beams <= 64; source and target of any alignment. */
typedef struct strix_amd_states {
    void *data;
    uint64_t buffer_bytes;
    uint64_t strides[3];     /* bytes: outer, row, inner */
} strix_amd_states;
typedef struct strix_amd_beam_reorder_desc {
    uint32_t struct_size;
    uint32_t abi_version;
    strix_amd_buffer parents;        /* int32 [prompts][beams] */
    strix_amd_states source;
    strix_amd_states target;
    uint64_t prompts;
    uint64_t outer;
    uint64_t inner;
    uint64_t bytes;
    uint32_t beams;
    uint32_t flags;                  /* 0 */
    uint64_t reserved[4];
} strix_amd_beam_reorder_desc;
strix_status strix_amd_beam_reorder(strix_context context, const strix_amd_beam_reorder_desc *desc,
    const strix_stream *stream);
strix_status strix_amd_beam_reorder_plan_create(strix_context context, const strix_amd_beam_reorder_desc *desc,
    const strix_stream *stream, strix_amd_op_plan *out);

#ifdef __cplusplus
}
#endif
#endif /* STRIX_TRELLIS_BEAM_H */
