/*
 * eif_hip_moe.h -- routing to experts on one MI355X: the choice of experts and their weights from a router's logits, the rows
 * sorted by expert as eif_hip_mx4_linear_grouped (eif_hip_mx.h) takes them, and the weighted sum of the experts' rows.
 *
 * No counterpart in the reference. As in eif_hip.h, pointers are DEVICE pointers unless a comment says otherwise, `stream` is a
 * hipStream_t (NULL = the null stream), calls are asynchronous on it and return 0 or a negative EIF_HIP_E_* code. The current
 * device must be the one that the memory and the stream belong to. Calls allocate nothing and keep nothing between them: they may be
 * captured into graphs, and any number of them may run at once as long as each has outputs and a workspace of its own. Strides are
 * in elements. No input may overlap an output (but `add` and `out` of eif_hip_moe_combine). Pointers are aligned to their
 * elements, else EIF_HIP_E_ARG. Results depend on the inputs alone, not on the order in which anything ran.
 */
#ifndef EIF_HIP_MOE_H
#define EIF_HIP_MOE_H

#include <stddef.h>
#include <stdint.h>

#include "eif_hip.h"
#include "eif_hip_mx.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { EIF_HIP_SCORE_SOFTMAX = 0, EIF_HIP_SCORE_SIGMOID = 1 };

/* How a token's experts are chosen (the struct is host memory, read during the call; bias is device memory). */
typedef struct eif_hip_moe_route_spec {
    int experts;        /* 1 .. 4096 */
    int top_k;          /* experts of a token, 1 .. min(experts, 64) */
    int score;          /* EIF_HIP_SCORE_* */
    const float *bias;  /* [experts], added to the scores for the choice alone, or NULL */
    int groups;         /* the experts form this many groups of experts / groups consecutive ones; 1 .. 64, a divisor of experts */
    int groups_kept;    /* groups whose experts may be chosen, 1 .. groups */
    int group_best;     /* a group is worth its best (1) or the sum of its two best (2) */
    int renormalise;    /* not 0: a token's weights are divided by their sum */
    float scale;        /* factor of the weights, finite */
} eif_hip_moe_route_spec;

/* Bytes of workspace that eif_hip_moe_sort and eif_hip_moe_route need for their sorted outputs (0: none, or sizes that they refuse). */
size_t eif_hip_moe_sort_bytes(int tokens, int top_k, int experts);

/* logits [tokens, ldl >= experts] of `type` (EIF_HIP_F32, _F16, _BF16; eif_hip_mx.h) -> ids [tokens, top_k] and weights
 * [tokens, top_k], a token's experts in the order of their choice.
 *   A logit of -inf or NaN, or a bias of -inf or NaN, shuts its expert out of the choice; +inf counts as the largest FP32 number.
 *   Score s: softmax over the token's logits (those of -inf and NaN count 0), or 1 / (1 + e^-l) (0 where e^-l is more than 64 bits
 *   hold, l below -709.78). Value v = s + bias. s and v are in 64 bits. Without a bias experts are compared by their logits, in whose
 *   order the scores are; else by v.
 *   Groups: a group is worth the largest of what its experts are compared by, or (group_best 2) the sum of the two largest v of its
 *   experts that may be chosen (of one, that one's); the groups_kept worth most keep their experts in the choice.
 *   The top_k best of the experts left are chosen. Equals go to the lowest index, of groups and of experts.
 *   Weight: s, divided by the sum of the chosen s where renormalise is set (softmax: over the chosen alone, which cannot vanish;
 *   sigmoid: 0 where the sum is 0), times scale, rounded to FP32 once.
 *   Where fewer than top_k experts are left, the places behind them have id -1 and weight 0.
 * tokens up to 2^25, tokens * top_k up to 2^30, else EIF_HIP_E_LIMIT.
 * offsets, row and slot (all or none; NULL: not sorted): as eif_hip_moe_sort makes them of ids, with its workspace. */
int eif_hip_moe_route(const void *logits, int type, int64_t ldl, int tokens, const eif_hip_moe_route_spec *spec, int32_t *ids,
                      float *weights, int32_t *offsets, int32_t *row, int32_t *slot, void *work, size_t work_bytes, void *stream);

/* Pairs of a token and an expert, ids [tokens, top_k], in order of their expert, a token's before the next one's:
 *   offsets [experts + 1]  pairs of the experts before each, and of all of them;
 *   row [tokens * top_k]   the token of the i-th pair in that order; what lies behind offsets[experts] is left as it was;
 *   slot [tokens * top_k]  the place of a pair in that order, -1 for an id outside of [0, experts), which has none.
 * offsets and row are what eif_hip_mx4_linear_grouped takes. A token may name an expert twice.
 * work: eif_hip_moe_sort_bytes bytes, aligned to 4 (NULL where that is 0), free once the call's work on the stream is done; fewer
 * bytes: EIF_HIP_E_ARG. experts 1 .. 4096, top_k 1 .. 4096, tokens * top_k up to 2^30, else EIF_HIP_E_LIMIT (below 1: EIF_HIP_E_ARG).
 * tokens = 0 writes offsets of 0. */
int eif_hip_moe_sort(const int32_t *ids, int tokens, int top_k, int experts, int32_t *offsets, int32_t *row, int32_t *slot, void *work,
                     size_t work_bytes, void *stream);

/* out[t] = add[t] + sum over k of weights[t, k] * y[slot[t, k]], k in order, FP32 sums, rounded once to `type`.
 *   y [rows, ldy] FP32, slot [tokens, top_k] (places outside of [0, rows) add nothing, whatever their weight), weights [tokens, top_k]
 *   or NULL (1), add [tokens, lda] FP32 or NULL (0), out [tokens, ldo] of `type`; add may be out itself (FP32, lda == ldo).
 * dim 1 .. 2^24 columns, tokens * top_k up to 2^30, tokens * ceil(dim / 256) up to 2^24 - 1, else EIF_HIP_E_LIMIT (below 1:
 * EIF_HIP_E_ARG). */
int eif_hip_moe_combine(const float *y, int64_t ldy, int rows, const int32_t *slot, const float *weights, int tokens, int top_k,
                        const float *add, int64_t lda, int dim, void *out, int type, int64_t ldo, void *stream);

#ifdef __cplusplus
}
#endif

#endif
