/*
 * isa_train.h - C ABI of what a training step needs around a transformer's blocks
 * (libisa_block_hip.so, gfx950): embeddings with their tables' gradients, dropout from a
 * counter-based generator, alone and in the norm's residual add, and two losses of tuning a
 * model: the clipped policy loss and the preference loss of pairs.
 *
 * Conventions, element types and errors (isa_block_last_error) are those of isa_block.h.
 */
#ifndef ISA_TRAIN_H
#define ISA_TRAIN_H

#include "isa_block.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ISA_TRAIN_ABI_VERSION 1

int isa_train_abi_version(void);

/* ---- embedding -------------------------------------------------------------------------
 *   y_t = round(scale weight[id_t] + places[place_t])
 * ids [tokens]; without `place_ids` token t stands at place t mod period. A row whose id or place is
 * outside its table is NaN. */
typedef struct isa_train_embedding {
    int type; /* of the tables, y and the gradients */
    int64_t tokens, dim;
    int64_t vocab, weight_stride; /* rows of weight, weight_stride elements apart */
    const int64_t* ids;
    const void* weight;
    float scale;
    int64_t places, places_stride; /* rows of the second table; 0: none */
    const int64_t* place_ids;      /* [tokens], or null */
    int64_t period;                /* of a second table without place_ids: >= 1, divides tokens */
    const void* place_weight;
} isa_train_embedding;
#define ISA_TRAIN_EMBEDDING_MAX_ROWS (1 << 24) /* of a table */
#define ISA_TRAIN_EMBEDDING_MAX_DIM (1 << 20)  /* tokens: at most 2^30 */

/* y [tokens][dim]. For a backward call: lists (256-byte aligned), which the call fills with the tokens of each row of
 * the tables whose gradient will be asked for (weight, places: 0 or 1), without those whose id is `skip` (-1: none) or
 * whose id or place is outside its table; else null, 0, 0. */
size_t isa_train_embedding_lists(const isa_train_embedding* e, int weight, int places);
int isa_train_embedding_forward(const isa_train_embedding* e, void* y, int weight, int places, int64_t skip,
                                void* lists, size_t lists_bytes, void* stream);

/* The tables' gradients of grad_y [tokens][dim], in fp32 with each row rounded once:
 *   grad_weight [vocab][dim]: scale (sum of grad_y_t over a row's list),  grad_places [places][dim]: the sum alone
 * e, ids and place_ids as they were in the forward call that filled lists, with the same `weight` and `places` here as
 * listed_weight and listed_places. Either gradient may be null: not computed. The tables are not read. */
size_t isa_train_embedding_backward_workspace(const isa_train_embedding* e, int weight, int places);
int isa_train_embedding_backward(const isa_train_embedding* e, const void* lists, size_t lists_bytes,
                                 const void* grad_y, void* grad_weight, void* grad_places, int listed_weight,
                                 int listed_places, void* workspace, size_t workspace_bytes, void* stream);

/* ---- dropout -----------------------------------------------------------------------------
 * Element (r, c) of [rows][dim] is dropped iff its 16-bit number is below `threshold`; what is kept is multiplied
 * by 65536 / (65536 - threshold). The number: Philox4x32 with 10 rounds of
 *   key seed[0],  counter {r ceil(dim / 8) + c / 8, seed[1] + site}   (64-bit numbers, lower words first)
 * gives eight, lower halves of words first; c mod 8 picks one. The result of a dropped element is 0, whatever
 * it held. */
typedef struct isa_train_dropout {
    const int64_t* seed; /* [2], device memory */
    int64_t site;
    int threshold; /* 0 .. 65536 */
} isa_train_dropout;

/* y [rows][dim] of x, rows x_stride apart; a gradient's dropout is the same call. */
int isa_train_dropout_apply(const isa_train_dropout* drop, int type, int64_t rows, int64_t dim, const void* x,
                            int64_t x_stride, void* y, void* stream);

/* isa_block_norm_forward and _backward with h = round(residual + dropout(x)). x, h and both gradients must be
 * set; grad_x has x_type. Workspace as isa_block_norm_backward_workspace. */
int isa_train_dropout_norm_forward(const isa_block_norm* norm, const isa_train_dropout* drop, const void* x,
                                   int64_t x_stride, const void* residual, int64_t residual_stride, void* y, void* h,
                                   float* mean, float* rstd, void* stream);
int isa_train_dropout_norm_backward(const isa_block_norm* norm, const isa_train_dropout* drop, const void* grad_y,
                                    const void* grad_h, const void* h, int64_t h_stride, const float* mean,
                                    const float* rstd, void* grad_x, void* grad_residual, void* grad_weight,
                                    void* grad_bias, void* workspace, size_t workspace_bytes, void* stream);

/* ---- clipped policy loss -----------------------------------------------------------------
 * Row r of the logits and its action a (`loss.targets`; ignore_index as there), l = x_a - log(sum_j exp(x_j)):
 *   ratio = exp(l - old_logp),  s = min(ratio A, clamp(ratio, low, high) A)
 *   loss_r = -s + kl (exp(ref_logp - l) - (ref_logp - l) - 1)
 *   slope_r = dloss_r / dl = -[ratio A <= clamp(ratio, low, high) A] ratio A + kl (1 - exp(ref_logp - l))
 * An action outside the vocabulary makes its row NaN. */
typedef struct isa_train_policy {
    isa_block_loss loss;
    const float *old_logp, *advantages; /* [rows] */
    const float* ref_logp;              /* [rows], or null with kl 0 */
    float low, high, kl;                /* 0 <= low <= high */
} isa_train_policy;

/* out: [1], or [rows] with ISA_BLOCK_NONE. logp [rows]: l, 0 in ignored rows. stats [rows][2], slope [rows] and
 * count [1] are for the backward call, or all null. Workspace as isa_block_loss_workspace. */
int isa_train_policy_forward(const isa_train_policy* p, int reduction, float* out, float* logp, float* stats,
                             float* slope, float* count, void* workspace, size_t workspace_bytes, void* stream);
/* grad_logits (rows grad_stride apart) = slope (one-hot - softmax) times grad_out as in isa_block_loss_backward */
int isa_train_policy_backward(const isa_block_loss* loss, int reduction, const float* stats, const float* slope,
                              const float* count, const float* grad_out, void* grad_logits, int64_t grad_stride,
                              void* stream);
/* The mean loss and grad_scale times its gradient in one pass over the logits. */
int isa_train_policy_with_grad(const isa_train_policy* p, float grad_scale, float* out, float* logp,
                               void* grad_logits, int64_t grad_stride, void* workspace, size_t workspace_bytes,
                               void* stream);

/* ---- preference loss ---------------------------------------------------------------------
 * loss.rows = 2 pairs tokens: `pairs` chosen sequences, then as many rejected ones. L_s is the sum of l (above)
 * over a sequence's targets that are not ignored, held in 64 bits:
 *   m = beta ((L_chosen - ref_chosen) - (L_rejected - ref_rejected)),  loss_pair = log(1 + exp(-m)) */
typedef struct isa_train_preference {
    isa_block_loss loss;
    int64_t pairs, tokens;
    const float* ref_logp; /* [2 pairs] */
    float beta;
} isa_train_preference;

size_t isa_train_preference_workspace(const isa_train_preference* p);

/* out: [1], or [pairs] with ISA_BLOCK_NONE. logp [2 pairs]: L. stats [rows][2] and slope [2 pairs] (dloss_pair / dL)
 * are for the backward call, or both null. */
int isa_train_preference_forward(const isa_train_preference* p, int reduction, float* out, float* logp, float* stats,
                                 float* slope, void* workspace, size_t workspace_bytes, void* stream);
int isa_train_preference_backward(const isa_train_preference* p, int reduction, const float* stats,
                                  const float* slope, const float* grad_out, void* grad_logits, int64_t grad_stride,
                                  void* stream);
/* The mean loss and grad_scale times its gradient. */
int isa_train_preference_with_grad(const isa_train_preference* p, float grad_scale, float* out, float* logp,
                                   void* grad_logits, int64_t grad_stride, void* workspace, size_t workspace_bytes,
                                   void* stream);

#ifdef __cplusplus
}
#endif
#endif
