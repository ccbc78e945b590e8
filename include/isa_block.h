/*
 * isa_block.h - C ABI of the MI355X (gfx950) kernels of a transformer block around its FFN
 * (libisa_block_hip.so): layer norm with the residual add, attention with a sliding window
 * and sinks, and the cross-entropy, each with its gradients.
 *
 * Conventions (those of isa_ekv.h):
 *   - Plain pointers and sizes; device memory of the current HIP device. The caller owns all
 *     memory; a workspace starts at a 256-byte aligned address and need not be cleared.
 *   - `stream` is a hipStream_t passed as void*; every call only enqueues work on it,
 *     allocates nothing, reads nothing back and may be captured in a HIP graph.
 *   - Return value: 0, ISA_BLOCK_EINVAL (<0) for an invalid argument (nothing was
 *     enqueued), >0 for a hipError_t; isa_block_last_error() has the calling thread's message.
 *   - No sum uses atomics: the same call gives the same bits.
 *   - Strides count elements.
 */
#ifndef ISA_BLOCK_H
#define ISA_BLOCK_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ISA_BLOCK_ABI_VERSION 1
#define ISA_BLOCK_EINVAL (-1)

/* Element types */
#define ISA_BLOCK_F32 0
#define ISA_BLOCK_BF16 1
#define ISA_BLOCK_F16 2

int isa_block_abi_version(void);
const char* isa_block_last_error(void);

/* ---- layer norm ----------------------------------------------------------------------
 *   h = round(x + residual)            (round to `type`; h = residual without x)
 *   y = (h - mean(h)) * rstd * weight + bias,   rstd = 1 / sqrt(var(h) + eps)
 * mean and var over a row of `dim` elements (var without Bessel's correction), in fp32 from
 * the row's registers in two passes. dim <= ISA_BLOCK_NORM_MAX_DIM. */
#define ISA_BLOCK_NORM_MAX_DIM 16384

typedef struct isa_block_norm {
    int type;        /* residual, h, y and their gradients */
    int x_type;      /* x and its gradient: `type`, or a 16-bit type beside ISA_BLOCK_F32 */
    int weight_type; /* weight, bias and their gradients: `type` or ISA_BLOCK_F32 */
    int64_t rows, dim;
    float eps;
    const void* weight; /* [dim] */
    const void* bias;   /* [dim], or null: none */
} isa_block_norm;

/* x (or null) and residual: rows of dim elements, x_stride and residual_stride apart. y [rows][dim];
 * h [rows][dim], with x only; mean, rstd [rows] fp32, both null where no backward follows. */
int isa_block_norm_forward(const isa_block_norm* norm, const void* x, int64_t x_stride, const void* residual,
                           int64_t residual_stride, void* y, void* h, float* mean, float* rstd, void* stream);

size_t isa_block_norm_backward_workspace(int64_t rows, int64_t dim);

/* Gradients for grad_y [rows][dim] of y and, if not null, grad_h [rows][dim] of h:
 *   dn = grad_y * weight,  n = (h - mean) rstd
 *   grad_residual = rstd (dn - mean(dn) - n mean(dn n)) + grad_h       (grad_x is the same)
 *   grad_weight = sum over rows of grad_y n,  grad_bias = sum over rows of grad_y
 * grad_x: written where x_type differs from type, else null. grad_weight null: neither it nor
 * grad_bias is computed (no workspace needed). h: rows h_stride apart. */
int isa_block_norm_backward(const isa_block_norm* norm, const void* grad_y, const void* grad_h, const void* h,
                            int64_t h_stride, const float* mean, const float* rstd, void* grad_x, void* grad_residual,
                            void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes,
                            void* stream);

/* ---- attention with a sliding window and sinks ----------------------------------------
 * Sequence b has L = key_lengths[b] keys (all `keys` without key_lengths; values are held to
 * 0 .. keys). Its queries are its last tokens: query i stands at p = L - queries + i and sees
 * key j iff 0 <= j <= p and (j < sinks or p - j < window). Query heads g * heads / kv_heads up
 * to the next g share key head g.
 *   out = softmax(scale q k^T over the keys seen) v,  0 where no key is seen. */
typedef struct isa_block_attention {
    int type; /* of q, k, v, out and the gradients */
    int64_t batch, queries, keys, heads, kv_heads, head_dim;
    int64_t window; /* 0: none */
    int64_t sinks;
    float scale;                /* > 0 */
    const int32_t* key_lengths; /* [batch], or null */
    /* [batch][queries][heads][head_dim] and [batch][keys][kv_heads][head_dim] with the strides of
     * batch, token and head; a head's elements are adjacent. Pointers are 16-byte aligned and
     * strides multiples of 8 elements, those of tokens at least head_dim elements and under
     * 16 MiB; head_dim is a multiple of 8, at most ISA_BLOCK_ATTENTION_MAX_DIM. */
    const void *q, *k, *v;
    int64_t q_strides[3], k_strides[3], v_strides[3];
} isa_block_attention;
#define ISA_BLOCK_ATTENTION_MAX_DIM 128

size_t isa_block_attention_forward_workspace(const isa_block_attention* att);

/* out [batch][queries][heads][head_dim]. For a backward call: lse [batch][heads][queries][2] fp32 (two
 * numbers whose sum is the base-2 logarithm of the sum of a row's exponentials, the first -inf for
 * a row that sees nothing), and with 16-bit types rest, shaped and typed as out: what out's rounding
 * left. Both may be null. */
int isa_block_attention_forward(const isa_block_attention* att, void* out, void* rest, float* lse, void* workspace,
                                size_t workspace_bytes, void* stream);

size_t isa_block_attention_backward_workspace(const isa_block_attention* att);

/* Gradients of q, k, v (contiguous, shaped as they are) for grad_out, strides as q's. rest may be
 * null: grad_out . out then carries out's rounding. Keys that no
 * query sees get zeros. grad_k and grad_v are sums over the query heads that share a key head.
 * grad_q null: not computed; grad_k and grad_v both null: neither is. */
int isa_block_attention_backward(const isa_block_attention* att, const void* out, const void* rest,
                                 const float* lse, const void* grad_out, const int64_t grad_out_strides[3], void* grad_q, void* grad_k,
                                 void* grad_v, void* workspace, size_t workspace_bytes, void* stream);

/* ---- cross-entropy ---------------------------------------------------------------------
 *   row r: loss_r = log(sum_j exp(x_rj)) - x_r,target; 0 where target == ignore_index
 * A target outside 0 .. vocab - 1 that is not ignore_index makes its row's loss and gradients NaN.
 * rows <= 2^24 (they are counted in fp32). */
typedef struct isa_block_loss {
    int type; /* of the logits and their gradient */
    int64_t rows, vocab;
    int64_t ignore_index;
    const void* logits; /* rows logits_stride apart */
    int64_t logits_stride;
    const int64_t* targets; /* [rows] */
} isa_block_loss;

#define ISA_BLOCK_MEAN 0 /* over the rows that are not ignored (NaN where there is none) */
#define ISA_BLOCK_SUM 1
#define ISA_BLOCK_NONE 2

size_t isa_block_loss_workspace(const isa_block_loss* loss);

/* loss: [1], or [rows] with ISA_BLOCK_NONE. stats: [rows][2] {row's maximum, log of the sum of
 * exp(x - maximum)} and count [1] (rows not ignored, as a float), for the backward call, or both null. */
int isa_block_loss_forward(const isa_block_loss* loss, int reduction, float* out, float* stats, float* count,
                           void* workspace, size_t workspace_bytes, void* stream);

/* grad_logits (rows grad_stride apart) = (softmax - one-hot) * grad_out[0] (ISA_BLOCK_NONE:
 * grad_out[r]), with ISA_BLOCK_MEAN divided by count[0]; zeros in ignored rows. */
int isa_block_loss_backward(const isa_block_loss* loss, int reduction, const float* stats, const float* count,
                            const float* grad_out, void* grad_logits, int64_t grad_stride, void* stream);

/* The mean loss and grad_scale times its gradient in one pass over the logits. */
int isa_block_loss_with_grad(const isa_block_loss* loss, float grad_scale, float* out, void* grad_logits,
                             int64_t grad_stride, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
