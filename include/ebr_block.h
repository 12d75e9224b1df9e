/* C ABI of the energy network's fused pointwise blocks in libebr_attn.so (gfx950): rms_norm over the last dimension
 * and the SwiGLU activation, each with its backward and the backward of that backward, as the graded latent descent
 * differentiates the energy twice; the group norm with an activation, likewise; and the ends of a training step, the
 * embedding of tokens with its table's gradient and the distillation loss with its gradient.
 *
 * Tensors are contiguous rows of one dtype (EBR_DTYPE_F32, _BF16, _F16 or _F64). Arithmetic is fp32 (fp64 for fp64);
 * outputs are rounded once to the dtype. Conventions otherwise as in ebr_attn.h (error codes, streams, ownership).
 */
#ifndef EBR_BLOCK_H
#define EBR_BLOCK_H

#include <stdint.h>

#include "ebr_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* y = x / sqrt(mean(x^2) + eps) per row of C elements, statistics in fp32.
 * Replaces the reference's rms_norm (models/layers.py:37-42) in the energy blocks (models/attention.py:264-266). */
int ebr_block_rmsnorm(int dtype, int64_t rows, int C, float eps, const void* x, void* y, void* stream);

/* dx of y = rms_norm(x) given dy. */
int ebr_block_rmsnorm_bwd(int dtype, int64_t rows, int C, float eps, const void* x, const void* dy, void* dx,
                          void* stream);

/* As ebr_block_rmsnorm_bwd, plus a gradient that is already there: dx = round(round(dx) + acc). */
int ebr_block_rmsnorm_bwd_add(int dtype, int64_t rows, int C, float eps, const void* x, const void* dy,
                              const void* acc, void* dx, void* stream);

/* The residual sum and its norm: sum = round(x + r), y = rms_norm(sum). */
int ebr_block_add_rmsnorm(int dtype, int64_t rows, int C, float eps, const void* x, const void* r, void* sum, void* y,
                          void* stream);

/* Gradients of <c, dx> with respect to x (gx) and dy (gdy), dx being ebr_block_rmsnorm_bwd's output. */
int ebr_block_rmsnorm_bwd2(int dtype, int64_t rows, int C, float eps, const void* x, const void* dy, const void* c,
                           void* gx, void* gdy, void* stream);

/* y = silu(gate) * up for rows of gu = [gate | up] (2 I elements each), y rows of I.
 * Replaces the reference's SwiGLU activation (models/layers.py:74-84: gate_up_proj(x).chunk(2), silu(gate) * up). */
int ebr_block_swiglu(int dtype, int64_t rows, int I, const void* gu, void* y, void* stream);

/* dgu = [dgate | dup] of y given dy. */
int ebr_block_swiglu_bwd(int dtype, int64_t rows, int I, const void* gu, const void* dy, void* dgu, void* stream);

/* As ebr_block_swiglu_bwd, plus a gradient that is already there: dgu = round(round(dgu) + acc). */
int ebr_block_swiglu_bwd_add(int dtype, int64_t rows, int I, const void* gu, const void* dy, const void* acc,
                             void* dgu, void* stream);

/* Gradients of <c, dgu> with respect to gu (ggu, rows of 2 I) and dy (gdy, rows of I). */
int ebr_block_swiglu_bwd2(int dtype, int64_t rows, int I, const void* gu, const void* dy, const void* c, void* ggu,
                          void* gdy, void* stream);

/* out[i] = round(sum over s of part[s][i]) of S (2, 4, 8 or 16) fp32 partial products [S, n]; out in bf16 or fp16. */
int ebr_block_split_sum(int dtype, int S, int64_t n, const float* part, void* out, void* stream);

/* y[n, :] = round(scale * w[ids[n], :]) for N tokens and a table w [V, C], contiguous; a row of zeros for a token outside
 * [0, V). ids: int64 where ids64, else int32. wdtype and ydtype are equal, or fp32 and a 16-bit type. N below 2^31 - 4096,
 * C below 2^18. */
int ebr_block_embed(int wdtype, int ydtype, int ids64, int64_t N, int64_t V, int C, double scale, const void* ids,
                    const void* w, void* y, void* stream);

/* Bytes of scratch that ebr_block_embed_bwd needs (16-byte aligned), -1 for sizes or types that it refuses. */
int64_t ebr_block_embed_bwd_scratch(int wdtype, int64_t N, int64_t V, int C);

/* dw[v, :] = round(scale * sum of dy[n, :] over the n with ids[n] = v): the whole [V, C], rows without a token as zeros.
 * Sums are fp32 (fp64 for fp64), always in the same order. */
int ebr_block_embed_bwd(int wdtype, int ydtype, int ids64, int64_t N, int64_t V, int C, double scale, const void* ids,
                        const void* dy, void* dw, void* scratch, void* stream);

/* How rows' losses go together. */
enum { EBR_REDUCE_NONE = 0, EBR_REDUCE_SUM = 1, EBR_REDUCE_MEAN = 2 };

/* Distillation from the K (at most 1024) top logits of a teacher at a temperature T from 1e-15 to 1e15: with p the softmax
 * of a row's teacher / T over the entries whose ids lie in [0, V), and q the softmax of its logits / T, loss = T^2 sum_k p_k
 * (log p_k - log q_id_k). A row without an entry of positive probability has loss 0 and is not counted in the mean (0 if
 * none is).
 * logits: N rows of V, row_stride elements apart; teacher (of tdtype) and ids (int64 where ids64, else int32): contiguous
 * [N, K]. loss: fp32 (fp64 for fp64 logits), [N] for EBR_REDUCE_NONE, else one. stats: [N, 4] of loss's type, 16-byte
 * aligned, and scale: one of it (not for EBR_REDUCE_NONE), both for the backward. */
int ebr_block_distill(int dtype, int tdtype, int ids64, int64_t N, int64_t V, int K, int64_t row_stride, double temperature,
                      int reduction, const void* logits, const void* teacher, const void* ids, void* stats, void* loss,
                      void* scale, void* scratch, void* stream);

/* Bytes of scratch that ebr_block_distill needs (16-byte aligned), -1 for sizes or types that it refuses. */
int64_t ebr_block_distill_scratch(int dtype, int64_t N, int64_t V, int K);

/* dx [N, V], contiguous, of that loss given its gradient (of loss's type; grad_stride 0: one, 1: one a row). scale: as the
 * forward left it, NULL for EBR_REDUCE_NONE. */
int ebr_block_distill_bwd(int dtype, int tdtype, int ids64, int64_t N, int64_t V, int K, int64_t row_stride,
                          double temperature, const void* logits, const void* teacher, const void* ids, const void* stats,
                          const void* scale, const void* grad, int64_t grad_stride, void* dx, void* stream);

/* Activations of the group norm. */
enum { EBR_ACT_NONE = 0, EBR_ACT_SILU = 1 };

/* y = f(w h + b), h = (x - mean) / sqrt(variance + eps), for x [B, L, C] contiguous, channels last: the statistics of each
 * sample and group are over its L cells and C / groups channels. w and b: fp32 (fp64 for fp64) [C], or NULL (1 and 0).
 * stats: [B, groups, 2] of that type, the mean and the factor, for the derivatives. scratch: 16-byte aligned, of
 * ebr_block_groupnorm_scratch's size for order 0. */
int ebr_block_groupnorm(int dtype, int act, int64_t B, int64_t L, int C, int groups, double eps, const void* x, const void* w,
                        const void* b, void* y, void* stats, void* scratch, void* stream);

/* dx, and dw and db (of w's type; NULL where not wanted), of y given dy. Scratch of order 1. */
int ebr_block_groupnorm_bwd(int dtype, int act, int64_t B, int64_t L, int C, int groups, const void* x, const void* w,
                            const void* b, const void* stats, const void* dy, void* dx, void* dw, void* db, void* scratch,
                            void* stream);

/* Gradients of <u, dx> + <uw, dw> + <ub, db> (uw, ub: NULL for zero) with respect to x (gx), dy (gdy), w (gw) and b (gb;
 * gw and gb NULL where not wanted). Scratch of order 2. */
int ebr_block_groupnorm_bwd2(int dtype, int act, int64_t B, int64_t L, int C, int groups, const void* x, const void* w,
                             const void* b, const void* stats, const void* dy, const void* u, const void* uw, const void* ub,
                             void* gx, void* gdy, void* gw, void* gb, void* scratch, void* stream);

/* Bytes of scratch of the group norm (order 0) and its derivatives (1, 2), for tensors of any alignment; -1 for sizes or types
 * that they refuse: more than 2^40 - 1 elements, or 2^24 - 1 workgroups or, where these do not hold whole groups, groups of
 * all samples. */
int64_t ebr_block_groupnorm_scratch(int dtype, int order, int64_t B, int64_t L, int C, int groups);

#ifdef __cplusplus
}
#endif

#endif /* EBR_BLOCK_H */
