/* C ABI of the optimizer's step in libebr_attn.so (gfx950): AdamW over many tensors in few launches, with moments in 32
 * bits or in 8, and the global norm of many gradients.
 *
 * Tensors are contiguous in memory, of any alignment that their elements have; they may be views of one buffer. The tables
 * are the host's and are read before the call returns; everything that they point to is the device's. Conventions otherwise
 * as in ebr_attn.h (error codes, streams, ownership): no call allocates, waits for the device or reads from it, so all of
 * them may be captured into a graph.
 */
#ifndef EBR_OPTIM_H
#define EBR_OPTIM_H

#include <stdint.h>

#include "ebr_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A gradient: n elements of dtype. */
typedef struct {
    const void* g;
    int64_t n;
    int32_t dtype;
    int32_t reserved; /* 0 */
} ebr_optim_grad;

/* A parameter with its gradient and moments: n elements each. Moments in 32 bits are of type fp32 (fp64 for an fp64
 * parameter), m the first and v the second. Moments in 8 bits are OCP e4m3 numbers, m the first and v the ROOT of the second,
 * with ms and vs their fp32 scales, one for each 256 consecutive elements: element i stands for m[i] * ms[i / 256] (ms and
 * vs are not read for 32 bits). step: the number of steps taken, one int64; the call adds 1 to it. */
typedef struct {
    void* p;
    const void* g;
    void* m;
    void* v;
    float* ms;
    float* vs;
    int64_t* step;
    int64_t n;
} ebr_optim_tensor;

/* norm[0] = sqrt(sum of g^2 over all gradients), summed in fp64 in a fixed order; single[0], where not NULL, the same in
 * fp32. At least one gradient; n may be 0. scratch: ebr_block_grad_norm_scratch bytes, 16-byte aligned. */
int ebr_block_grad_norm(int64_t count, const ebr_optim_grad* grads, double* norm, float* single, void* scratch,
                        void* stream);
int64_t ebr_block_grad_norm_scratch(int64_t count, const ebr_optim_grad* grads);

/* One AdamW step of count tensors (fewer than 2^24, and 2^40 elements), whose parameters are of ptype and gradients of gtype (ptype, or a 16-bit type with fp32
 * parameters), bits 32 or 8 (fp64: 32). With t the step's number, counted from 1:
 *   g <- g min(1, max_norm / (norm[0] + 1e-6))   where norm is not NULL: of all the gradients, as the call above leaves it
 *   m <- beta1 m + (1 - beta1) g,   v <- beta2 v + (1 - beta2) g^2
 *   p <- p (1 - lr decay) - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
 * lr is read from lr_dev (fp32, the device's) where that is not NULL. Arithmetic is fp32 (fp64 for fp64 parameters), the
 * parameter's sum rounded once. In 8 bits the moments are taken in fp64 and stored, after the parameter's step has used them
 * as they are, against their block's largest: scale = largest / 448 (0, and all numbers 0, where that is below 2^-126), and a
 * number y = moment / scale between two neighbours k s and (k + 1) s becomes floor(y / s + t) s, with t in [0, 1) the 24 upper
 * bits of (i * 0x85EBCA77 + step * 0x9E3779B1) mod 2^32 for the first moment, and of that plus 2^31 for the root: over the
 * steps t takes its values evenly, so that nothing is lost on average and no number stays where it is for good. A root above
 * 0 never becomes 0. scratch: ebr_block_adamw_scratch bytes, 16-byte aligned. No two of the
 * tensors that are written share memory, nor does what is read with them (but a gradient may be its own parameter). */
int ebr_block_adamw(int ptype, int gtype, int bits, int64_t count, const ebr_optim_tensor* tensors, double lr,
                    const float* lr_dev, double beta1, double beta2, double eps, double decay, const double* norm,
                    double max_norm, void* scratch, void* stream);
int64_t ebr_block_adamw_scratch(int64_t count);

#ifdef __cplusplus
}
#endif

#endif /* EBR_OPTIM_H */
