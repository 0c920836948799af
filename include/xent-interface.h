/* xent-interface.h — host interface of the cross entropy of a softmax over a vocabulary.
 *
 * Entries in the form the other pipelines have (inputs first, outputs last, 0 on success, a negative
 * halide_error_code_t otherwise); they have no counterpart in the reference.  H and W have one element type
 * (float32, float16, or bfloat16 as type code 4 with 16 bits), the gradients that type or float32; Loss, Lse and
 * DLoss are float32, Labels int32 or int64.
 */
#ifndef T2SP_XENT_INTERFACE_H
#define T2SP_XENT_INTERFACE_H
#include "t2sp_buffer.h"
#include "t2sp_runtime.h"
#ifdef __cplusplus
extern "C" {
#endif

/* Lse[t] = log sum_v exp z[t,v], Loss[t] = Lse[t] - z[t, Labels[t]] with z = H W^T, which is not kept; Loss is 0 where
 * the label is outside 0 .. V - 1.  H: (D, T), W: (D, V), Labels, Loss, Lse: (T). */
int xent(struct halide_buffer_t *H, struct halide_buffer_t *W, struct halide_buffer_t *Labels, struct halide_buffer_t *Loss,
         struct halide_buffer_t *Lse);

/* dH = g W (D, T) and dW = g^T H (D, V) with g[t,v] = (exp(z[t,v] - Lse[t]) - [v == Labels[t]]) * DLoss[t]; tokens
 * whose label is outside 0 .. V - 1 take no part and get zeros. */
int xent_grad(struct halide_buffer_t *H, struct halide_buffer_t *W, struct halide_buffer_t *Labels, struct halide_buffer_t *Lse,
              struct halide_buffer_t *DLoss, struct halide_buffer_t *dH, struct halide_buffer_t *dW);

/* The same, returning the kernel time in ns (negative error code on failure). */
double xent_ns(struct halide_buffer_t *H, struct halide_buffer_t *W, struct halide_buffer_t *Labels, struct halide_buffer_t *Loss,
               struct halide_buffer_t *Lse);
double xent_grad_ns(struct halide_buffer_t *H, struct halide_buffer_t *W, struct halide_buffer_t *Labels,
                    struct halide_buffer_t *Lse, struct halide_buffer_t *DLoss, struct halide_buffer_t *dH,
                    struct halide_buffer_t *dW);

/* The argv form and the argument table (see gemm-interface.h); the table lists float32 and int32, the
 * types named above are accepted too. */
int xent_argv(void **args);
int xent_grad_argv(void **args);
const struct halide_filter_metadata_t *xent_metadata(void);
const struct halide_filter_metadata_t *xent_grad_metadata(void);

#ifdef __cplusplus
}
#endif
#endif
