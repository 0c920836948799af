/* gemm_grouped-interface.h — host interface of the products grouped by expert.
 *
 * Entries in the form the other pipelines have (inputs first, output last, 0 on success, a negative
 * halide_error_code_t otherwise); they have no counterpart in the reference.  Element types: float32,
 * float16 (halide_type_float, 16 bits) and bfloat16 (type code 4, 16 bits: halide_type_bfloat of later
 * Halide versions), the same for both operands; the result has that type or float32.  Offsets are int32 or
 * int64.  Buffers on the device are used where they lie, host buffers are staged, as everywhere.
 */
#ifndef T2SP_GEMM_GROUPED_INTERFACE_H
#define T2SP_GEMM_GROUPED_INTERFACE_H
#include "t2sp_buffer.h"
#include "t2sp_runtime.h"
#ifdef __cplusplus
extern "C" {
#endif

/* Y[r] = X[r] * op(W[e]) for the rows Offsets[e] <= r < Offsets[e+1].  X: (K, T), rows sorted by group; W: (N, K, E),
 * or (K, N, E) when OpB; Offsets: (E + 1), not decreasing (values are clamped to 0 .. T and taken as their running maximum); Y: (N, T).  Rows of Y
 * outside every group keep what they held. */
int gemm_grouped(int32_t OpB, struct halide_buffer_t *X, struct halide_buffer_t *W, struct halide_buffer_t *Offsets,
                 struct halide_buffer_t *Y);

/* dW[e] = X_e^T * dY_e, zeros for an empty group.  X: (K, T), dY: (N, T), Offsets: (E + 1), dW: (N, K, E). */
int gemm_grouped_wgrad(struct halide_buffer_t *X, struct halide_buffer_t *dY, struct halide_buffer_t *Offsets,
                       struct halide_buffer_t *dW);

/* The same, returning the kernel time in ns (negative error code on failure). */
double gemm_grouped_ns(int32_t OpB, struct halide_buffer_t *X, struct halide_buffer_t *W, struct halide_buffer_t *Offsets,
                       struct halide_buffer_t *Y);
double gemm_grouped_wgrad_ns(struct halide_buffer_t *X, struct halide_buffer_t *dY, struct halide_buffer_t *Offsets,
                             struct halide_buffer_t *dW);

/* The argv form and the argument table (see gemm-interface.h); the table lists float32 and int32, the
 * types named above are accepted too. */
int gemm_grouped_argv(void **args);
int gemm_grouped_wgrad_argv(void **args);
const struct halide_filter_metadata_t *gemm_grouped_metadata(void);
const struct halide_filter_metadata_t *gemm_grouped_wgrad_metadata(void);

#ifdef __cplusplus
}
#endif
#endif
