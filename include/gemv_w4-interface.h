/* gemv_w4-interface.h — host interface of the products with 4-bit weights and group scales.
 *
 * An entry in the form the other pipelines have (inputs first, output last, 0 on success, a negative
 * halide_error_code_t otherwise); it has no counterpart in the reference.  X, S, Z and Y have one element
 * type (float32, float16, or bfloat16 as type code 4 with 16 bits), Q is uint8, Ids int32.  The entry lays the
 * numbers out for the kernel on every call; a program that keeps its weights on the device does that once
 * with t2sp_w4_pack and calls t2sp_gemv_w4 (t2sp_hip.h).
 */
#ifndef T2SP_GEMV_W4_INTERFACE_H
#define T2SP_GEMV_W4_INTERFACE_H
#include "t2sp_buffer.h"
#include "t2sp_runtime.h"
#ifdef __cplusplus
extern "C" {
#endif

/* Y[n,m] = sum_k X[k,m] * (Q[k,n] - Z[k/Group,n]) * S[k/Group,n].  X: (K, M); Q: (K, N), one number per byte in its low
 * four bits; S, Z: (ceil(K / Group), N), Z = NULL: 8 everywhere; Group: 32, 64, 128, ... (powers of two); Y: (N, M).
 * With Ids (M) not NULL, Q, S and Z have a third dimension E and row m takes matrix Ids[m]; an id outside
 * 0 .. E - 1 gives a row of zeros. */
int gemv_w4(int32_t Group, struct halide_buffer_t *X, struct halide_buffer_t *Q, struct halide_buffer_t *S,
            struct halide_buffer_t *Z, struct halide_buffer_t *Ids, struct halide_buffer_t *Y);

/* gemv_w4() that returns the kernel time in ns (negative error code on failure). */
double gemv_w4_ns(int32_t Group, struct halide_buffer_t *X, struct halide_buffer_t *Q, struct halide_buffer_t *S,
                  struct halide_buffer_t *Z, struct halide_buffer_t *Ids, struct halide_buffer_t *Y);

/* The argv form and the argument table (see gemm-interface.h); the table lists float32 operands. */
int gemv_w4_argv(void **args);
const struct halide_filter_metadata_t *gemv_w4_metadata(void);

#ifdef __cplusplus
}
#endif
#endif
