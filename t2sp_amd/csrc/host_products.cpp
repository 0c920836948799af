// host_products.cpp — the operator entry points of the products of a language model's layers:
//   gemm_grouped, gemm_grouped_wgrad (gemm_grouped-interface.h), xent, xent_grad (xent-interface.h) and
//   gemv_w4 (gemv_w4-interface.h).
// They check and stage halide_buffer_t arguments like the other entries and call the thin layer of t2sp_hip.h.
#include "gemm_grouped-interface.h"
#include "gemv_w4-interface.h"
#include "runtime.hpp"
#include "t2sp_hip.h"
#include "xent-interface.h"

using namespace t2sp;

namespace {

constexpr int BFLOAT_CODE = 4;           // halide_type_bfloat of the Halide versions that have it

// T2SP_TYPE_* of a buffer of elements, or -1.
int element_type(const halide_buffer_t *b) {
    if (!b || b->type.lanes != 1) return -1;
    if (b->type.code == halide_type_float) return b->type.bits == 32 ? T2SP_TYPE_F32 : b->type.bits == 16 ? T2SP_TYPE_F16 : -1;
    return b->type.code == BFLOAT_CODE && b->type.bits == 16 ? T2SP_TYPE_BF16 : -1;
}
int element_bytes(int type) { return type == T2SP_TYPE_F32 ? 4 : 2; }

int check_elements(const halide_buffer_t *b, int type, const char *op, const char *name, int dims, Span *s) {
    return check_buffer_typed(b, op, name, dims, dims, s, type == T2SP_TYPE_BF16 ? BFLOAT_CODE : halide_type_float, 8 * element_bytes(type));
}
// The type of the first operand, checked; a negative code otherwise.
int first_operand(const halide_buffer_t *b, const char *op, const char *name, int dims, Span *s) {
    if (!b) return report(halide_error_code_buffer_argument_is_null, op, "buffer argument is NULL");
    const int type = element_type(b);
    if (type < 0) return report(halide_error_code_bad_type, op, "elements must be float32, float16 or bfloat16");
    const int err = check_elements(b, type, op, name, dims, s);
    return err ? err : type;
}
int check_result(const halide_buffer_t *b, int type, const char *op, const char *name, int dims, Span *s, int *out_type) {
    *out_type = b && element_type(b) == T2SP_TYPE_F32 ? T2SP_TYPE_F32 : type;
    return check_elements(b, *out_type, op, name, dims, s);
}
// int32 or int64; sets the bits.
int check_integers(const halide_buffer_t *b, const char *op, const char *name, int n, Span *s, int *bits) {
    *bits = b && b->type.bits == 64 ? 64 : 32;
    if (const int err = check_buffer_typed(b, op, name, 1, 1, s, halide_type_int, *bits)) return err;
    return b->dim[0].extent == n ? 0 : report(halide_error_code_constraint_violated, op, "the vector of integers has another length");
}
int64_t row_stride(const halide_buffer_t *b) {       // a single row's stride carries no information
    const int64_t cols = b->dim[0].extent;
    return b->dim[1].extent > 1 || b->dim[1].stride > cols ? b->dim[1].stride : cols;
}
int64_t matrix_stride(const halide_buffer_t *b) {
    const int64_t all = row_stride(b) * b->dim[1].extent;
    return b->dim[2].extent > 1 || b->dim[2].stride > all ? b->dim[2].stride : all;
}

// Device memory of one call, returned to the pool at its end.
struct Room {
    void *p = nullptr;
    size_t bytes = 0;
    int take(size_t n, const char *op) {
        bytes = n;
        if (n == 0) return 0;
        p = pool().get(n);
        return p ? 0 : report(halide_error_code_device_malloc_failed, op, "device allocation failed");
    }
    ~Room() { if (p) pool().put(p); }
};

}  // namespace

extern "C" int gemm_grouped(int32_t opb, halide_buffer_t *X, halide_buffer_t *W, halide_buffer_t *Offsets, halide_buffer_t *Y) {
    static const char *op = "gemm_grouped";
    std::lock_guard<std::mutex> lock(api_mutex());
    Span sx, sw, so, sy;
    int err, bits, out_type;
    const int type = first_operand(X, op, "X", 2, &sx);
    if (type < 0) return type;
    if ((err = check_elements(W, type, op, "W", 3, &sw))) return err;
    const int K = X->dim[0].extent, T = X->dim[1].extent, E = W->dim[2].extent, N = W->dim[opb ? 1 : 0].extent;
    if (E < 1 || E == INT32_MAX) return report(halide_error_code_constraint_violated, op, "no matrices");
    if ((err = check_integers(Offsets, op, "Offsets", E + 1, &so, &bits))) return err;
    if ((err = check_result(Y, type, op, "Y", 2, &sy, &out_type))) return err;
    if (W->dim[opb ? 0 : 1].extent != K || Y->dim[0].extent != N || Y->dim[1].extent != T)
        return report(halide_error_code_constraint_violated, op, "X (K, T), W (N, K, E) or (K, N, E), Y (N, T) disagree");
    if (K == 0) return report(halide_error_code_constraint_violated, op, "empty reduction extent");
    if (T == 0 || N == 0) return 0;
    Staged dx, dw, doff, dy;
    if ((err = dx.input(X, sx, op, element_bytes(type)))) return err;
    if ((err = dw.input(W, sw, op, element_bytes(type)))) return err;
    if ((err = doff.input(Offsets, so, op, bits / 8))) return err;
    if ((err = dy.output(Y, sy, op, true, element_bytes(out_type)))) return err;
    const int64_t ldx = row_stride(X), ldw = row_stride(W), sm = matrix_stride(W);
    Room room;
    if ((err = room.take(t2sp_gemm_grouped_workspace_bytes(type, opb != 0, dx.ptr(), dw.ptr(), T, E, K, N, ldx, ldw, sm), op))) return err;
    KernelTimer timer;
    err = t2sp_gemm_grouped(type, out_type, opb != 0, dx.ptr(), dw.ptr(), doff.ptr(), bits, dy.ptr(), T, E, K, N, ldx, ldw, sm, row_stride(Y), room.p,
                            room.bytes, api_stream());
    if (err) return report(err, op, "kernel launch failed");
    if ((err = timer.stop_and_sync(op))) return err;
    return dy.finish(op);
}

extern "C" int gemm_grouped_wgrad(halide_buffer_t *X, halide_buffer_t *dY, halide_buffer_t *Offsets, halide_buffer_t *dW) {
    static const char *op = "gemm_grouped_wgrad";
    std::lock_guard<std::mutex> lock(api_mutex());
    Span sx, sd, so, sw;
    int err, bits, out_type;
    const int type = first_operand(X, op, "X", 2, &sx);
    if (type < 0) return type;
    if ((err = check_elements(dY, type, op, "dY", 2, &sd))) return err;
    if ((err = check_result(dW, type, op, "dW", 3, &sw, &out_type))) return err;
    const int K = X->dim[0].extent, T = X->dim[1].extent, N = dY->dim[0].extent, E = dW->dim[2].extent;
    if (E < 1 || E == INT32_MAX) return report(halide_error_code_constraint_violated, op, "no matrices");
    if ((err = check_integers(Offsets, op, "Offsets", E + 1, &so, &bits))) return err;
    if (dY->dim[1].extent != T || dW->dim[0].extent != N || dW->dim[1].extent != K)
        return report(halide_error_code_constraint_violated, op, "X (K, T), dY (N, T), dW (N, K, E) disagree");
    if (K == 0 || N == 0) return 0;
    Staged dx, dd, doff, dw;
    if ((err = dx.input(X, sx, op, element_bytes(type)))) return err;
    if ((err = dd.input(dY, sd, op, element_bytes(type)))) return err;
    if ((err = doff.input(Offsets, so, op, bits / 8))) return err;
    if ((err = dw.output(dW, sw, op, false, element_bytes(out_type)))) return err;
    const int64_t ldx = row_stride(X), ldy = row_stride(dY);
    Room room;
    if ((err = room.take(t2sp_gemm_grouped_wgrad_workspace_bytes(type, dx.ptr(), dd.ptr(), T, E, K, N, ldx, ldy), op))) return err;
    KernelTimer timer;
    err = t2sp_gemm_grouped_wgrad(type, out_type, dx.ptr(), dd.ptr(), doff.ptr(), bits, dw.ptr(), T, E, K, N, ldx, ldy, row_stride(dW),
                                  matrix_stride(dW), room.p, room.bytes, api_stream());
    if (err) return report(err, op, "kernel launch failed");
    if ((err = timer.stop_and_sync(op))) return err;
    return dw.finish(op);
}

extern "C" int xent(halide_buffer_t *H, halide_buffer_t *W, halide_buffer_t *Labels, halide_buffer_t *Loss, halide_buffer_t *Lse) {
    static const char *op = "xent";
    std::lock_guard<std::mutex> lock(api_mutex());
    Span sh, sw, sl, so, se;
    int err, bits;
    const int type = first_operand(H, op, "H", 2, &sh);
    if (type < 0) return type;
    if ((err = check_elements(W, type, op, "W", 2, &sw))) return err;
    const int D = H->dim[0].extent, T = H->dim[1].extent, V = W->dim[1].extent;
    if ((err = check_integers(Labels, op, "Labels", T, &sl, &bits))) return err;
    if ((err = check_buffer(Loss, op, "Loss", 1, 1, &so))) return err;
    if ((err = check_buffer(Lse, op, "Lse", 1, 1, &se))) return err;
    if (W->dim[0].extent != D || Loss->dim[0].extent != T || Lse->dim[0].extent != T || D == 0 || V == 0)
        return report(halide_error_code_constraint_violated, op, "H (D, T), W (D, V), Loss (T), Lse (T) disagree or are empty");
    if (T == 0) return 0;
    Staged dh, dw, dl, dloss, dlse;
    if ((err = dh.input(H, sh, op, element_bytes(type)))) return err;
    if ((err = dw.input(W, sw, op, element_bytes(type)))) return err;
    if ((err = dl.input(Labels, sl, op, bits / 8))) return err;
    if ((err = dloss.output(Loss, so, op))) return err;
    if ((err = dlse.output(Lse, se, op))) return err;
    const int64_t ldh = row_stride(H), ldw = row_stride(W);
    Room room;
    if ((err = room.take(t2sp_xent_workspace_bytes(type, dh.ptr(), dw.ptr(), T, V, D, ldh, ldw), op))) return err;
    KernelTimer timer;
    err = t2sp_xent(type, dh.ptr(), dw.ptr(), dl.ptr(), bits, dloss.ptr(), dlse.ptr(), T, V, D, ldh, ldw, room.p, room.bytes, api_stream());
    if (err) return report(err, op, "kernel launch failed");
    if ((err = timer.stop_and_sync(op))) return err;
    if ((err = dloss.finish(op))) return err;
    return dlse.finish(op);
}

extern "C" int xent_grad(halide_buffer_t *H, halide_buffer_t *W, halide_buffer_t *Labels, halide_buffer_t *Lse, halide_buffer_t *DLoss,
                         halide_buffer_t *dH, halide_buffer_t *dW) {
    static const char *op = "xent_grad";
    std::lock_guard<std::mutex> lock(api_mutex());
    Span sh, sw, sl, se, sd, sgh, sgw;
    int err, bits, out_h, out_w;
    const int type = first_operand(H, op, "H", 2, &sh);
    if (type < 0) return type;
    if ((err = check_elements(W, type, op, "W", 2, &sw))) return err;
    const int D = H->dim[0].extent, T = H->dim[1].extent, V = W->dim[1].extent;
    if ((err = check_integers(Labels, op, "Labels", T, &sl, &bits))) return err;
    if ((err = check_buffer(Lse, op, "Lse", 1, 1, &se))) return err;
    if ((err = check_buffer(DLoss, op, "DLoss", 1, 1, &sd))) return err;
    if ((err = check_result(dH, type, op, "dH", 2, &sgh, &out_h))) return err;
    if ((err = check_result(dW, type, op, "dW", 2, &sgw, &out_w))) return err;
    if (out_h != out_w) return report(halide_error_code_bad_type, op, "dH and dW must have one type");
    if (W->dim[0].extent != D || Lse->dim[0].extent != T || DLoss->dim[0].extent != T || dH->dim[0].extent != D || dH->dim[1].extent != T ||
        dW->dim[0].extent != D || dW->dim[1].extent != V || D == 0 || V == 0)
        return report(halide_error_code_constraint_violated, op, "H, dH (D, T), W, dW (D, V), Lse, DLoss (T) disagree or are empty");
    Staged dh, dw, dl, dlse, dd, gh, gw;
    if ((err = dh.input(H, sh, op, element_bytes(type)))) return err;
    if ((err = dw.input(W, sw, op, element_bytes(type)))) return err;
    if ((err = dl.input(Labels, sl, op, bits / 8))) return err;
    if ((err = dlse.input(Lse, se, op))) return err;
    if ((err = dd.input(DLoss, sd, op))) return err;
    if ((err = gh.output(dH, sgh, op, false, element_bytes(out_h)))) return err;
    if ((err = gw.output(dW, sgw, op, false, element_bytes(out_w)))) return err;
    const int64_t ldh = row_stride(H), ldw = row_stride(W);
    Room room;
    if ((err = room.take(t2sp_xent_grad_workspace_bytes(type, dh.ptr(), dw.ptr(), T, V, D, ldh, ldw), op))) return err;
    KernelTimer timer;
    err = t2sp_xent_grad(type, out_h, dh.ptr(), dw.ptr(), dl.ptr(), bits, dlse.ptr(), dd.ptr(), gh.ptr(), gw.ptr(), T, V, D, ldh, ldw, row_stride(dH),
                         row_stride(dW), room.p, room.bytes, api_stream());
    if (err) return report(err, op, "kernel launch failed");
    if ((err = timer.stop_and_sync(op))) return err;
    if ((err = gh.finish(op))) return err;
    return gw.finish(op);
}

extern "C" int gemv_w4(int32_t group, halide_buffer_t *X, halide_buffer_t *Q, halide_buffer_t *S, halide_buffer_t *Z, halide_buffer_t *Ids,
                       halide_buffer_t *Y) {
    static const char *op = "gemv_w4";
    std::lock_guard<std::mutex> lock(api_mutex());
    Span sx, sq, ss, sz, si, sy;
    int err;
    const int type = first_operand(X, op, "X", 2, &sx);
    if (type < 0) return type;
    const int dims = Ids ? 3 : 2;
    if ((err = check_buffer_typed(Q, op, "Q", dims, dims, &sq, halide_type_uint, 8))) return err;
    if ((err = check_elements(S, type, op, "S", dims, &ss))) return err;
    if (Z && (err = check_elements(Z, type, op, "Z", dims, &sz))) return err;
    if ((err = check_elements(Y, type, op, "Y", 2, &sy))) return err;
    const int K = X->dim[0].extent, M = X->dim[1].extent, N = Q->dim[1].extent, E = Ids ? Q->dim[2].extent : 1;
    if (Ids && (err = check_buffer_typed(Ids, op, "Ids", 1, 1, &si, halide_type_int, 32))) return err;
    int64_t q_bytes, s_elements;
    if (t2sp_w4_sizes(N, K, group, &q_bytes, &s_elements)) return report(halide_error_code_constraint_violated, op, "group must be a power of two from 32 on; K and N not empty");
    const int groups = (int)(((int64_t)K + group - 1) / group);
    auto side_ok = [&](const halide_buffer_t *b) { return b->dim[0].extent == groups && b->dim[1].extent == N && (!Ids || b->dim[2].extent == E); };
    if (Q->dim[0].extent != K || E < 1 || !side_ok(S) || (Z && !side_ok(Z)) || Y->dim[0].extent != N || Y->dim[1].extent != M ||
        (Ids && Ids->dim[0].extent != M))
        return report(halide_error_code_constraint_violated, op, "X (K, M), Q (K, N), S and Z (ceil(K / Group), N), Y (N, M) disagree");
    if (M == 0) return 0;
    Staged dx, dq, ds, dz, di, dy;
    if ((err = dx.input(X, sx, op, element_bytes(type)))) return err;
    if ((err = dq.input(Q, sq, op, 1))) return err;
    if ((err = ds.input(S, ss, op, element_bytes(type)))) return err;
    if (Z && (err = dz.input(Z, sz, op, element_bytes(type)))) return err;
    if (Ids && (err = di.input(Ids, si, op, 4))) return err;
    if ((err = dy.output(Y, sy, op, false, element_bytes(type)))) return err;
    Room pq, ps, pz;
    const size_t side = (size_t)E * s_elements * element_bytes(type);
    if ((err = pq.take((size_t)E * q_bytes, op)) || (err = ps.take(side, op)) || (err = pz.take(Z ? side : 0, op))) return err;
    auto each = [&](const halide_buffer_t *b) { return b && b->dimensions == 3 ? matrix_stride(b) : (int64_t)0; };
    KernelTimer timer;
    err = t2sp_w4_pack(type, reinterpret_cast<const uint8_t *>(dq.ptr()), ds.ptr(), Z ? dz.ptr() : nullptr, E, N, K, group, row_stride(Q), each(Q),
                       row_stride(S), each(S), Z ? row_stride(Z) : 0, each(Z), pq.p, ps.p, pz.p, api_stream());
    if (!err)
        err = t2sp_gemv_w4(type, dx.ptr(), pq.p, ps.p, pz.p, Ids ? reinterpret_cast<const int *>(di.ptr()) : nullptr, dy.ptr(), M, N, K, E, group,
                           row_stride(X), row_stride(Y), api_stream());
    if (err) return report(err, op, "kernel launch failed");
    if ((err = timer.stop_and_sync(op))) return err;
    return dy.finish(op);
}

#define T2SP_NS(fn, params, args)                                  \
    extern "C" double fn##_ns params {                             \
        const int rc = fn args;                                    \
        return rc == 0 ? t2sp_last_kernel_ns() : (double)rc;       \
    }
T2SP_NS(gemm_grouped, (int32_t o, halide_buffer_t *a, halide_buffer_t *b, halide_buffer_t *c, halide_buffer_t *d), (o, a, b, c, d))
T2SP_NS(gemm_grouped_wgrad, (halide_buffer_t *a, halide_buffer_t *b, halide_buffer_t *c, halide_buffer_t *d), (a, b, c, d))
T2SP_NS(xent, (halide_buffer_t *a, halide_buffer_t *b, halide_buffer_t *c, halide_buffer_t *d, halide_buffer_t *e), (a, b, c, d, e))
T2SP_NS(xent_grad, (halide_buffer_t *a, halide_buffer_t *b, halide_buffer_t *c, halide_buffer_t *d, halide_buffer_t *e, halide_buffer_t *f,
                    halide_buffer_t *g), (a, b, c, d, e, f, g))
T2SP_NS(gemv_w4, (int32_t o, halide_buffer_t *a, halide_buffer_t *b, halide_buffer_t *c, halide_buffer_t *d, halide_buffer_t *e, halide_buffer_t *f),
        (o, a, b, c, d, e, f))
