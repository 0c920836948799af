"""Python mirror of the products of a language model's layers (include/t2sp_hip.h, second half): products
grouped by expert, cross entropy over a vocabulary, products with 4-bit weights.

torch CUDA tensors go to the thin layer: kernels are enqueued on the current stream of the tensors' device and
the call returns without waiting, so it can be captured into a HIP graph; workspaces and fresh results come from
torch's allocator, which keeps them apart between streams and captured graphs.  Element types are float32, float16
and bfloat16.  numpy arrays (float32 or float16, host memory) go through the operator entries
(include/gemm_grouped-interface.h, xent-interface.h, gemv_w4-interface.h), which stage them through the device.
Misuse raises T2spError with the Halide error code that the entry would return."""
import ctypes

import numpy as np

from ._lib import lib
from .buffer import HalideBuffer
from .ops import T2spError, _check, _is_torch, host_empty

BAD_TYPE, SHAPE, BAD_DIMENSIONS, OUT_OF_BOUNDS, NULL_BUFFER = -3, -8, -43, -4, -12
_codes = None


def _type_codes():
    global _codes
    if _codes is None:
        import torch
        _codes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    return _codes


def _need(op, ok, code=SHAPE):
    if not ok:
        raise T2spError(op, code)


def _tensors(op, dims, *tensors):
    """Common checks of floating-point CUDA tensors: one element type, one device, the stated ranks, unit stride along
    the last axis.  Returns the T2SP_TYPE_* code."""
    first = tensors[0]
    code = _type_codes().get(first.dtype)
    _need(op, code is not None, BAD_TYPE)
    for t, d in zip(tensors, dims):
        _need(op, t.dtype == first.dtype, BAD_TYPE)
        _need(op, t.dim() == d, BAD_DIMENSIONS)
        _need(op, t.is_cuda and t.device == first.device)
        _need(op, t.shape[-1] <= 1 or t.stride(-1) == 1)
    return code


def _integers(op, t, like, n):
    """Bits of a contiguous vector of n integers on the device of `like`."""
    import torch
    _need(op, t.dtype in (torch.int32, torch.int64), BAD_TYPE)
    _need(op, t.dim() == 1, BAD_DIMENSIONS)
    _need(op, t.device == like.device and t.shape[0] == n and (n <= 1 or t.stride(0) == 1))
    return 32 if t.dtype == torch.int32 else 64


def _result(op, out, shape, like, dtype, types):
    import torch
    if out is None:
        return torch.empty(shape, dtype=dtype, device=like.device)
    _need(op, out.dtype in types, BAD_TYPE)
    _need(op, out.dim() == len(shape), BAD_DIMENSIONS)
    _need(op, tuple(out.shape) == tuple(shape) and out.device == like.device and (shape[-1] <= 1 or out.stride(-1) == 1))
    return out


def _row(t):
    """Elements between rows (a single row's stride carries no information)."""
    return t.stride(-2) if t.shape[-2] > 1 else max(t.stride(-2), t.shape[-1])


def _matrix(t):
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1] * _row(t))


class _On:
    """Makes the tensors' device current around a call."""

    def __init__(self, t):
        import torch
        self.index = t.device.index
        self.back = torch.cuda.current_device()
        self.set = torch.cuda.set_device

    def __enter__(self):
        if self.index != self.back:
            self.set(self.index)

    def __exit__(self, *exc):
        if self.index != self.back:
            self.set(self.back)


def _stream(t):
    import torch
    return torch.cuda.current_stream(t.device).cuda_stream


def _room(nbytes, like):
    """(pointer, bytes, owner) of a workspace.  The owner may be dropped after the call: torch's allocator hands the memory
    out again only to work that is ordered behind it."""
    if not nbytes:
        return None, 0, None
    import torch
    t = torch.empty(nbytes, dtype=torch.uint8, device=like.device)
    return t.data_ptr(), nbytes, t


def gemm_grouped(X, W, offsets, opb=0, out=None, out_dtype=None):
    """Y[r] = X[r] @ op(W[e]) for the rows offsets[e] <= r < offsets[e + 1] of group e.

    X: (T, K) rows sorted by group; W: (E, K, N), or (E, N, K) when opb; offsets: E + 1 int32 or int64 on the device,
    not decreasing (they are clamped to 0 .. T).  Y: (T, N) of X's type, or float32 (out_dtype, or the type of `out`).
    Rows outside every group are left as they were (in a fresh result: whatever its memory held).  The gradient of X is
    gemm_grouped(dY, W, offsets, opb=1 - opb)."""
    op = "gemm_grouped"
    if not _is_torch(X):
        return _host_grouped(op, X, W, offsets, opb, out)
    import torch
    code = _tensors(op, (2, 3), X, W)
    T, K = X.shape
    E, N = W.shape[0], W.shape[1] if opb else W.shape[2]
    _need(op, (W.shape[2] if opb else W.shape[1]) == K and E >= 1 and K >= 1 and N >= 1)
    bits = _integers(op, offsets, X, E + 1)
    Y = _result(op, out, (T, N), X, out_dtype or X.dtype, (X.dtype, torch.float32))
    _need(op, Y.dtype in (X.dtype, torch.float32), BAD_TYPE)
    L = lib()
    x, w, ldx, ldw, sw = X.data_ptr(), W.data_ptr(), _row(X), _row(W), _matrix(W)
    with _On(X):
        ws, nbytes, owner = _room(L.t2sp_gemm_grouped_workspace_bytes(code, opb, x, w, T, E, K, N, ldx, ldw, sw), X)
        _check(op, L.t2sp_gemm_grouped(code, _type_codes()[Y.dtype], opb, x, w, offsets.data_ptr(), bits, Y.data_ptr(), T, E, K, N,
                                       ldx, ldw, sw, _row(Y), ws, nbytes, _stream(X)))
    return Y


def gemm_grouped_wgrad(X, dY, offsets, out=None, out_dtype=None):
    """dW[e] = X_e.T @ dY_e over the rows offsets[e] <= r < offsets[e + 1] of each group, zeros for an empty one.

    X: (T, K), dY: (T, N), offsets as in gemm_grouped.  dW: (E, K, N) of X's type, or float32."""
    op = "gemm_grouped_wgrad"
    if not _is_torch(X):
        return _host_wgrad(op, X, dY, offsets, out)
    import torch
    code = _tensors(op, (2, 2), X, dY)
    T, K = X.shape
    N, E = dY.shape[1], offsets.shape[0] - 1
    _need(op, dY.shape[0] == T and E >= 1 and K >= 1 and N >= 1)
    bits = _integers(op, offsets, X, E + 1)
    dW = _result(op, out, (E, K, N), X, out_dtype or X.dtype, (X.dtype, torch.float32))
    _need(op, dW.dtype in (X.dtype, torch.float32), BAD_TYPE)
    L = lib()
    x, dy, ldx, ldy = X.data_ptr(), dY.data_ptr(), _row(X), _row(dY)
    with _On(X):
        ws, nbytes, owner = _room(L.t2sp_gemm_grouped_wgrad_workspace_bytes(code, x, dy, T, E, K, N, ldx, ldy), X)
        _check(op, L.t2sp_gemm_grouped_wgrad(code, _type_codes()[dW.dtype], x, dy, offsets.data_ptr(), bits, dW.data_ptr(), T, E, K,
                                             N, ldx, ldy, _row(dW), _matrix(dW), ws, nbytes, _stream(X)))
    return dW


def _xent_args(op, H, W, labels):
    code = _tensors(op, (2, 2), H, W)
    T, D = H.shape
    V = W.shape[0]
    _need(op, W.shape[1] == D and D >= 1 and V >= 1)
    return code, T, V, D, _integers(op, labels, H, T)


def _floats(op, t, like, n):
    import torch
    _need(op, t.dtype == torch.float32, BAD_TYPE)
    _need(op, t.dim() == 1, BAD_DIMENSIONS)
    _need(op, t.device == like.device and t.shape[0] == n and (n <= 1 or t.stride(0) == 1))
    return t


def xent(H, W, labels, loss=None, lse=None):
    """Cross entropy of a softmax over a vocabulary, from hidden states: (loss, lse), float32 vectors of one value per token.

    H: (T, D), W: (V, D), labels: T int32 or int64; z = H @ W.T is not kept.  lse[t] = log sum exp z[t],
    loss[t] = lse[t] - z[t, labels[t]], 0 where the label is outside 0 .. V - 1."""
    op = "xent"
    if not _is_torch(H):
        return _host_xent(op, H, W, labels, loss, lse)
    import torch
    code, T, V, D, bits = _xent_args(op, H, W, labels)
    loss = torch.empty(T, dtype=torch.float32, device=H.device) if loss is None else _floats(op, loss, H, T)
    lse = torch.empty(T, dtype=torch.float32, device=H.device) if lse is None else _floats(op, lse, H, T)
    L = lib()
    h, w, ldh, ldw = H.data_ptr(), W.data_ptr(), _row(H), _row(W)
    with _On(H):
        ws, nbytes, owner = _room(L.t2sp_xent_workspace_bytes(code, h, w, T, V, D, ldh, ldw), H)
        _check(op, L.t2sp_xent(code, h, w, labels.data_ptr(), bits, loss.data_ptr(), lse.data_ptr(), T, V, D, ldh, ldw, ws, nbytes, _stream(H)))
    return loss, lse


def xent_grad(H, W, labels, lse, dloss, dH=None, dW=None, out_dtype=None, wanted=(True, True)):
    """Gradients (dH, dW) of sum_t dloss[t] * loss[t] (see xent): dH = g @ W, dW = g.T @ H with
    g[t, v] = (exp(z[t, v] - lse[t]) - [v == labels[t]]) * dloss[t]; tokens without a label take no part.

    lse: what xent returned; dloss: T float32.  The results have H's type, or float32 (out_dtype, or the type of dH / dW).
    `wanted` leaves one out (its place in the result is None)."""
    op = "xent_grad"
    if not _is_torch(H):
        return _host_xent_grad(op, H, W, labels, lse, dloss, dH, dW, wanted)
    import torch
    code, T, V, D, bits = _xent_args(op, H, W, labels)
    _floats(op, lse, H, T)
    _floats(op, dloss, H, T)
    types = (H.dtype, torch.float32)
    dtype = out_dtype or (dH.dtype if dH is not None else dW.dtype if dW is not None else H.dtype)
    dH = _result(op, dH, (T, D), H, dtype, types) if wanted[0] or dH is not None else None
    dW = _result(op, dW, (V, D), H, dtype, types) if wanted[1] or dW is not None else None
    _need(op, dtype in types and all(t is None or t.dtype == dtype for t in (dH, dW)), BAD_TYPE)
    L = lib()
    h, w, ldh, ldw = H.data_ptr(), W.data_ptr(), _row(H), _row(W)
    with _On(H):
        ws, nbytes, owner = _room(L.t2sp_xent_grad_workspace_bytes(code, h, w, T, V, D, ldh, ldw), H)
        _check(op, L.t2sp_xent_grad(code, _type_codes()[dtype], h, w, labels.data_ptr(), bits, lse.data_ptr(), dloss.data_ptr(),
                                    dH.data_ptr() if dH is not None else None, dW.data_ptr() if dW is not None else None, T, V, D, ldh, ldw,
                                    _row(dH) if dH is not None else D, _row(dW) if dW is not None else D, ws, nbytes, _stream(H)))
    return dH, dW


class W4:
    """Matrices of 4-bit numbers in the layout of the kernels (pack_w4): E matrices of N x K, or one (E is None)."""

    def __init__(self, E, N, K, group, Q, S, Z):
        self.E, self.N, self.K, self.group, self.Q, self.S, self.Z = E, N, K, group, Q, S, Z
        self.code = _type_codes()[S.dtype]


def pack_w4(q, scales, zeros=None, group=128):
    """Lays 4-bit numbers out for gemv_w4, once: W[n, k] = (q[n, k] - zeros[n, k // group]) * scales[n, k // group], with
    zeros = 8 when there are none.

    q: uint8 (N, K), or (E, N, K) for E matrices, one number in the low four bits of each byte; scales, zeros:
    (..., N, ceil(K / group)) of the type of the rows they will meet (float32, float16 or bfloat16).  group: a power of two
    from 32 on; at least K for one scale per row."""
    import torch
    op = "pack_w4"
    _need(op, q.dtype == torch.uint8, BAD_TYPE)
    _need(op, q.dim() in (2, 3), BAD_DIMENSIONS)
    _need(op, q.is_cuda and (q.shape[-1] <= 1 or q.stride(-1) == 1))
    code = _tensors(op, (q.dim(),) * 2, *((scales,) if zeros is None else (scales, zeros)))
    N, K = q.shape[-2:]
    group = int(group)
    qb, se = ctypes.c_int64(), ctypes.c_int64()
    L = lib()
    _check(op, L.t2sp_w4_sizes(N, K, group, ctypes.byref(qb), ctypes.byref(se)))
    E = q.shape[0] if q.dim() == 3 else 1
    want = tuple(q.shape[:-1]) + (-(-K // group),)
    _need(op, E >= 1 and tuple(scales.shape) == want and (zeros is None or tuple(zeros.shape) == want) and scales.device == q.device)
    Q = torch.empty(E * qb.value, dtype=torch.uint8, device=q.device)
    S = torch.empty(E * se.value, dtype=scales.dtype, device=q.device)
    Z = torch.empty_like(S) if zeros is not None else None
    each = lambda t: _matrix(t) if t.dim() == 3 else 0
    with _On(q):
        _check(op, L.t2sp_w4_pack(code, q.data_ptr(), scales.data_ptr(), zeros.data_ptr() if zeros is not None else None, E, N, K, group,
                                  _row(q), each(q), _row(scales), each(scales), _row(zeros) if zeros is not None else 0,
                                  each(zeros) if zeros is not None else 0, Q.data_ptr(), S.data_ptr(), Z.data_ptr() if Z is not None else None,
                                  _stream(q)))
    return W4(E if q.dim() == 3 else None, N, K, group, Q, S, Z)


def gemv_w4(x, w, ids=None, out=None):
    """y = x @ W.T for a few rows x (M, K) and 4-bit weights w (pack_w4), y (M, N) of x's type.

    With matrices for E experts, ids (M int32) picks the matrix of each row; a row whose id is outside 0 .. E - 1 is zeros."""
    import torch
    op = "gemv_w4"
    _need(op, x.dtype == w.S.dtype, BAD_TYPE)
    _need(op, x.dim() == 2, BAD_DIMENSIONS)
    M, K = x.shape
    _need(op, K == w.K and x.is_cuda and x.device == w.Q.device and (K <= 1 or x.stride(1) == 1) and (ids is None) == (w.E is None))
    if ids is not None:
        _need(op, ids.dtype == torch.int32, BAD_TYPE)
        _integers(op, ids, x, M)
    y = _result(op, out, (M, w.N), x, x.dtype, (x.dtype,))
    with _On(x):
        _check(op, lib().t2sp_gemv_w4(w.code, x.data_ptr(), w.Q.data_ptr(), w.S.data_ptr(), w.Z.data_ptr() if w.Z is not None else None,
                                      ids.data_ptr() if ids is not None else None, y.data_ptr(), M, w.N, K, w.E or 1, w.group, _row(x), _row(y),
                                      _stream(x)))
    return y
