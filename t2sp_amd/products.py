"""Python mirror of the products of a language model's layers (include/t2sp_hip.h, second half): products
grouped by expert, cross entropy over a vocabulary, products with 4-bit weights.

torch CUDA tensors go to the thin layer: kernels are enqueued on the current stream of the tensors' device and
the call returns without waiting, so it can be captured into a HIP graph; workspaces and fresh results come from
torch's allocator, which keeps them apart between streams and captured graphs.  Element types are float32, float16
and bfloat16.  numpy arrays (float32 or float16, host memory) go through the operator entries
(include/gemm_grouped-interface.h, xent-interface.h, gemv_w4-interface.h), which stage them through the device.
Rows of a matrix may lie any distance apart but must not overlap (an expanded tensor is refused with -8: pass a copy).
Results carry no autograd graph, whatever their operands require; the gradients are calls of their own.
Misuse raises T2spError with the Halide error code that the entry would return."""
import ctypes

import numpy as np

from ._lib import lib
from .buffer import HalideBuffer, NUMPY_TYPES
from .ops import T2spError, _check, _is_torch, host_empty

BAD_TYPE, SHAPE, BAD_DIMENSIONS = -3, -8, -43
_F32 = 0                                     # T2SP_TYPE_F32
_MAX_ROW_BYTES = 1 << 23                     # T2SP_MAX_ROW_BYTES
_codes = None                                # torch dtype -> T2SP_TYPE_*; set with the other torch names on first use


def _torch():
    """Names of torch that every call needs (the package itself imports without torch)."""
    global _codes, _int_bits, _current_device, _set_device, _raw_stream, torch
    if _codes is None:
        import torch
        _int_bits = {torch.int32: 32, torch.int64: 64}
        # a call's cost on the host is a good part of a small product's: the plain numbers, where torch has them, save
        # 2 us of the 4 that current_stream() and current_device() take
        _current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
        _set_device = torch.cuda.set_device
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
        if torch.cuda.is_available():
            torch.cuda.init()
        _codes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    return _codes


def _need(op, ok, code=SHAPE):
    if not ok:
        raise T2spError(op, code)


def _tensors(op, dims, *tensors):
    """Common checks of floating-point CUDA tensors: one element type, one device, the stated ranks, unit stride along
    the last axis.  Returns the T2SP_TYPE_* code and the device's index."""
    first = tensors[0]
    code, index = _torch().get(first.dtype), first.get_device()
    if code is None:
        raise T2spError(op, BAD_TYPE)
    for t, d in zip(tensors, dims):
        if t.dtype is not first.dtype:
            raise T2spError(op, BAD_TYPE)
        if t.dim() != d:
            raise T2spError(op, BAD_DIMENSIONS)
        if index < 0 or t.get_device() != index or (t.stride(-1) != 1 and t.shape[-1] > 1):
            raise T2spError(op, SHAPE)
    return code, index


def _vector(op, t, types, index, n):
    """Checks a contiguous vector of n elements on the device; returns types[its dtype]."""
    kind = types.get(t.dtype)
    _need(op, kind is not None, BAD_TYPE)
    _need(op, t.dim() == 1, BAD_DIMENSIONS)
    _need(op, t.get_device() == index and t.shape[0] == n and (n <= 1 or t.stride(0) == 1))
    return kind


def _result(op, out, shape, like, dtype=None):
    """(result, its T2SP_TYPE_*): `out` checked, or a fresh one of `dtype` (the type of `like`); that type or float32."""
    if out is None:
        if dtype is None or dtype is like.dtype:
            return like.new_empty(shape), _codes[like.dtype]
        _need(op, dtype is torch.float32, BAD_TYPE)
        return like.new_empty(shape, dtype=dtype), _F32
    _need(op, (out.dtype is like.dtype or out.dtype is torch.float32) and (dtype is None or dtype is out.dtype), BAD_TYPE)
    _need(op, out.dim() == len(shape), BAD_DIMENSIONS)
    _need(op, tuple(out.shape) == shape and out.get_device() == like.get_device() and (shape[-1] <= 1 or out.stride(-1) == 1))
    return out, _codes[out.dtype]


def _row(t):
    """Elements between rows (a single row's stride carries no information)."""
    return t.stride(-2) if t.shape[-2] > 1 else t.shape[-1]


def _matrix(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * _row(t)


class _On:
    """Makes device `index` current around a call (used when it is not)."""

    def __init__(self, index, back):
        self.index, self.back = index, back

    def __enter__(self):
        _set_device(self.index)

    def __exit__(self, *exc):
        _set_device(self.back)


def _room(like, nbytes):
    """A workspace, or None.  Its owner may be dropped after the call: torch's allocator hands the memory out again only to
    work that is ordered behind it."""
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


# ---------------------------------------------------------------------------------------------- numpy: the operator entries
def _entry(op, *args):
    wrapped = [HalideBuffer.wrap(a) if isinstance(a, np.ndarray) else a for a in args]
    _check(op, getattr(lib(), op)(*[a.ref if isinstance(a, HalideBuffer) else a for a in wrapped]))


def _host_out(op, out, shape, like, dtype=None):
    """`out`, or a fresh array of `dtype` (`like`, the operands' type); that type or float32."""
    if dtype is not None:
        try:
            dtype = np.dtype(dtype)
        except TypeError:
            raise T2spError(op, BAD_TYPE)
        _need(op, dtype == like or dtype == np.float32, BAD_TYPE)
    if out is None:
        dtype = dtype or like
        return host_empty(shape) if dtype == np.float32 else np.empty(shape, dtype)
    _need(op, isinstance(out, np.ndarray) and (dtype is None or dtype == out.dtype), BAD_TYPE)
    return out


def _host_arrays(op, *arrays):
    for a in arrays:
        _need(op, isinstance(a, np.ndarray) and a.dtype.name in NUMPY_TYPES, BAD_TYPE)


def _host_grouped(op, X, W, offsets, opb, out, dtype):
    _host_arrays(op, X, W, offsets)
    _need(op, X.ndim == 2 and W.ndim == 3, BAD_DIMENSIONS)
    Y = _host_out(op, out, (X.shape[0], W.shape[1] if opb else W.shape[2]), X.dtype, dtype)
    _entry(op, int(bool(opb)), X, W, offsets, Y)
    return Y


def _host_wgrad(op, X, dY, offsets, out, dtype):
    _host_arrays(op, X, dY, offsets)
    _need(op, X.ndim == 2 and dY.ndim == 2 and offsets.ndim == 1, BAD_DIMENSIONS)
    _need(op, offsets.shape[0] >= 2)
    dW = _host_out(op, out, (offsets.shape[0] - 1, X.shape[1], dY.shape[1]), X.dtype, dtype)
    _entry(op, X, dY, offsets, dW)
    return dW


def _host_xent(op, H, W, labels, loss, lse):
    _host_arrays(op, H, W, labels)
    _need(op, H.ndim == 2, BAD_DIMENSIONS)
    loss, lse = (_host_out(op, t, (H.shape[0],), np.float32) for t in (loss, lse))
    _entry(op, H, W, labels, loss, lse)
    return loss, lse


def _host_xent_grad(op, H, W, labels, lse, dloss, dH, dW, dtype):
    _host_arrays(op, H, W, labels, lse, dloss)
    if dtype is None:
        dtype = getattr(dH if dH is not None else dW, "dtype", None)
    dH, dW = _host_out(op, dH, H.shape, H.dtype, dtype), _host_out(op, dW, W.shape, H.dtype, dtype)
    _entry(op, H, W, labels, lse, dloss, dH, dW)
    return dH, dW


def _host_gemv_w4(op, x, w, ids, out):
    _host_arrays(op, x, *(() if ids is None else (ids,)))
    _need(op, x.ndim == 2, BAD_DIMENSIONS)
    _need(op, (ids is None) == (w.E is None) and isinstance(w.Q, np.ndarray))
    y = _host_out(op, out, (x.shape[0], w.N), x.dtype)
    _entry(op, w.group, x, w.Q, w.S, w.Z, ids, y)
    return y


# ---------------------------------------------------------------------------------------------- torch: the thin layer
def gemm_grouped(X, W, offsets, opb=0, out=None, out_dtype=None):
    """Y[r] = X[r] @ op(W[e]) for the rows offsets[e] <= r < offsets[e + 1] of group e.

    X: (T, K) rows sorted by group; W: (E, K, N), or (E, N, K) when opb; offsets: E + 1 int32 or int64 on the device,
    not decreasing (they are clamped to 0 .. T and taken as their running maximum).  Y: (T, N) of X's type, or float32 (out_dtype, or the type of `out`).
    Rows outside every group are left as they were (in a fresh result: whatever its memory held).  The gradient of X is
    gemm_grouped(dY, W, offsets, opb=1 - opb)."""
    op = "gemm_grouped"
    if not _is_torch(X):
        return _host_grouped(op, X, W, offsets, opb, out, out_dtype)
    code, index = _tensors(op, (2, 3), X, W)
    (T, K), (E, N) = X.shape, W.shape[:2]
    opb = 1 if opb else 0
    if opb:
        _need(op, W.shape[2] == K)
    else:
        _need(op, N == K)
        N = W.shape[2]
    _need(op, E >= 1 and K >= 1 and N >= 1)
    bits = _vector(op, offsets, _int_bits, index, E + 1)
    Y, out_code = _result(op, out, (T, N), X, out_dtype)
    back = _current_device()
    if back != index:
        with _On(index, back):
            return gemm_grouped(X, W, offsets, opb, Y)
    L = lib()
    x, w, ldx, ldw, sw = X.data_ptr(), W.data_ptr(), _row(X), _row(W), _matrix(W)
    nbytes = L.t2sp_gemm_grouped_workspace_bytes(code, opb, x, w, T, E, K, N, ldx, ldw, sw)
    room = _room(X, nbytes)
    _check(op, L.t2sp_gemm_grouped(code, out_code, opb, x, w, offsets.data_ptr(), bits, Y.data_ptr(), T, E, K, N, ldx, ldw, sw, _row(Y),
                                   room.data_ptr() if nbytes else None, nbytes, _raw_stream(index)))
    return Y


def gemm_grouped_wgrad(X, dY, offsets, out=None, out_dtype=None):
    """dW[e] = X_e.T @ dY_e over the rows offsets[e] <= r < offsets[e + 1] of each group, zeros for an empty one.

    X: (T, K), dY: (T, N), offsets as in gemm_grouped.  dW: (E, K, N) of X's type, or float32."""
    op = "gemm_grouped_wgrad"
    if not _is_torch(X):
        return _host_wgrad(op, X, dY, offsets, out, out_dtype)
    code, index = _tensors(op, (2, 2), X, dY)
    T, K = X.shape
    N, E = dY.shape[1], offsets.shape[0] - 1 if offsets.dim() else 0
    _need(op, dY.shape[0] == T and E >= 1 and K >= 1 and N >= 1)
    bits = _vector(op, offsets, _int_bits, index, E + 1)
    dW, out_code = _result(op, out, (E, K, N), X, out_dtype)
    back = _current_device()
    if back != index:
        with _On(index, back):
            return gemm_grouped_wgrad(X, dY, offsets, dW)
    L = lib()
    x, dy, ldx, ldy = X.data_ptr(), dY.data_ptr(), _row(X), _row(dY)
    nbytes = L.t2sp_gemm_grouped_wgrad_workspace_bytes(code, x, dy, T, E, K, N, ldx, ldy)
    room = _room(X, nbytes)
    _check(op, L.t2sp_gemm_grouped_wgrad(code, out_code, x, dy, offsets.data_ptr(), bits, dW.data_ptr(), T, E, K, N, ldx, ldy, _row(dW),
                                         _matrix(dW), room.data_ptr() if nbytes else None, nbytes, _raw_stream(index)))
    return dW


def _xent_args(op, H, W, labels):
    code, index = _tensors(op, (2, 2), H, W)
    T, D = H.shape
    V = W.shape[0]
    _need(op, W.shape[1] == D and D >= 1 and V >= 1)
    return code, index, T, V, D, _vector(op, labels, _int_bits, index, T)


def _floats(op, t, index, n):
    _vector(op, t, {torch.float32: 32}, index, n)
    return t


def xent(H, W, labels, loss=None, lse=None):
    """Cross entropy of a softmax over a vocabulary, from hidden states: (loss, lse), float32 vectors of one value per token.

    H: (T, D), W: (V, D), labels: T int32 or int64; z = H @ W.T is not kept.  lse[t] = log sum exp z[t],
    loss[t] = lse[t] - z[t, labels[t]], 0 where the label is outside 0 .. V - 1."""
    op = "xent"
    if not _is_torch(H):
        return _host_xent(op, H, W, labels, loss, lse)
    code, index, T, V, D, bits = _xent_args(op, H, W, labels)
    loss = H.new_empty(T, dtype=torch.float32) if loss is None else _floats(op, loss, index, T)
    lse = H.new_empty(T, dtype=torch.float32) if lse is None else _floats(op, lse, index, T)
    back = _current_device()
    if back != index:
        with _On(index, back):
            return xent(H, W, labels, loss, lse)
    L = lib()
    h, w, ldh, ldw = H.data_ptr(), W.data_ptr(), _row(H), _row(W)
    nbytes = L.t2sp_xent_workspace_bytes(code, h, w, T, V, D, ldh, ldw)
    room = _room(H, nbytes)
    _check(op, L.t2sp_xent(code, h, w, labels.data_ptr(), bits, loss.data_ptr(), lse.data_ptr(), T, V, D, ldh, ldw,
                           room.data_ptr() if nbytes else None, nbytes, _raw_stream(index)))
    return loss, lse


def xent_grad(H, W, labels, lse, dloss, dH=None, dW=None, out_dtype=None, wanted=(True, True), rounded=False):
    """Gradients (dH, dW) of sum_t dloss[t] * loss[t] (see xent): dH = g @ W, dW = g.T @ H with
    g[t, v] = (exp(z[t, v] - lse[t]) - [v == labels[t]]) * dloss[t]; tokens without a label take no part.

    lse: what xent returned; dloss: T float32.  The results have H's type, or float32 (out_dtype, or the type of dH / dW).
    `wanted` leaves one out (its place in the result is None; numpy arrays: both are computed).
    16-bit types: g enters the products with 16 (bfloat16) or 22 (half) of a float's 24 bits, as the sum of two numbers of
    the type.  rounded=True takes it rounded to one, for up to a third less time and an error of half a step of the type in every g
    (tensors only).  float16: in dW, tokens whose weight |dloss| max |H[t]| is below 2^-30 of the heaviest's lose bits."""
    op = "xent_grad"
    if not _is_torch(H):
        return _host_xent_grad(op, H, W, labels, lse, dloss, dH, dW, out_dtype)
    code, index, T, V, D, bits = _xent_args(op, H, W, labels)
    _floats(op, lse, index, T)
    _floats(op, dloss, index, T)
    out_code = None
    dtype = out_dtype or (dH.dtype if dH is not None else dW.dtype if dW is not None else None)
    if wanted[0] or dH is not None:
        dH, out_code = _result(op, dH, (T, D), H, dtype)
    if wanted[1] or dW is not None:
        dW, other = _result(op, dW, (V, D), H, dtype)
        _need(op, out_code in (None, other), BAD_TYPE)
        out_code = other
    if out_code is None:
        return None, None
    back = _current_device()
    if back != index:
        with _On(index, back):
            return xent_grad(H, W, labels, lse, dloss, dH, dW, wanted=(False, False), rounded=rounded)      # (what is wanted is allocated by now)
    L = lib()
    h, w, ldh, ldw = H.data_ptr(), W.data_ptr(), _row(H), _row(W)
    nbytes = L.t2sp_xent_grad_workspace_bytes(code, h, w, T, V, D, ldh, ldw)
    room = _room(H, nbytes)
    grad = L.t2sp_xent_grad_rounded if rounded else L.t2sp_xent_grad
    _check(op, grad(code, out_code, h, w, labels.data_ptr(), bits, lse.data_ptr(), dloss.data_ptr(),
                    dH.data_ptr() if dH is not None else None, dW.data_ptr() if dW is not None else None, T, V, D, ldh, ldw,
                    _row(dH) if dH is not None else D, _row(dW) if dW is not None else D,
                    room.data_ptr() if nbytes else None, nbytes, _raw_stream(index)))
    return dH, dW


class W4:
    """Matrices of 4-bit numbers in the layout of the kernels (pack_w4): E matrices of N x K, or one (E is None)."""

    def __init__(self, E, N, K, group, Q, S, Z):
        self.E, self.N, self.K, self.group, self.Q, self.S, self.Z = E, N, K, group, Q, S, Z
        if isinstance(Q, np.ndarray):        # host arrays as they are: the entry lays them out on the device
            return
        self.dtype, self.code, self.index = S.dtype, _torch()[S.dtype], S.get_device()
        self.max_ld = _MAX_ROW_BYTES // S.element_size()
        self.pointers = Q.data_ptr(), S.data_ptr(), Z.data_ptr() if Z is not None else None


def pack_w4(q, scales, zeros=None, group=128):
    """Lays 4-bit numbers out for gemv_w4, once: W[n, k] = (q[n, k] - zeros[n, k // group]) * scales[n, k // group], with
    zeros = 8 when there are none.

    q: uint8 (N, K), or (E, N, K) for E matrices, one number in the low four bits of each byte; scales, zeros:
    (..., N, ceil(K / group)) of the type of the rows they will meet (float32, float16 or bfloat16).  group: a power of two
    from 32 on; at least K for one scale per row."""
    op = "pack_w4"
    if not _is_torch(q):
        _host_arrays(op, q, scales, *(() if zeros is None else (zeros,)))
        _need(op, q.ndim in (2, 3), BAD_DIMENSIONS)
        return W4(q.shape[0] if q.ndim == 3 else None, q.shape[-2], q.shape[-1], int(group), q, scales, zeros)
    code, index = _tensors(op, (q.dim(),) * 2, *((scales,) if zeros is None else (scales, zeros)))
    _need(op, q.dtype is torch.uint8, BAD_TYPE)
    _need(op, q.dim() in (2, 3), BAD_DIMENSIONS)
    _need(op, q.get_device() == index and (q.shape[-1] <= 1 or q.stride(-1) == 1))
    N, K = q.shape[-2:]
    group = int(group)
    qb, se = ctypes.c_int64(), ctypes.c_int64()
    L = lib()
    _check(op, L.t2sp_w4_sizes(N, K, group, ctypes.byref(qb), ctypes.byref(se)))
    E = q.shape[0] if q.dim() == 3 else 1
    want = tuple(q.shape[:-1]) + (-(-K // group),)
    _need(op, E >= 1 and tuple(scales.shape) == want and (zeros is None or tuple(zeros.shape) == want))
    Q = q.new_empty(E * qb.value)
    S = scales.new_empty(E * se.value)
    Z = torch.empty_like(S) if zeros is not None else None
    each = lambda t: _matrix(t) if t.dim() == 3 else 0
    with _On(index, _current_device()):
        _check(op, L.t2sp_w4_pack(code, q.data_ptr(), scales.data_ptr(), zeros.data_ptr() if zeros is not None else None, E, N, K, group,
                                  _row(q), each(q), _row(scales), each(scales), _row(zeros) if zeros is not None else 0,
                                  each(zeros) if zeros is not None else 0, Q.data_ptr(), S.data_ptr(), Z.data_ptr() if Z is not None else None,
                                  _raw_stream(index)))
    return W4(E if q.dim() == 3 else None, N, K, group, Q, S, Z)


def gemv_w4(x, w, ids=None, out=None):
    """y = x @ W.T for a few rows x (M, K) and 4-bit weights w (pack_w4), y (M, N) of x's type.

    With matrices for E experts, ids (M int32) picks the matrix of each row; a row whose id is outside 0 .. E - 1 is zeros."""
    op = "gemv_w4"
    if not _is_torch(x):
        return _host_gemv_w4(op, x, w, ids, out)
    if x.dtype is not getattr(w, "dtype", None):
        raise T2spError(op, BAD_TYPE)
    if x.dim() != 2:
        raise T2spError(op, BAD_DIMENSIONS)
    (M, K), index = x.shape, w.index
    ldx = x.stride(0) if M > 1 else K
    if ldx > w.max_ld:                       # (rows that lie further apart than the kernel reaches, such as every sequence's last one)
        x, ldx = x.contiguous(), K
    if K != w.K or x.get_device() != index or (x.stride(1) != 1 and K > 1) or (ids is None) != (w.E is None):
        raise T2spError(op, SHAPE)
    if ids is not None:
        _vector(op, ids, {torch.int32: 32}, index, M)
    if out is None:
        out, ldy = x.new_empty((M, w.N)), w.N
    else:
        _need(op, out.dtype is x.dtype, BAD_TYPE)
        _result(op, out, (M, w.N), x)
        ldy = _row(out)
    back = _current_device()
    if back != index:
        with _On(index, back):
            return gemv_w4(x, w, ids, out)
    Q, S, Z = w.pointers
    _check(op, lib().t2sp_gemv_w4(w.code, x.data_ptr(), Q, S, Z, None if ids is None else ids.data_ptr(), out.data_ptr(), M, w.N, K, w.E or 1, w.group,
                                  ldx, ldy, _raw_stream(index)))
    return out
