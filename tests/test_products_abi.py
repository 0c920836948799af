"""CPU-only checks of the products of a language model's layers (gemm_grouped, xent, gemv_w4): the entries and the thin
layer refuse misuse with a code before any device work, workspace sizes are what the calls ask for, the argument tables and
argv forms stand next to the entries, and no extents or strides make the host side end otherwise than with a code."""
import ctypes
import random

import numpy as np
import pytest

import t2sp_amd
from t2sp_amd.buffer import HalideBuffer
from test_abi import _metadata

F32, F16, BF16 = 0, 1, 2
P = 0x7f0000000000          # an aligned address that no call below may touch


def on_gpu():
    return t2sp_amd.lib().t2sp_device_count() > 0


def buf(shape, dtype=np.float32):
    return HalideBuffer.from_numpy(np.zeros(shape, dtype))


def test_grouped_entry_refusals():
    L = t2sp_amd.lib()
    x, w, o, y = buf((6, 8)), buf((3, 8, 5)), buf(4, np.int32), buf((6, 5))
    assert L.gemm_grouped(0, None, w.ref, o.ref, y.ref) == -12
    assert L.gemm_grouped(0, x.ref, w.ref, None, y.ref) == -12
    assert L.gemm_grouped(0, x.ref, w.ref, o.ref, None) == -12
    assert L.gemm_grouped(0, buf((6, 8), np.int32).ref, w.ref, o.ref, y.ref) == -3
    assert L.gemm_grouped(0, x.ref, buf((3, 8, 5), np.float16).ref, o.ref, y.ref) == -3        # one type for both
    assert L.gemm_grouped(0, x.ref, w.ref, buf(4).ref, y.ref) == -3                            # offsets are integers
    assert L.gemm_grouped(0, x.ref, w.ref, o.ref, buf((6, 5), np.float16).ref) == -3           # a float result cannot be half
    assert L.gemm_grouped(0, x.ref, buf((8, 5)).ref, o.ref, y.ref) == -43
    assert L.gemm_grouped(0, x.ref, w.ref, buf(5, np.int32).ref, y.ref) == -8                  # E + 1 offsets
    assert L.gemm_grouped(1, x.ref, w.ref, o.ref, y.ref) == -8                                 # W is (E, N, K) then
    assert L.gemm_grouped(0, x.ref, w.ref, o.ref, buf((5, 5)).ref) == -8
    assert L.gemm_grouped(0, x.ref, buf((0, 8, 5)).ref, buf(1, np.int32).ref, y.ref) == -8     # no matrices
    assert L.gemm_grouped(0, buf((0, 8)).ref, w.ref, o.ref, buf((0, 5)).ref) == 0              # no rows: nothing to do
    assert L.gemm_grouped_wgrad(x.ref, buf((5, 5)).ref, o.ref, buf((3, 8, 5)).ref) == -8
    assert L.gemm_grouped_wgrad(x.ref, y.ref, buf(3, np.int32).ref, buf((3, 8, 5)).ref) == -8
    assert L.gemm_grouped_wgrad(x.ref, None, o.ref, buf((3, 8, 5)).ref) == -12
    assert L.gemm_grouped_ns(0, None, w.ref, o.ref, y.ref) == -12.0


def test_xent_entry_refusals():
    L = t2sp_amd.lib()
    h, w, lab, v = buf((6, 8)), buf((20, 8)), buf(6, np.int64), buf(6)
    assert L.xent(None, w.ref, lab.ref, v.ref, v.ref) == -12
    assert L.xent(h.ref, buf((20, 7)).ref, lab.ref, v.ref, v.ref) == -8
    assert L.xent(h.ref, w.ref, buf(5, np.int64).ref, v.ref, v.ref) == -8
    assert L.xent(h.ref, w.ref, buf(6).ref, v.ref, v.ref) == -3
    assert L.xent(h.ref, w.ref, lab.ref, buf(6, np.float16).ref, v.ref) == -3                  # losses are float
    assert L.xent(h.ref, w.ref, lab.ref, v.ref, buf(7).ref) == -8
    assert L.xent(h.ref, buf((0, 8)).ref, lab.ref, v.ref, v.ref) == -8                         # no vocabulary
    assert L.xent(buf((0, 8)).ref, w.ref, buf(0, np.int64).ref, buf(0).ref, buf(0).ref) == 0
    assert L.xent_grad(h.ref, w.ref, lab.ref, v.ref, v.ref, buf((6, 8)).ref, buf((20, 7)).ref) == -8
    assert L.xent_grad(h.ref, w.ref, lab.ref, v.ref, buf(5).ref, buf((6, 8)).ref, buf((20, 8)).ref) == -8
    assert L.xent_grad(h.ref, w.ref, lab.ref, v.ref, v.ref, None, buf((20, 8)).ref) == -12
    hh, hw = buf((6, 8), np.float16), buf((20, 8), np.float16)
    assert L.xent_grad(hh.ref, hw.ref, lab.ref, v.ref, v.ref, buf((6, 8)).ref, buf((20, 8), np.float16).ref) == -3


def test_gemv_w4_entry_refusals():
    L = t2sp_amd.lib()
    x, q, s, y = buf((2, 70)), buf((5, 70), np.uint8), buf((5, 3)), buf((2, 5))
    assert L.gemv_w4(32, None, q.ref, s.ref, None, None, y.ref) == -12
    assert L.gemv_w4(32, x.ref, buf((5, 70)).ref, s.ref, None, None, y.ref) == -3
    for group in (0, -32, 16, 33, 48, 96):
        assert L.gemv_w4(group, x.ref, q.ref, s.ref, None, None, y.ref) == -8
    assert L.gemv_w4(64, x.ref, q.ref, s.ref, None, None, y.ref) == -8                         # two groups of 64
    assert L.gemv_w4(32, x.ref, q.ref, s.ref, buf((5, 2)).ref, None, y.ref) == -8
    assert L.gemv_w4(32, x.ref, q.ref, s.ref, None, buf(2, np.int32).ref, y.ref) == -43        # ids want (E, N, K)
    assert L.gemv_w4(32, x.ref, buf((3, 5, 70), np.uint8).ref, buf((3, 5, 3)).ref, None, buf(3, np.int32).ref, y.ref) == -8
    assert L.gemv_w4(32, buf((0, 70)).ref, q.ref, s.ref, None, None, buf((0, 5)).ref) == 0


def test_python_mirror_refuses_with_codes():
    def code(f, *a, **k):
        with pytest.raises(t2sp_amd.T2spError) as e:
            f(*a, **k)
        return e.value.code
    X, W, o = np.zeros((6, 8), np.float32), np.zeros((3, 8, 5), np.float32), np.zeros(4, np.int32)
    assert code(t2sp_amd.gemm_grouped, X, W, o.astype(np.float32)) == -3
    assert code(t2sp_amd.gemm_grouped, X, W[0], o) == -43
    assert code(t2sp_amd.gemm_grouped, X.astype(np.float64), W, o) == -3
    assert code(t2sp_amd.gemm_grouped_wgrad, X, X, np.zeros(1, np.int32)) == -8
    assert code(t2sp_amd.xent, X, np.zeros((9, 7), np.float32), np.zeros(6, np.int64)) == -8
    w = t2sp_amd.pack_w4(np.zeros((5, 64), np.uint8), np.zeros((5, 1), np.float32), group=64)
    assert code(t2sp_amd.gemv_w4, np.zeros((2, 63), np.float32), w) == -8
    assert code(t2sp_amd.gemv_w4, np.zeros((2, 64), np.float32), w, ids=np.zeros(2, np.int32)) == -8
    torch = pytest.importorskip("torch")                     # tensors that are not on a GPU
    assert code(t2sp_amd.gemm_grouped, torch.zeros(6, 8), torch.zeros(3, 8, 5), torch.zeros(4, dtype=torch.int32)) == -8
    assert code(t2sp_amd.gemm_grouped, torch.zeros(6, 8, dtype=torch.float64), torch.zeros(3, 8, 5), torch.zeros(4)) == -3
    assert code(t2sp_amd.xent, torch.zeros(6, 8), torch.zeros(9, 8), torch.zeros(6, dtype=torch.int64)) == -8


def test_thin_layer_refusals():
    if on_gpu():
        pytest.skip("made-up addresses: for machines without a device")
    L = t2sp_amd.lib()
    g = lambda **k: L.t2sp_gemm_grouped(*[dict(dict(type=BF16, out=BF16, opb=0, X=P, W=P, o=P, bits=32, Y=P, T=8, E=2, K=64, N=64, ldx=64, ldw=64,
                                                    sw=4096, ldy=64, ws=None, wb=0, st=None), **k)[n]
                                          for n in ("type", "out", "opb", "X", "W", "o", "bits", "Y", "T", "E", "K", "N", "ldx", "ldw", "sw", "ldy", "ws",
                                                    "wb", "st")])
    for bad in (dict(type=3), dict(type=-1), dict(out=F16), dict(bits=16), dict(T=-1), dict(E=0), dict(K=0), dict(N=0), dict(ldx=63), dict(ldw=63),
                dict(ldy=63), dict(sw=-1), dict(ldx=1 << 40), dict(X=None), dict(W=None), dict(o=None), dict(Y=None), dict(K=1 << 23, ldx=1 << 23),
                dict(X=P + 2), dict(K=63), dict(N=63), dict(X=P + 2, ws=P, wb=8 * 64 * 2 - 1), dict(X=P + 2, ws=P + 8, wb=1 << 20),
                dict(E=1 << 30, opb=1, N=8)):
        assert g(**bad) == -8, bad
    assert g(T=0) == 0 and g(T=0, X=None) == 0
    assert L.t2sp_gemm_grouped_workspace_bytes(BF16, 0, P, P, 8, 2, 64, 64, 64, 64, 4096) == 0
    assert L.t2sp_gemm_grouped_workspace_bytes(BF16, 0, P + 2, P, 8, 2, 64, 64, 64, 64, 4096) == 8 * 64 * 2
    assert L.t2sp_gemm_grouped_workspace_bytes(BF16, 0, P, P, 8, 2, 64, 63, 64, 63, 63 * 64) == 2 * 64 * 64 * 2
    assert L.t2sp_gemm_grouped_workspace_bytes(F32, 1, P, P, 8, 2, 6, 5, 6, 6, 30) == 8 * 8 * 4 + 2 * 5 * 8 * 4
    w = lambda **k: L.t2sp_gemm_grouped_wgrad(*[dict(dict(type=F16, out=F32, X=P, dY=P, o=P, bits=64, dW=P, T=8, E=2, K=64, N=32, ldx=64, ldy=32, ldw=32,
                                                          sw=2048, ws=None, wb=0, st=None), **k)[n]
                                                for n in ("type", "out", "X", "dY", "o", "bits", "dW", "T", "E", "K", "N", "ldx", "ldy", "ldw", "sw", "ws",
                                                          "wb", "st")])
    for bad in (dict(type=7), dict(out=BF16), dict(bits=0), dict(E=0), dict(sw=2047), dict(ldw=31), dict(dW=None), dict(o=None), dict(dY=None),
                dict(N=31, ldy=31), dict(dY=P + 2)):
        assert w(**bad) == -8, bad
    x = lambda **k: L.t2sp_xent(*[dict(dict(type=BF16, H=P, W=P, l=P, bits=64, loss=P, lse=P, T=8, V=100, D=64, ldh=64, ldw=64, ws=P, wb=1 << 30, st=None),
                                       **k)[n] for n in ("type", "H", "W", "l", "bits", "loss", "lse", "T", "V", "D", "ldh", "ldw", "ws", "wb", "st")])
    need = L.t2sp_xent_workspace_bytes(BF16, P, P, 8, 100, 64, 64, 64)
    assert need > 0
    for bad in (dict(type=9), dict(bits=8), dict(T=-1), dict(V=0), dict(D=0), dict(ldh=63), dict(ldw=63), dict(H=None), dict(W=None), dict(l=None),
                dict(loss=None), dict(ws=None), dict(wb=need - 1), dict(ws=P + 4)):
        assert x(**bad) == -8, bad
    assert x(T=0) == 0
    gr = lambda **k: L.t2sp_xent_grad(*[dict(dict(type=BF16, out=BF16, H=P, W=P, l=P, bits=64, lse=P, dl=P, dH=P, dW=P, T=8, V=100, D=64, ldh=64, ldw=64,
                                                  lddh=64, lddw=64, ws=P, wb=1 << 40, st=None), **k)[n]
                                        for n in ("type", "out", "H", "W", "l", "bits", "lse", "dl", "dH", "dW", "T", "V", "D", "ldh", "ldw", "lddh", "lddw",
                                                  "ws", "wb", "st")])
    for bad in (dict(out=F16), dict(lddh=63), dict(lddw=63), dict(lse=None), dict(dl=None), dict(wb=100), dict(ws=None)):
        assert gr(**bad) == -8, bad
    assert gr(dH=None, dW=None) == 0 and gr(T=0, dW=None) == 0
    qb, se = ctypes.c_int64(), ctypes.c_int64()
    assert L.t2sp_w4_sizes(17, 129, 32, ctypes.byref(qb), ctypes.byref(se)) == 0
    assert qb.value == 2 * 2 * 1024 and se.value == 2 * 16 * 8
    assert L.t2sp_w4_sizes(16, 1024, 256, ctypes.byref(qb), ctypes.byref(se)) == 0 and se.value == 16 * 4
    for bad in ((0, 64, 32), (16, 0, 32), (16, 64, 0), (16, 64, 31), (16, 64, 16), (16, 64, 96)):
        assert L.t2sp_w4_sizes(*bad, ctypes.byref(qb), ctypes.byref(se)) == -8
    v = lambda **k: L.t2sp_gemv_w4(*[dict(dict(type=BF16, x=P, Q=P, S=P, Z=None, ids=None, y=P, M=2, N=16, K=64, E=1, group=64, ldx=64, ldy=16, st=None),
                                          **k)[n] for n in ("type", "x", "Q", "S", "Z", "ids", "y", "M", "N", "K", "E", "group", "ldx", "ldy", "st")])
    for bad in (dict(type=3), dict(M=-1), dict(E=0), dict(E=2), dict(group=33), dict(ldx=63), dict(ldy=15), dict(x=None), dict(Q=None), dict(S=None),
                dict(y=None), dict(Q=P + 8), dict(S=P + 8), dict(Z=P + 8), dict(M=65536, ids=P), dict(ldx=1 << 23)):
        assert v(**bad) == -8, bad
    assert v(M=0) == 0


def test_thin_layer_survives_random_extents_and_strides():
    if on_gpu():
        pytest.skip("made-up addresses: for machines without a device")
    L = t2sp_amd.lib()
    rng = random.Random(5)
    ext = [0, 1, 2, 7, 8, 63, 64, 100, 1000, 4096, 65535, 1 << 20, 1 << 22, 1 << 23, 1 << 30, (1 << 31) - 1, -1]
    strd = [0, 1, 7, 8, 64, 4096, 1 << 20, 1 << 23, 1 << 31, (1 << 31) + 1, 1 << 40, -1]
    e, s = lambda: rng.choice(ext), lambda: rng.choice(strd)
    p = lambda: rng.choice([None, P, P, P + 2, P + 16])
    for _ in range(4000):
        t, ot, b = rng.randint(-1, 3), rng.randint(-1, 3), rng.choice([32, 64, 8])
        wb = rng.choice([0, 1 << 20, 1 << 50])
        rcs = [L.t2sp_gemm_grouped(t, ot, rng.randint(0, 1), p(), p(), p(), b, p(), e(), e(), e(), e(), s(), s(), s(), s(), p(), wb, None),
               L.t2sp_gemm_grouped_wgrad(t, ot, p(), p(), p(), b, p(), e(), e(), e(), e(), s(), s(), s(), s(), p(), wb, None),
               L.t2sp_xent(t, p(), p(), p(), b, p(), p(), e(), e(), e(), s(), s(), p(), wb, None),
               L.t2sp_xent_grad(t, ot, p(), p(), p(), b, p(), p(), p(), p(), e(), e(), e(), s(), s(), s(), s(), p(), wb, None),
               L.t2sp_gemv_w4(t, p(), p(), p(), p(), p(), p(), e(), e(), e(), e(), rng.choice([32, 64, 128, 1 << 25, 1 << 26, 5]), s(), s(), None),
               L.t2sp_w4_pack(t, p(), p(), p(), e(), e(), e(), rng.choice([32, 64, 128, 5]), s(), s(), s(), s(), s(), s(), p(), p(), p(), None)]
        assert all(rc <= 0 for rc in rcs), rcs
        assert L.t2sp_xent_grad_workspace_bytes(t, p(), p(), e(), e(), e(), s(), s()) >= 0


def test_tables_and_argv_forms():
    L = t2sp_amd.lib()
    names = {"gemm_grouped": (5, 4), "gemm_grouped_wgrad": (4, 3), "xent": (5, 3), "xent_grad": (7, 5), "gemv_w4": (7, 6)}
    for fn, (args, inputs) in names.items():
        m = _metadata(L, fn)
        assert len(m) == args and [a[1] == 2 for a in m] == [False] * inputs + [True] * (args - inputs)
        assert getattr(L, fn + "_argv")(None) == -12
    arr = (ctypes.c_void_p * 4)(None, None, None, None)
    assert L.gemm_grouped_wgrad_argv(arr) == -12


def test_workspace_of_the_matrices_gradient():
    """Planes for sums in parts (few small matrices, many rows); none for many tiles or few rows, up to the largest extents."""
    L, big = t2sp_amd.lib(), 1 << 30
    size = lambda T, E, K, N: L.t2sp_gemm_grouped_wgrad_workspace_bytes(BF16, P, P, T, E, K, N, K, N)
    parts, rest = divmod(size(8192, 1, 512, 512), 512 * 512 * 4)
    assert parts >= 2 and rest == 0
    assert size(8192, 64, 2048, 2048) == 0 and size(64, 1, 512, 512) == 0 and size(0, 1, 512, 512) == 0
    assert size(0, big, big, big) == 0
