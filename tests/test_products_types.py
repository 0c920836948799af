"""The result's type of the products of a language model's layers, for numpy arrays and tensors: the operands' type or float32,
as out_dtype or the type of `out` says; anything else is refused."""
import numpy as np
import pytest

import t2sp_amd


def code(f, *a, **k):
    with pytest.raises(t2sp_amd.T2spError) as e:
        f(*a, **k)
    return e.value.code


def test_host_results_have_the_type_asked_for():
    """Calls without rows end before any device work."""
    X, W, off = np.zeros((0, 8), np.float16), np.zeros((3, 8, 5), np.float16), np.zeros(4, np.int32)
    assert t2sp_amd.gemm_grouped(X, W, off).dtype == np.float16
    for t in (np.float32, "float32", np.dtype(np.float32)):
        assert t2sp_amd.gemm_grouped(X, W, off, out_dtype=t).dtype == np.float32
    assert t2sp_amd.gemm_grouped(X, W, off, out_dtype=np.float16).dtype == np.float16
    assert t2sp_amd.gemm_grouped(X.astype(np.float32), W.astype(np.float32), off, out_dtype=np.float32).dtype == np.float32


def test_host_types_that_are_refused():
    X, W, off = np.zeros((6, 8), np.float16), np.zeros((3, 8, 5), np.float16), np.zeros(4, np.int32)
    V, lab, lse = np.zeros((20, 8), np.float16), np.zeros(6, np.int64), np.zeros(6, np.float32)
    for bad in (np.float64, np.int32, "nothing", object()):
        assert code(t2sp_amd.gemm_grouped, X, W, off, out_dtype=bad) == -3
        assert code(t2sp_amd.gemm_grouped_wgrad, X, np.zeros((6, 5), np.float16), off, out_dtype=bad) == -3
        assert code(t2sp_amd.xent_grad, X, V, lab, lse, lse, out_dtype=bad) == -3
    assert code(t2sp_amd.gemm_grouped, X.astype(np.float32), W.astype(np.float32), off, out_dtype=np.float16) == -3
    assert code(t2sp_amd.gemm_grouped, X, W, off, out=np.zeros((6, 5), np.float16), out_dtype=np.float32) == -3
    assert code(t2sp_amd.xent_grad, X, V, lab, lse, lse, dH=np.zeros((6, 8), np.float16), out_dtype=np.float32) == -3
    assert code(t2sp_amd.xent_grad, X, V, lab, lse, lse, dH=np.zeros((6, 8), np.float16), dW=np.zeros((20, 8), np.float32)) == -3


@pytest.mark.gpu
def test_host_results_in_float():
    import torch
    rng = np.random.default_rng(0)
    X, W, D = (rng.standard_normal(s).astype(np.float16) for s in ((9, 24), (3, 24, 40), (9, 40)))
    off = np.array([0, 4, 4, 9], np.int32)
    dev = lambda a: torch.from_numpy(a).cuda()
    same = lambda a, b: a.dtype == np.float32 and np.array_equal(a, b.cpu().numpy())
    assert same(t2sp_amd.gemm_grouped(X, W, off, out_dtype=np.float32), t2sp_amd.gemm_grouped(dev(X), dev(W), dev(off), out_dtype=torch.float32))
    assert same(t2sp_amd.gemm_grouped_wgrad(X, D, off, out_dtype=np.float32),
                t2sp_amd.gemm_grouped_wgrad(dev(X), dev(D), dev(off), out_dtype=torch.float32))
    V, lab, d = rng.standard_normal((33, 24)).astype(np.float16), np.arange(9) * 3, np.full(9, 1 / 9, np.float32)
    _, lse = t2sp_amd.xent(X, V, lab)
    want = t2sp_amd.xent_grad(dev(X), dev(V), dev(lab), dev(lse), dev(d), out_dtype=torch.float32)
    for got in (t2sp_amd.xent_grad(X, V, lab, lse, d, out_dtype=np.float32), t2sp_amd.xent_grad(X, V, lab, lse, d, dW=np.empty((33, 24), np.float32))):
        assert same(got[0], want[0]) and same(got[1], want[1])


@pytest.mark.gpu
def test_a_result_of_another_type_than_asked_for_is_refused():
    import torch
    X, W = torch.zeros((4, 8), dtype=torch.bfloat16, device="cuda"), torch.zeros((1, 8, 8), dtype=torch.bfloat16, device="cuda")
    off = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    assert code(t2sp_amd.gemm_grouped, X, W, off, out=torch.empty_like(X), out_dtype=torch.float32) == -3
    assert code(t2sp_amd.gemm_grouped, X, W, off, out=torch.empty_like(X, dtype=torch.float32), out_dtype=torch.bfloat16) == -3
    assert code(t2sp_amd.gemm_grouped_wgrad, X, X, off, out=torch.empty_like(W), out_dtype=torch.float32) == -3
    lab, lse = torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(4, device="cuda")
    assert code(t2sp_amd.xent_grad, X, W[0], lab, lse, lse, dH=torch.empty_like(X), out_dtype=torch.float32) == -3
    out = torch.empty_like(X, dtype=torch.float32)
    assert t2sp_amd.gemm_grouped(X, W, off, out=out, out_dtype=torch.float32) is out


@pytest.mark.gpu
def test_host_arrays_without_rows():
    H, V, lab, none = np.zeros((0, 8), np.float32), np.ones((20, 8), np.float32), np.zeros(0, np.int64), np.zeros(0, np.float32)
    dH, dW = t2sp_amd.xent_grad(H, V, lab, none, none)
    assert dH.shape == (0, 8) and dW.shape == (20, 8) and (dW == 0).all()
    dW = t2sp_amd.gemm_grouped_wgrad(np.zeros((0, 8), np.float16), np.zeros((0, 5), np.float16), np.zeros(4, np.int32))
    assert dW.shape == (3, 8, 5) and (dW == 0).all()


def test_the_rounded_gradient_refuses_what_the_other_does():
    L = t2sp_amd.lib()
    if L.t2sp_device_count() > 0:
        pytest.skip("made-up addresses: for machines without a device")
    P = 0x7f0000000000
    names = ("type", "out", "H", "W", "l", "bits", "lse", "dl", "dH", "dW", "T", "V", "D", "ldh", "ldw", "lddh", "lddw", "ws", "wb", "st")
    good = dict(type=2, out=2, H=P, W=P, l=P, bits=64, lse=P, dl=P, dH=P, dW=P, T=8, V=100, D=64, ldh=64, ldw=64, lddh=64, lddw=64, ws=P, wb=1 << 40,
                st=None)
    for f in (L.t2sp_xent_grad, L.t2sp_xent_grad_rounded):
        call = lambda **k: f(*[dict(good, **k)[n] for n in names])
        for bad in (dict(type=3), dict(out=1), dict(bits=8), dict(T=-1), dict(V=0), dict(D=0), dict(ldh=63), dict(lddw=63), dict(H=None), dict(lse=None),
                    dict(ws=None), dict(ws=P + 8), dict(wb=1 << 10)):
            assert call(**bad) == -8, bad
        assert call(dH=None, dW=None) == 0 and call(T=0, dW=None) == 0
    sizes = [L.t2sp_xent_grad_workspace_bytes(t, P, P, 8192, 128000, 4096, 4096, 4096) for t in (0, 1, 2)]
    assert min(sizes) > 8192 * 4096 * 4 * 2 and max(sizes) < 2 << 30
