"""GPU tests of the products grouped by expert in every form that a launch may take, and for offsets of any values.
Tolerances as derived in test_grouped_gpu.py."""
import numpy as np
import pytest

import t2sp_amd
import test_products_plans as plans
from test_grouped_gpu import TYPES, check_forward, check_wgrad, make, within

pytestmark = pytest.mark.gpu


def expect(X, W, D, offsets, opb):
    """Y and dW for offsets of any values: clamped, running maximum."""
    import torch
    T = X.shape[0]
    o = np.maximum.accumulate(np.clip(np.asarray(offsets, dtype=np.int64), 0, T))
    filled = torch.full((T, W.shape[1] if opb else W.shape[2]), 5.0, dtype=X.dtype, device="cuda")
    Y = t2sp_amd.gemm_grouped(X, W, torch.tensor(offsets, dtype=torch.int64).cuda(), opb=opb, out=filled)
    dW = t2sp_amd.gemm_grouped_wgrad(X, D, torch.tensor(offsets, dtype=torch.int64).cuda())
    outside = np.ones(T, bool)
    for e, (lo, hi) in enumerate(zip(o[:-1], o[1:])):
        x, d, w = X[lo:hi].double(), D[lo:hi].double(), W[e].double().t() if opb else W[e].double()
        within(Y[lo:hi], x @ w, x.abs() @ w.abs(), X.shape[1], Y.dtype)
        within(dW[e], x.t() @ d, x.abs().t() @ d.abs(), max(hi - lo, 1), dW.dtype)
        outside[lo:hi] = False
    assert (Y[torch.from_numpy(outside).cuda()] == 5).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("opb", [0, 1])
@pytest.mark.parametrize("T", [64, 700])
def test_offsets_that_decrease(dtype, opb, T):
    """A row belongs to the first group that reaches it; groups that overlap it otherwise are shorter or empty."""
    X, W, D = make((T, 64), dtype, 1), make((3, 72, 64) if opb else (3, 64, 72), dtype, 2), make((T, 72), dtype, 3)
    for o in ([0, 40, 20, 64], [50, 20, 30, 64], [0, T, 0, T], [T, 0, 0, 0], [-7, 30, 10, 1 << 40], [0, 10, 5, 3]):
        expect(X, W, D, o, opb)


@pytest.mark.parametrize("E", [5, 64, 65, 200])
@pytest.mark.parametrize("T", [90, 1500])
def test_offsets_of_any_values(E, T):
    """Every group reaches over most of the others': more row tiles than T rows can make, unless the rows are told apart."""
    rng = np.random.default_rng(E + T)
    X, W, D = make((T, 64), "bfloat16", 4), make((E, 64, 72), "bfloat16", 5), make((T, 72), "bfloat16", 6)
    expect(X, W, D, [(T if i % 2 else 0) for i in range(E + 1)], 0)
    expect(X, W, D, rng.integers(-T, 2 * T, E + 1).tolist(), 0)
    up = np.sort(rng.integers(0, T, E + 1))
    up[rng.integers(0, E + 1, 3)] = 0
    expect(X, W, D, up.tolist(), 0)


def on_full_card():
    """The tables of forms are for 256 compute units."""
    L = t2sp_amd.lib()
    if L.t2sp_machine_cus() != 256 or L.t2sp_machine_xcds() != 8:
        pytest.skip("the forms of these sizes are known for a full card only")
    return L


@pytest.mark.parametrize("case", range(len(plans.FORWARD)))
def test_every_form_of_the_product(case):
    """Results of the operands' type and in float; rows in front of and behind the groups are left."""
    import torch
    form, types, opb, sizes, K, N = plans.FORWARD[case]
    T, E = sum(sizes), len(sizes)
    for dtype in types:
        assert plans.forward_form(on_full_card(), dtype, opb, T, E, K, N) == form
        X, W = make((T, K), dtype, 1), make((E, N, K) if opb else (E, K, N), dtype, 2, K ** -0.5)
        check_forward(X, W, sizes, opb)
        if dtype != "float32":
            check_forward(X, W, sizes, opb, out_dtype=torch.float32)
        first = sizes[0] // 2                               # the same launch with the offsets moved: other rows per tile
        o = np.concatenate([[first], np.cumsum(sizes)])
        Y = torch.full((T, N), 3.0, dtype=X.dtype, device="cuda")
        t2sp_amd.gemm_grouped(X, W, torch.tensor(o, dtype=torch.int32).cuda(), opb=opb, out=Y)
        assert (Y[:first] == 3).all()
        within(Y[first:sizes[0]], X[first:sizes[0]].double() @ (W[0].double().t() if opb else W[0].double()),
               X[first:sizes[0]].double().abs() @ (W[0].double().abs().t() if opb else W[0].double().abs()), K, Y.dtype)


@pytest.mark.parametrize("case", range(len(plans.WGRAD)))
def test_every_form_of_the_gradient_of_the_matrices(case):
    import torch
    tile, parts, types, sizes, K, N = plans.WGRAD[case]
    T = sum(sizes)
    for dtype in types:
        assert plans.wgrad_form(on_full_card(), dtype, T, len(sizes), K, N) == (tile, parts)
        X, D = make((T, K), dtype, 3), make((T, N), dtype, 4)
        check_wgrad(X, D, sizes)
        if dtype != "float32":
            check_wgrad(X, D, sizes, out_dtype=torch.float32)
