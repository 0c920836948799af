"""GPU tests of the products grouped by expert (gemm_grouped, gemm_grouped_wgrad) against float64.

Tolerances.  Operands are exact in their type, products of two 16-bit elements are exact in float32 (8 + 8 and 11 + 11
bits of mantissa against 24; a product of two floats rounds once).  A sum of n terms in float32 in any order is off by at
most (n - 1 + r) u / (1 - (n + r) u) * sum |a b| with u = 2^-24 and r = 1 for rounded products (Higham, Accuracy and
Stability of Numerical Algorithms, section 3.1).  The rounding to the result's type adds half a step of the value: u_T
|y|, u_T = 2^-8 for bfloat16, 2^-11 for half (eps / 2), nothing for float, and half the smallest step where results are
subnormal."""
import numpy as np
import pytest

import t2sp_amd

pytestmark = pytest.mark.gpu
TYPES = ["float32", "float16", "bfloat16"]


def dt(name):
    import torch
    return getattr(torch, name)


def make(shape, dtype, seed, std=1.0):
    import torch
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dt(dtype)).cuda()


def offs(sizes, start=0, bits=32):
    import torch
    return torch.tensor(np.concatenate([[start], start + np.cumsum(sizes)]), dtype=torch.int32 if bits == 32 else torch.int64).cuda()


def within(got, want, mag, n, out_type):
    """got against the float64 value `want` with `mag` = sum |a b| over n terms."""
    import torch
    u = 2.0 ** -24
    bound = (n + 1) * u / (1 - (n + 1) * u) * mag
    if out_type != torch.float32:
        bound = bound + torch.finfo(out_type).eps / 2 * (want.abs() + bound) + torch.finfo(out_type).smallest_normal * torch.finfo(out_type).eps / 2
    err = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all()
    assert (err <= bound).all(), float((err / bound.clamp(min=1e-300)).max())


def check_forward(X, W, sizes, opb, start=0, **kw):
    import torch
    o = offs(sizes, start)
    Y = t2sp_amd.gemm_grouped(X, W, o, opb=opb, **kw)
    at = start
    for e, m in enumerate(sizes):
        Wd = W[e].double().t() if opb else W[e].double()
        x = X[at:at + m].double()
        within(Y[at:at + m], x @ Wd, x.abs() @ Wd.abs(), X.shape[1], Y.dtype)
        at += m
    return Y


def check_wgrad(X, dY, sizes, start=0, **kw):
    o = offs(sizes, start)
    dW = t2sp_amd.gemm_grouped_wgrad(X, dY, o, **kw)
    at = start
    for e, m in enumerate(sizes):
        x, d = X[at:at + m].double(), dY[at:at + m].double()
        within(dW[e], x.t() @ d, x.abs().t() @ d.abs(), max(m, 1), dW.dtype)
        if m == 0:
            assert (dW[e] == 0).all()
        at += m


SIZES = [([1], 64, 64), ([5], 8, 8), ([3, 0, 1, 7], 96, 72), ([0, 0, 130, 0], 64, 136), ([40, 300, 17], 264, 520), ([257, 256, 255, 1], 136, 264),
         ([700, 900], 64, 1024)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("opb", [0, 1])
@pytest.mark.parametrize("sizes,K,N", SIZES)
def test_forward(dtype, opb, sizes, K, N):
    E, T = len(sizes), sum(sizes)
    check_forward(make((T, K), dtype, 1), make((E, N, K) if opb else (E, K, N), dtype, 2), sizes, opb)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes,K,N", SIZES)
def test_wgrad(dtype, sizes, K, N):
    T = sum(sizes)
    check_wgrad(make((T, K), dtype, 3), make((T, N), dtype, 4), sizes)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("opb", [0, 1])
@pytest.mark.parametrize("K,N", [(1, 1), (7, 3), (65, 40), (40, 65), (101, 333)])
def test_sizes_off_the_vector_grid(dtype, opb, K, N):
    sizes = [9, 0, 131, 1]
    X, W = make((141, K), dtype, 5), make((4, N, K) if opb else (4, K, N), dtype, 6)
    check_forward(X, W, sizes, opb)
    check_wgrad(X, make((141, N), dtype, 7), sizes)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strided_and_unaligned_views(dtype):
    import torch
    X0, W0, D0 = make((90, 80), dtype, 8), make((3, 66, 104), dtype, 9), make((90, 120), dtype, 10)
    sizes = [30, 20, 39]
    for dx, dw in ((0, 0), (1, 0), (0, 1), (3, 5), (8, 16)):
        X, W, D = X0[:, dx:dx + 64], W0[:, 1:65, dw:dw + 72], D0[:, dw:dw + 72]
        check_forward(X, W, sizes, 0, start=1)
        check_wgrad(X, D, sizes, start=1)
        check_forward(D, W, sizes, 1, start=1)
    out = torch.full((90, 200), 7.0, dtype=dt(dtype), device="cuda")
    view = out[:, 3:75]                                     # rows of the result that start off the 16-byte grid
    got = t2sp_amd.gemm_grouped(X0[:, :64], W0[:, 1:65, :72], offs(sizes, 1), out=view)
    assert got is view and (out[:, :3] == 7).all() and (out[:, 75:] == 7).all() and (out[0] == 7).all()
    assert torch.equal(view[1:], t2sp_amd.gemm_grouped(X0[:, :64].contiguous(), W0[:, 1:65, :72].contiguous(), offs(sizes, 1))[1:])


@pytest.mark.parametrize("bits", [32, 64])
def test_rows_outside_every_group_are_left_and_never_read(bits):
    import torch
    sizes, K, N = [5, 0, 70, 2], 72, 88
    X, W, D = make((100, K), "bfloat16", 11), make((4, K, N), "bfloat16", 12), make((100, N), "bfloat16", 13)
    o = offs(sizes, 9, bits)
    want, dwant = t2sp_amd.gemm_grouped(X, W, o), t2sp_amd.gemm_grouped_wgrad(X, D, o)
    for t in (X, D):                                        # poison what belongs to no group
        t[:9] = float("nan")
        t[86:] = float("inf")
    Y = torch.full((100, N), 3.0, dtype=torch.bfloat16, device="cuda")
    t2sp_amd.gemm_grouped(X, W, o, out=Y)
    assert (Y[:9] == 3).all() and (Y[86:] == 3).all() and torch.equal(Y[9:86], want[9:86])
    assert torch.equal(t2sp_amd.gemm_grouped_wgrad(X, D, o), dwant)


def test_not_a_number_stays_in_its_group_row_and_reduction():
    """The k behind the end of a row, the rows behind a group and the columns behind a matrix hold NaN."""
    import torch
    sizes, K, N = [3, 140, 33], 72, 136
    X0, W0 = torch.full((176, 80), float("nan"), device="cuda"), torch.full((3, 80, 144), float("nan"), device="cuda")
    X0[:, :K], W0[:, :K, :N] = make((176, K), "float32", 14), make((3, K, N), "float32", 15)
    for name in TYPES:
        X, W = X0.to(dt(name), copy=True)[:, :K], W0.to(dt(name))[:, :K, :N]
        check_forward(X, W, sizes, 0)
        check_forward(W0.to(dt(name))[0, :K, :N].contiguous(), W0.to(dt(name))[:, :K, :N], [K, 0, 0], 1)
        X[3] = float("nan")                                 # first row of the second group
        Y = t2sp_amd.gemm_grouped(X, W, offs(sizes))
        assert torch.isnan(Y[3]).all() and torch.isfinite(torch.cat([Y[:3], Y[4:]]).float()).all()
        dW = t2sp_amd.gemm_grouped_wgrad(X, make((176, N), name, 16), offs(sizes))
        assert torch.isnan(dW[1]).all() and torch.isfinite(dW[0].float()).all() and torch.isfinite(dW[2].float()).all()


def test_wild_offsets_stay_inside_the_buffers():
    import torch
    X, W = make((64, 64), "bfloat16", 17), make((3, 64, 64), "bfloat16", 18)
    guard = torch.full((80, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    Y = guard[8:72]
    for o in ([-5, 10, 20, 1 << 30], [64, 64, 64, 64], [50, 20, 30, 64], [-(1 << 31), 0, 0, (1 << 31) - 1]):
        t2sp_amd.gemm_grouped(X, W, torch.tensor(o, dtype=torch.int32).cuda(), out=Y)
        t2sp_amd.gemm_grouped_wgrad(X, X, torch.tensor(o, dtype=torch.int32).cuda())
        torch.cuda.synchronize()
        assert (guard[:8] == 5).all() and (guard[72:] == 5).all()
    big = torch.tensor([0, 10, 20, 1 << 40]).cuda()
    assert torch.equal(t2sp_amd.gemm_grouped(X, W, big)[20:], t2sp_amd.gemm_grouped(X, W, offs([10, 10, 44]))[20:])


def test_many_groups_and_empty_runs():
    """More groups than the 64 one scan covers; runs of empty ones; one row each."""
    rng = np.random.default_rng(0)
    sizes = [int(s) for s in rng.integers(0, 4, 200)]
    sizes[10:90] = [0] * 80
    X, W = make((sum(sizes), 64), "float16", 19), make((200, 64, 72), "float16", 20)
    check_forward(X, W, sizes, 0)
    check_wgrad(X, make((sum(sizes), 72), "float16", 21), sizes)
    check_forward(make((64, 64), "float16", 22), make((64, 128, 64), "float16", 23), [1] * 64, 1)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_float_results_of_16_bit_operands(dtype):
    import torch
    X, W, D = make((150, 136), dtype, 24), make((2, 136, 264), dtype, 25), make((150, 264), dtype, 26)
    Y = check_forward(X, W, [100, 50], 0, out_dtype=torch.float32)
    assert Y.dtype == torch.float32
    check_wgrad(X, D, [100, 50], out_dtype=torch.float32)


def test_large_tiles_and_uneven_groups():
    """The largest tile in each direction, with groups that end inside one."""
    sizes = [1500, 37, 1024, 900, 0, 635]
    X, W, D = make((4096, 512), "bfloat16", 27), make((6, 512, 1032), "bfloat16", 28, 0.05), make((4096, 1032), "bfloat16", 29)
    check_forward(X, W, sizes, 0)
    check_forward(D, W, sizes, 1)
    check_wgrad(X, D, sizes)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes,K,N", [([4100], 128, 64), ([3000, 0, 1, 500], 96, 200), ([33, 2500], 65, 41), ([15, 1, 2000, 0, 900], 8, 9)])
def test_small_matrices_from_many_rows(dtype, sizes, K, N):
    """Sums over the rows in parts: empty groups, groups shorter than a part, rows off the vector grid, results in a strided view, which
    keeps what lies around it, float results of 16-bit operands, and the same bits every time."""
    import torch
    E, T = len(sizes), sum(sizes)
    X, D = make((T + 7, K), dtype, 50), make((T + 7, N), dtype, 51)
    check_wgrad(X, D, sizes, 3)
    check_wgrad(X, D, sizes, 3, out_dtype=torch.float32)
    whole = torch.full((E, K + 2, N + 3), 7.0, dtype=dt(dtype), device="cuda")
    check_wgrad(X, D, sizes, 3, out=whole[:, 1:K + 1, 2:N + 2])
    inside = torch.zeros_like(whole, dtype=torch.bool)
    inside[:, 1:K + 1, 2:N + 2] = True
    assert (whole[~inside] == 7.0).all()
    again = t2sp_amd.gemm_grouped_wgrad(X, D, offs(sizes, 3))
    assert torch.equal(again, whole[:, 1:K + 1, 2:N + 2])


def test_no_rows():
    import torch
    X, W = make((0, 64), "bfloat16", 30), make((2, 64, 64), "bfloat16", 31)
    o = offs([0, 0])
    assert t2sp_amd.gemm_grouped(X, W, o).shape == (0, 64)
    assert (t2sp_amd.gemm_grouped_wgrad(X, X, o) == 0).all()


def test_gradients_against_differences():
    """L = sum(S * Y): dX = S op(W)^T and dW = X^T S; directional differences of L in float64, from the forward product of
    float operands.  L is linear in X and in W, so a difference with any step h is exact but for rounding: each Y element is
    off by at most (K + 1) u sum |x w|, so the difference quotient by at most twice that, summed, over h."""
    import torch
    sizes, K, N = [20, 0, 45], 48, 40
    X, W, S = make((65, K), "float32", 32), make((3, K, N), "float32", 33), make((65, N), "float32", 34)
    o = offs(sizes)
    dX, dW = t2sp_amd.gemm_grouped(S, W, o, opb=1), t2sp_amd.gemm_grouped_wgrad(X, S, o)
    for which, grad in (("x", dX), ("w", dW)):
        V = make(tuple(grad.shape), "float32", 35)
        h = 1.0
        at = lambda s: (S.double() * t2sp_amd.gemm_grouped(X + s * V if which == "x" else X, W + s * V if which == "w" else W, o).double()).sum()
        diff = (at(h) - at(-h)) / (2 * h)
        mag = sum((S[a:b].double().abs() * ((X[a:b].double().abs() + (V[a:b].double().abs() if which == "x" else 0))
                                            @ (W[e].double().abs() + (V[e].double().abs() if which == "w" else 0)))).sum()
                  for e, (a, b) in enumerate(zip([0, 20, 20], [20, 20, 65])))
        # + one rounding of X + sV (relative u of each operand) on both sides, + the gradient's own sums
        bound = 2 * (K + 3) * 2.0 ** -24 * mag / (2 * h) * 2 + 70 * 2.0 ** -24 * mag
        assert abs(diff - (grad.double() * V.double()).sum()) <= bound


def test_on_a_side_stream_and_in_a_graph():
    import torch
    sizes, K, N = [60, 0, 200], 65, 72                       # (65: the operands pass through the workspace)
    X, W, D = make((260, K), "bfloat16", 36), make((3, K, N), "bfloat16", 37), make((260, N), "bfloat16", 38)
    o = offs(sizes)
    want = (t2sp_amd.gemm_grouped(X, W, o), t2sp_amd.gemm_grouped(D, W, o, opb=1), t2sp_amd.gemm_grouped_wgrad(X, D, o))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = (t2sp_amd.gemm_grouped(X, W, o), t2sp_amd.gemm_grouped(D, W, o, opb=1), t2sp_amd.gemm_grouped_wgrad(X, D, o))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = []
    for _ in range(2):                                       # two graphs of the same call: workspaces of their own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = (t2sp_amd.gemm_grouped(X, W, o), t2sp_amd.gemm_grouped(D, W, o, opb=1), t2sp_amd.gemm_grouped_wgrad(X, D, o))
        graphs.append((g, res))
    for _ in range(3):
        for g, res in graphs:
            for r in res:
                r.fill_(float("nan"))
            torch.cuda.synchronize()
            g.replay()
        torch.cuda.synchronize()
        for g, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(want, res))
    o.copy_(offs([100, 100, 60]))                            # the sizes are read at replay
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1][0], t2sp_amd.gemm_grouped(X, W, o))


def test_the_same_bits_every_time():
    import torch
    X, W, D = make((512, 264), "bfloat16", 39), make((4, 264, 136), "bfloat16", 40), make((512, 136), "bfloat16", 41)
    o = offs([100, 200, 12, 200])
    first = (t2sp_amd.gemm_grouped(X, W, o), t2sp_amd.gemm_grouped_wgrad(X, D, o))
    for _ in range(5):
        again = (t2sp_amd.gemm_grouped(X, W, o), t2sp_amd.gemm_grouped_wgrad(X, D, o))
        assert all(torch.equal(a, b) for a, b in zip(first, again))
