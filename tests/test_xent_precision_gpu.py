"""GPU tests of how exactly the gradients of the cross entropy are held: float results of 16-bit operands against float64.

Logits are exact here (operands are small multiples of 1/4 whose products and sums a float holds in any order), so that what is
left is the exponentials, the representation of p - [label] and the sums.  u = 2^-24, u_T = eps / 2 of the operands' type,
ee = (3 |z - lse| + 2) u the relative error of an exponential, el = 3 max ee + V u + 2u (|lse| + 1) that of lse (both as derived
in test_xent_gpu.py):
  g     p (el + ee) and two roundings in float (the difference, the token's weight): 2u |g|; then as the sum of n = 2
        numbers of the type, each of which rounds what those before it leave: u_T^n |g| (half: not below half
        of its smallest step, 2^-25, on a scale of m 2^15 with |dloss| = m 2^x, m >= 1/2: 2^-39 |dloss|); one number alone: u_T |g|
  dH    sum |dg w| + (n V + 8) u sum |g w| (1 + u_T),   dW  sum |dg h| + (n T + 8) u sum |g h| (1 + u_T)   (n numbers: n times
        the terms)"""
import numpy as np
import pytest

import t2sp_amd
from test_xent_gpu import dt, labels_for, mean_of, rounding, U

pytestmark = pytest.mark.gpu


def quarters(shape, dtype, seed, most):
    import torch
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(-most, most + 1, shape, generator=g).float() / 4).to(dt(dtype)).cuda()


def bounds(H, W, labels, dloss, rounded=False):
    """dH, dW in float64 and how far float results may be off."""
    import torch
    T, V = H.shape[0], W.shape[0]
    valid = (labels >= 0) & (labels < V)
    h, w = H.double(), W.double()
    lab = torch.where(valid, labels, torch.zeros_like(labels)).long()
    z = h @ w.t()
    lse = torch.logsumexp(z, 1)
    p = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(z)
    hot[torch.arange(T, device="cuda"), lab] = 1.0
    l = torch.where(valid, dloss.double(), torch.zeros_like(lse))
    g = (p - hot) * l[:, None]
    ee = (3 * (z - lse[:, None]).abs() + 2) * U
    el = 3 * ee.max(1).values + V * U + 2 * U * (lse.abs() + 1)
    ut = rounding(H.dtype)
    numbers = 1 if rounded or H.dtype == torch.float32 else 2
    dg = p * l.abs()[:, None] * (el[:, None] + ee) * 1.01 + (2 * U + ut ** numbers) * 1.01 * g.abs()
    if H.dtype == torch.float16:
        dg = dg + 2.0 ** -39 * l.abs()[:, None]
    dH, dW = g @ w, g.t() @ h
    bH = dg @ w.abs() + (numbers * V + 8) * U * (1 + ut) * (g.abs() @ w.abs()) + 2 * U * dH.abs()
    bW = dg.t() @ h.abs() + (numbers * T + 8) * U * (1 + ut) * (g.abs().t() @ h.abs()) + 2 * U * dW.abs()
    return dH, dW, bH, bW


def within(got, want, bound):
    import torch
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs()
    assert (err <= bound + 1e-45).all(), float((err / (bound + 1e-45)).max())


SHAPES = [(5, 60, 8), (70, 50, 64), (130, 70, 40), (300, 150, 264)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("T,V,D", SHAPES)
def test_gradients_hold_more_than_the_operands_bits(dtype, T, V, D):
    import torch
    H, W, lab = quarters((T, D), dtype, 1, 4), quarters((V, D), dtype, 2, max(1, 64 // D)), labels_for(T, V, 3)
    d = mean_of(lab, V)
    _, lse = t2sp_amd.xent(H, W, lab)
    dH, dW = t2sp_amd.xent_grad(H, W, lab, lse, d, out_dtype=torch.float32)
    wH, wW, bH, bW = bounds(H, W, lab, d)
    within(dH, wH, bH)
    within(dW, wW, bW)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("T,V,D", SHAPES)
def test_rounded_on_request(dtype, T, V, D):
    import torch
    H, W, lab = quarters((T, D), dtype, 1, 4), quarters((V, D), dtype, 2, max(1, 64 // D)), labels_for(T, V, 3)
    d = mean_of(lab, V)
    _, lse = t2sp_amd.xent(H, W, lab)
    dH, dW = t2sp_amd.xent_grad(H, W, lab, lse, d, out_dtype=torch.float32, rounded=True)
    wH, wW, bH, bW = bounds(H, W, lab, d, True)
    within(dH, wH, bH)
    within(dW, wW, bW)
    full = t2sp_amd.xent_grad(H, W, lab, lse, d, out_dtype=torch.float32)
    assert (torch.equal(dH, full[0]) and torch.equal(dW, full[1])) == (dtype == "float32")
    alone, none = t2sp_amd.xent_grad(H, W, lab, lse, d, out_dtype=torch.float32, wanted=(True, False), rounded=True)
    assert none is None and torch.equal(alone, dH)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("ratio", [1e-3, 1e-5, 1e-6, 1e-7, 5e-9])
@pytest.mark.parametrize("T", [40, 2100])
def test_a_heavy_token_that_contributes_nothing(dtype, ratio, T):
    """One well-predicted token of weight 1, the others lighter: all of dW is theirs.  Rows of H differ in size too (by powers of
    two, so that logits stay exact).  half: p - [label] of light tokens is stored times m 2^b with b down to 5 and |dloss| =
    m 2^x, 1/2 <= m < 1: half of the smallest step, 2^-25, is 2^-25 / (m 2^5) <= 2^-29 of the weight."""
    import torch
    V, D = 60, 64
    H, W, lab = quarters((T, D), dtype, 1, 4), quarters((V, D), dtype, 2, 1), labels_for(T, V, 3)
    H[1::3] *= 0.25
    lab[0] = 7
    W[:, 0] = 0.0
    W[7, 0] = 8.0
    H[0] = 0.0
    H[0, 0] = 4.0                                            # its label's logit is 32, the others' 0
    d = ratio * (0.5 + torch.rand(T, generator=torch.Generator().manual_seed(4))).cuda()
    d[0] = 1.0
    d[5] = 0.0
    _, lse = t2sp_amd.xent(H, W, lab)
    dH, dW = t2sp_amd.xent_grad(H, W, lab, lse, d, out_dtype=torch.float32)
    wH, wW, bH, bW = bounds(H, W, lab, d)
    valid = (lab >= 0) & (lab < V)
    l = torch.where(valid, d.double().abs(), torch.zeros_like(d.double()))[:, None]
    step = 2.0 ** -29 if dtype == "float16" else 0.0
    within(dH, wH, bH + step * l * W.double().abs().sum(0))
    within(dW, wW, bW + step * (l * H.double().abs()).sum(0))
    assert float((dW.double() - wW).norm() / wW.norm()) < 2e-5
    only, none = t2sp_amd.xent_grad(H, W, lab, lse, d, out_dtype=torch.float32, wanted=(True, False))
    assert none is None and torch.equal(only, dH)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -20, 2.0 ** 60])
def test_weights_of_any_size(dtype, scale):
    """A power of two in all weights multiplies float gradients by it exactly."""
    import torch
    H, W, lab = quarters((70, 64), dtype, 1, 4), quarters((50, 64), dtype, 2, 1), labels_for(70, 50, 3)
    d = torch.randn(70, generator=torch.Generator().manual_seed(5)).cuda()
    _, lse = t2sp_amd.xent(H, W, lab)
    a = t2sp_amd.xent_grad(H, W, lab, lse, d, out_dtype=torch.float32)
    b = t2sp_amd.xent_grad(H, W, lab, lse, d * scale, out_dtype=torch.float32)
    assert torch.equal(a[0] * scale, b[0]) and torch.equal(a[1] * scale, b[1])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_a_weight_that_is_not_finite_stays_in_its_token(dtype):
    import torch
    H, W, lab = quarters((40, 64), dtype, 1, 4), quarters((50, 64), dtype, 2, 1), labels_for(40, 50, 3, 0.0)
    d = mean_of(lab, 50)
    _, lse = t2sp_amd.xent(H, W, lab)
    want, _ = t2sp_amd.xent_grad(H, W, lab, lse, d, out_dtype=torch.float32)
    for bad in (float("nan"), float("inf")):
        d2 = d.clone()
        d2[9] = bad
        dH, dW = t2sp_amd.xent_grad(H, W, lab, lse, d2, out_dtype=torch.float32)
        assert not torch.isfinite(dH[9]).any() and not torch.isfinite(dW).any()
        assert torch.equal(torch.cat([dH[:9], dH[10:]]), torch.cat([want[:9], want[10:]]))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("V", [5, 300, 5000])
def test_infinite_logits(dtype, V):
    """lse of a token with a logit at +inf is +inf (log sum exp), and so is its loss unless that logit is the label's; all logits at
    -inf give -inf; other tokens are what they were."""
    import torch
    T, D = 70, 64
    inf = float("inf")
    H, W, lab = quarters((T, D), dtype, 1, 4), quarters((V, D), dtype, 2, 1), labels_for(T, V, 3, 0.0)
    H[:, 0] = 0.0
    W[:, 0] = -1.0
    W[V - 1, 0] = 1.0
    W[0, 0] = 1.0
    loss0, lse0 = t2sp_amd.xent(H, W, lab)
    H[3], H[9] = 0.0, 0.0
    H[3, 0], H[9, 0] = inf, -inf                             # +inf at the words 0 and V - 1, -inf at the others; the reverse
    H[11, 5] = float("nan")
    H[13, 0] = inf                                           # with finite terms beside it
    lab[3], lab[9] = 1, 0
    loss, lse = t2sp_amd.xent(H, W, lab)
    for t in (3, 9, 13):
        assert lse[t] == inf
    assert loss[3] == inf and loss[9] == inf and torch.isnan(lse[11]) and torch.isnan(loss[11])
    loss2, lse2 = t2sp_amd.xent(H, W, torch.full((T,), V - 1, device="cuda"))
    assert lse2[3] == inf and torch.isnan(loss2[3])
    rest = torch.ones(T, dtype=torch.bool, device="cuda")
    rest[[3, 9, 11, 13]] = False
    assert torch.equal(loss[rest], loss0[rest]) and torch.equal(lse[rest], lse0[rest])
    W[:, 0] = -1.0
    lse3 = t2sp_amd.xent(H, W, lab)[1]
    assert lse3[3] == -inf and lse3[9] == inf and torch.equal(lse3[rest], lse0[rest])


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("rounded", [False, True])
def test_replayed_graphs_of_both_forms(dtype, rounded):
    """Weights and hidden states that change between replays; two graphs and eager calls in turn."""
    import torch
    T, V, D = 130, 500, 72
    H, W, lab = quarters((T, D), dtype, 1, 4), quarters((V, D), dtype, 2, 1), labels_for(T, V, 3)
    d = mean_of(lab, V)

    def step():
        loss, lse = t2sp_amd.xent(H, W, lab)
        return (loss, lse) + t2sp_amd.xent_grad(H, W, lab, lse, d, rounded=rounded)
    step()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, res))
    gen = torch.Generator().manual_seed(6)
    for turn in range(4):
        d.copy_(torch.randn(T, generator=gen) * 10.0 ** (-2 * turn))
        H.copy_((torch.randint(-4, 5, (T, D), generator=gen).float() / 4).to(dt(dtype)))
        want = step()
        for g, res in graphs:
            for r in res:
                r.fill_(float("nan"))
            g.replay()
        torch.cuda.synchronize()
        for g, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(want, res))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rounded", [False, True])
def test_equal_weights_change_no_bit(dtype, rounded):
    """The gradients for weights of 1 / 7 are those for weights of 1, multiplied by float(1 / 7)."""
    import torch
    H, W, lab = quarters((70, 64), dtype, 1, 4), quarters((50, 64), dtype, 2, 1), labels_for(70, 50, 3)
    _, lse = t2sp_amd.xent(H, W, lab)
    one = torch.ones(70, device="cuda")
    a = t2sp_amd.xent_grad(H, W, lab, lse, one, out_dtype=torch.float32, rounded=rounded)
    b = t2sp_amd.xent_grad(H, W, lab, lse, one / 7, out_dtype=torch.float32, rounded=rounded)
    assert torch.equal(a[0] * (one[0] / 7), b[0]) and torch.equal(a[1] * (one[0] / 7), b[1])
