"""GPU tests of how exactly the gradients of the cross entropy are held: float results of 16-bit operands against float64.

Logits are exact here (operands are small multiples of 1/4 whose products and sums a float holds in any order), so that what is
left is the exponentials, the representation of p - [label] and the sums.  u = 2^-24, u_T = eps / 2 of the operands' type,
ee = (3 |z - lse| + 2) u the relative error of an exponential, el = 3 max ee + V u + 2u (|lse| + 1) that of lse (both as derived
in test_xent_gpu.py):
  g     p (el + ee) and two roundings in float (the difference, the token's weight): 2u |g|; then as the sum of n = 2
        numbers of the type, each of which rounds what those before it leave: u_T^n |g| (half: not below half
        of its smallest step 2^-24, on a scale of 2^15: 2^-40 of the largest weight's); one number alone: u_T |g|
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
        dg = dg + 2.0 ** -40 * l.abs()[:, None]
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
