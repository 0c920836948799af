"""GPU tests of the cross entropy over a vocabulary (xent, xent_grad) against float64.

Tolerances, u = 2^-24, u_T = eps / 2 of the operands' type (0 for float, whose results round once more by u):
  z     a sum of D products in any order: |dz| <= (D + 1) u sum |h w| =: ez
  exp   of x = z - m or z - lse, as 2^(x log2 e): the product rounds by u |x| log2 e, i.e. u |x| relative in the result (twice:
        constant and product), the difference by u |x|, the instruction by 2u: relative error ee = (3 |x| + 2) u
  lse   log of a sum of V such terms: |dlse| <= max ez + max ee + V u + 2u (|lse| + 1); a tile's terms are rescaled twice
        more by such an exponential: 3 max ee in all
  loss  |dlse| + ez at the label + u (|loss| + |lse|)
  g     p (ez + |dlse| + ee), then its rounding u_T |p - hot| (half: at least 2^-25 / 2^15, its scale being 2^15)
  dH    |dloss| (sum |dg w| + (V + 4) u sum |g w|) + 2u |dH|, then the result's rounding
  dW    sum |dg l h| + (u_T + 2u) sum |g l h| (l h rounded to the type, l = dloss / max) + (T + 4) u sum |g l h|, times
        max |dloss|, then the result's rounding (half: terms below its smallest step add 2^-25 each)."""
import numpy as np
import pytest

import t2sp_amd

pytestmark = pytest.mark.gpu
TYPES = ["float32", "float16", "bfloat16"]
U = 2.0 ** -24


def dt(name):
    import torch
    return getattr(torch, name)


def make(shape, dtype, seed, std=1.0):
    import torch
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dt(dtype)).cuda()


def labels_for(T, V, seed, ignored=0.2, bits=64):
    import torch
    rng = np.random.default_rng(seed)
    lab = rng.integers(0, V, T)
    lab[rng.random(T) < ignored] = -100
    return torch.tensor(lab, dtype=torch.int64 if bits == 64 else torch.int32).cuda()


def rounding(t):
    import torch
    return 0.0 if t == torch.float32 else torch.finfo(t).eps / 2


def tiny(t):
    import torch
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def check(H, W, labels, dloss, out_dtype=None, views=None):
    """Loss and gradients against float64, with the bounds above; `views` are the tensors passed to the calls instead."""
    import torch
    T, D = H.shape
    V = W.shape[0]
    h, w = H.double(), W.double()
    valid = (labels >= 0) & (labels < V)
    h = torch.where(valid[:, None], h, torch.zeros_like(h))
    lab = torch.where(valid, labels, torch.zeros_like(labels)).long()
    z = h @ w.t()
    ez = (D + 1) * U * (h.abs() @ w.abs().t())
    lse = torch.logsumexp(z, 1)
    span = (z.max(1).values - z.min(1).values)
    elz = ez.max(1).values + 3 * (3 * span + 2) * U + V * U + 2 * U * (lse.abs() + 1)
    rows = torch.arange(T, device="cuda")
    want = torch.where(valid, lse - z[rows, lab], torch.zeros_like(lse))
    a, b = views or (H, W)
    loss, got_lse = t2sp_amd.xent(a, b, labels)
    assert loss.dtype == torch.float32 and got_lse.shape == (T,)
    assert (loss[~valid] == 0).all()
    assert ((loss.double() - want).abs() <= elz + ez[rows, lab] + U * (want.abs() + lse.abs()))[valid].all()
    assert ((got_lse.double() - lse).abs() <= elz)[valid].all()

    dH, dW = t2sp_amd.xent_grad(a, b, labels, got_lse, dloss, out_dtype=out_dtype)
    ut = rounding(H.dtype)
    p = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(z)
    hot[rows, lab] = 1.0
    g = torch.where(valid[:, None], p - hot, torch.zeros_like(p))
    ee = (3 * (z - lse[:, None]).abs() + 2) * U
    dg = p * (ez + elz[:, None] + ee) * 1.01 + ut * 1.01 * (g.abs() + U) + (2.0 ** -40 if H.dtype == torch.float16 else 0) + U * g.abs()
    dg = torch.where(valid[:, None], dg, torch.zeros_like(dg))
    dl = torch.where(valid, dloss.double(), torch.zeros_like(dloss.double()))
    out = dH.dtype
    uo = rounding(out)

    def close(got, want, bound):
        bound = bound + 2 * U * want.abs() + uo * (want.abs() + bound) + tiny(out)
        err = (got.double() - want).abs()
        assert torch.isfinite(got.double()).all()
        assert (err <= bound).all(), float((err / bound.clamp(min=1e-300)).max())

    close(dH, dl[:, None] * (g @ w), dl.abs()[:, None] * (dg @ w.abs() + (V + 4) * U * (g.abs() @ w.abs())))
    assert (dH[~valid] == 0).all()
    top = float(dl.abs().max())
    l = dl / top if top else dl
    lh = l[:, None] * h
    step = 2.0 ** -25 if H.dtype == torch.float16 else 0.0
    close(dW, top * (g.t() @ lh), top * (dg.t() @ lh.abs() * (1 + ut) + (ut + 2 * U + (T + 4) * U) * (g.abs().t() @ lh.abs())
                                         + step * g.abs().sum(0)[:, None]))
    return loss, got_lse, dH, dW


def mean_of(labels, V):
    import torch
    valid = (labels >= 0) & (labels < V)
    return valid.float() / max(int(valid.sum()), 1)


SHAPES = [(1, 1, 8), (1, 300, 64), (2, 17, 40), (63, 130, 64), (65, 129, 72), (130, 1000, 128), (257, 513, 264), (300, 5003, 64), (700, 260, 136)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,D", SHAPES)
def test_loss_and_gradients(dtype, T, V, D):
    lab = labels_for(T, V, 1, 0.0 if T < 3 else 0.2)
    check(make((T, D), dtype, 2), make((V, D), dtype, 3, 2.0 * D ** -0.5), lab, mean_of(lab, V))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,D", [(3, 5, 1), (33, 129, 7), (66, 257, 101), (129, 300, 1022)])
def test_widths_off_the_vector_grid(dtype, T, V, D):
    lab = labels_for(T, V, 4, bits=32)
    check(make((T, D), dtype, 5), make((V, D), dtype, 6, D ** -0.5), lab, mean_of(lab, V))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,D", [(2100, 300, 64), (1500, 709, 65), (4000, 3, 8)])
def test_many_tokens_and_a_small_matrix(dtype, T, V, D):
    """The gradient of W as sums over parts of the tokens."""
    lab = labels_for(T, V, 40, 0.3)
    check(make((T, D), dtype, 41), make((V, D), dtype, 42, 2.0 * D ** -0.5), lab, mean_of(lab, V))
    if dtype != "float32":
        check(make((T, D), dtype, 41), make((V, D), dtype, 42, 2.0 * D ** -0.5), lab, mean_of(lab, V), out_dtype=dt("float32"))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strided_and_unaligned_views(dtype):
    import torch
    H0, W0 = make((70, 100), dtype, 7), make((333, 120), dtype, 8, 0.2)
    lab = labels_for(70, 333, 9)
    for dh, dw in ((0, 0), (1, 0), (0, 3), (8, 16)):
        H, W = H0[:, dh:dh + 64], W0[:, dw:dw + 64]
        check(H.contiguous(), W.contiguous(), lab, mean_of(lab, 333), views=(H, W))
    H, W = H0[:, :64].contiguous(), W0[:, :64].contiguous()
    _, lse = t2sp_amd.xent(H, W, lab)
    dH, dW = t2sp_amd.xent_grad(H, W, lab, lse, mean_of(lab, 333))
    oh, ow = (torch.full((n, 90), 7.0, dtype=dt(dtype), device="cuda") for n in (70, 333))
    t2sp_amd.xent_grad(H, W, lab, lse, mean_of(lab, 333), dH=oh[:, 3:67], dW=ow[:, 5:69])
    assert torch.equal(oh[:, 3:67], dH) and torch.equal(ow[:, 5:69], dW)
    assert (oh[:, :3] == 7).all() and (oh[:, 67:] == 7).all() and (ow[:, :5] == 7).all() and (ow[:, 69:] == 7).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_uneven_weights_of_the_tokens(dtype):
    import torch
    lab = labels_for(150, 400, 10)
    d = make((150,), "float32", 11)
    d[::7] = 0.0
    d[::5] *= 1e-3
    check(make((150, 96), dtype, 12), make((400, 96), dtype, 13, 0.2), lab, d)
    check(make((150, 96), dtype, 12), make((400, 96), dtype, 13, 0.2), lab, torch.zeros(150, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
def test_what_stands_in_rows_without_a_label_reaches_nothing(dtype):
    import torch
    T, V, D = 140, 270, 72
    H, W, lab = make((T, D), dtype, 14), make((V, D), dtype, 15, 0.2), labels_for(T, V, 16, 0.4)
    lab[3], lab[4], lab[5] = V, -1, 1 << 40
    d = mean_of(lab, V)
    want = check(H, W, lab, d)
    off = ~((lab >= 0) & (lab < V))
    H2, d2 = H.clone(), d.clone()
    H2[off] = float("nan")
    H2[3] = float("inf")
    d2[off] = float("nan")
    d2[4] = float("inf")
    loss, lse = t2sp_amd.xent(H2, W, lab)
    dH, dW = t2sp_amd.xent_grad(H2, W, lab, lse, d2)
    assert torch.equal(loss, want[0]) and torch.equal(dH, want[2]) and torch.equal(dW, want[3])
    none = torch.full((T,), -100, device="cuda")
    loss, lse = t2sp_amd.xent(H2, W, none)
    dH, dW = t2sp_amd.xent_grad(H2, W, none, lse, d2)
    assert (loss == 0).all() and (dH == 0).all() and (dW == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_large_and_small_logits(dtype):
    """Logits up to about +-60 (exponentials beyond float's range without the maximum), and all equal ones."""
    import torch
    lab = labels_for(90, 300, 17)
    check(make((90, 64), dtype, 18, 2.0), make((300, 64), dtype, 19, 1.0), lab, mean_of(lab, 300))
    H, W = make((90, 64), dtype, 20), torch.zeros((300, 64), dtype=dt(dtype), device="cuda")
    check(H, W, lab, mean_of(lab, 300))
    big = torch.zeros((4, 64), dtype=dt(dtype), device="cuda")
    big[:, 0] = 128.0
    Wb = torch.zeros((5, 64), dtype=dt(dtype), device="cuda")
    Wb[:, 0] = torch.tensor([100.0, -100.0, 99.0, 0.0, 100.0])
    loss, lse = t2sp_amd.xent(big, Wb, torch.tensor([0, 1, 2, 4]).cuda())
    ln2 = float(np.log(2.0))
    assert torch.allclose(lse, torch.full((4,), 12800.0 + ln2, device="cuda"), rtol=2 * U, atol=0)
    assert torch.allclose(loss, torch.tensor([ln2, 25600 + ln2, 128 + ln2, ln2], device="cuda"), rtol=4 * U, atol=12800 * 2 * U)


def test_not_a_number_stays_in_its_token():
    import torch
    H, W = make((40, 64), "bfloat16", 21), make((300, 64), "bfloat16", 22, 0.2)
    lab = labels_for(40, 300, 23, 0.0)
    H[7] = float("nan")
    loss, lse = t2sp_amd.xent(H, W, lab)
    assert torch.isnan(loss[7]) and torch.isfinite(torch.cat([loss[:7], loss[8:]])).all()
    dH, _ = t2sp_amd.xent_grad(H, W, lab, lse, mean_of(lab, 300))
    assert torch.isnan(dH[7]).all() and torch.isfinite(torch.cat([dH[:7], dH[8:]]).float()).all()


def test_several_pieces_of_the_vocabulary():
    """A vocabulary of more than one piece, the last one short and odd (17 000 tokens' pieces are 4096 words)."""
    import torch
    T, V, D = 17000, 9001, 64
    H, W = make((T, D), "bfloat16", 24), make((V, D), "bfloat16", 25, 0.25)
    lab = labels_for(T, V, 26, 0.05)
    check(H, W, lab, mean_of(lab, V))


def test_one_gradient_alone():
    import torch
    H, W, lab = make((50, 64), "float16", 27), make((300, 64), "float16", 28, 0.2), labels_for(50, 300, 29)
    d = mean_of(lab, 300)
    _, lse = t2sp_amd.xent(H, W, lab)
    both = t2sp_amd.xent_grad(H, W, lab, lse, d)
    a, none = t2sp_amd.xent_grad(H, W, lab, lse, d, wanted=(True, False))
    assert none is None and torch.equal(a, both[0])
    none, b = t2sp_amd.xent_grad(H, W, lab, lse, d, wanted=(False, True))
    assert none is None and torch.equal(b, both[1])
    fH, fW = t2sp_amd.xent_grad(H, W, lab, lse, d, out_dtype=torch.float32)
    assert fH.dtype == fW.dtype == torch.float32 and torch.equal(fH.half(), both[0]) and torch.equal(fW.half(), both[1])


def test_no_tokens():
    import torch
    H, W = make((0, 64), "bfloat16", 30), make((300, 64), "bfloat16", 31)
    lab = torch.zeros(0, dtype=torch.int64, device="cuda")
    loss, lse = t2sp_amd.xent(H, W, lab)
    assert loss.shape == lse.shape == (0,)
    dH, dW = t2sp_amd.xent_grad(H, W, lab, lse, lse)
    assert dH.shape == (0, 64) and (dW == 0).all()


def test_gradients_against_differences():
    """Central differences of sum(dloss * loss) from the operator's own float loss, along a random direction.  The loss has a
    third derivative of at most about s^3 along a direction that changes a token's logits by s; with steps h the truncation is
    h^2 / 6 * sum |dloss| (2 s)^3, the rounding of the losses 2 * 1e-6 * (1 + |loss|) * sum |dloss| / (2 h)."""
    import torch
    T, V, D = 40, 200, 48
    H, W, lab = make((T, D), "float32", 32), make((V, D), "float32", 33, 0.3), labels_for(T, V, 34)
    d = make((T,), "float32", 35)
    valid = lab >= 0
    _, lse = t2sp_amd.xent(H, W, lab)
    dH, dW = t2sp_amd.xent_grad(H, W, lab, lse, d)
    h = 2.0 ** -6
    for grad, which in ((dH, 0), (dW, 1)):
        Vv = make(tuple(grad.shape), "float32", 36, 0.05)
        at = lambda s: (d.double() * t2sp_amd.xent(H + s * Vv if which == 0 else H, W + s * Vv if which == 1 else W, lab)[0].double()).sum()
        diff = (at(h) - at(-h)) / (2 * h)
        s = ((Vv.double() @ W.double().t()) if which == 0 else (H.double() @ Vv.double().t())).abs().max(1).values
        loss = t2sp_amd.xent(H, W, lab)[0].double()
        dv = torch.where(valid, d.double().abs(), torch.zeros_like(loss))
        bound = h * h / 6 * (dv * (2 * s) ** 3).sum() + (dv * 2e-6 * (1 + loss.abs() + lse.double().abs())).sum() / h
        got = (grad.double() * Vv.double()).sum()
        assert abs(diff - got) <= bound + 1e-5 * abs(got), (float(diff), float(got), float(bound))


def test_on_a_side_stream_and_in_graphs():
    import torch
    T, V, D = 300, 1003, 70
    H, W, lab = make((T, D), "bfloat16", 37), make((V, D), "bfloat16", 38, 0.2), labels_for(T, V, 39)
    d = mean_of(lab, V)

    def step():
        loss, lse = t2sp_amd.xent(H, W, lab)
        return (loss, lse) + t2sp_amd.xent_grad(H, W, lab, lse, d)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
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


def test_the_same_bits_every_time():
    import torch
    H, W, lab = make((500, 128), "float16", 40), make((3000, 128), "float16", 41, 0.2), labels_for(500, 3000, 42)
    d = mean_of(lab, 3000)
    first = None
    for _ in range(4):
        loss, lse = t2sp_amd.xent(H, W, lab)
        res = (loss, lse) + t2sp_amd.xent_grad(H, W, lab, lse, d)
        first = first or res
        assert all(torch.equal(a, b) for a, b in zip(first, res))
