"""GPU tests of the products of a language model's layers together: a training step of an expert layer with its output loss, a
token served by 4-bit experts, the operator entries on host arrays, and calls from several streams and threads at once.

Bounds are carried along with the values: for a product Y = A B of n terms, with |dA| <= eA and |dB| <= eB elementwise,
|dY| <= eA (|B| + eB) + |A| eB + (n + 1) u (|A| + eA) (|B| + eB), u = 2^-24 (each test names the other roundings)."""
import threading

import numpy as np
import pytest

import t2sp_amd

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


class Bounded:
    """A float64 value and a bound on the error of the float32 value that stands for it."""

    def __init__(self, v, e=None):
        import torch
        self.v = v.double()
        self.e = torch.zeros_like(self.v) if e is None else e

    def mm(self, other):
        a, b = self.v.abs(), other.v.abs()
        n = self.v.shape[-1]
        e = self.e @ (b + other.e) + a @ other.e + (n + 1) * U * ((a + self.e) @ (b + other.e))
        return Bounded(self.v @ other.v, e)

    def t(self):
        return Bounded(self.v.t(), self.e.t())

    def rows(self, index):
        return Bounded(self.v[index], self.e[index])

    def times(self, f):                                        # by a factor that is exact, rounded once
        return Bounded(self.v * f, (self.e * f.abs()) * (1 + U) + U * (self.v * f).abs())

    def check(self, got):
        import torch
        err = (got.double() - self.v).abs()
        assert torch.isfinite(got.double()).all()
        assert (err <= self.e + 1e-300).all(), float((err / self.e.clamp(min=1e-300)).max())


def normal(shape, seed, std=1.0):
    import torch
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).cuda()


def by_group(f, bounds):
    """Concatenates f(e, slice) over groups."""
    import torch
    parts = [f(e, slice(bounds[e], bounds[e + 1])) for e in range(len(bounds) - 1)]
    return Bounded(torch.cat([p.v for p in parts]), torch.cat([p.e for p in parts]))


def test_a_training_step_of_an_expert_layer_and_its_loss():
    """Each token goes to two of five experts (one of them gets none): x -> W1[e] -> max(., 0) -> W2[e] -> weighted sum -> loss
    over a vocabulary; all gradients.  The kinks use the mask that the forward pass found."""
    import torch
    T, E, D, F, V = 150, 5, 40, 72, 333
    X, W1, W2, Wv = normal((T, D), 1), normal((E, D, F), 2, D ** -0.5), normal((E, F, D), 3, F ** -0.5), normal((V, D), 4, 0.3)
    gates = torch.softmax(normal((T, E), 5) + torch.tensor([0.0, 0, -1e9, 0.5, 0]).cuda(), 1)
    p, chosen = gates.topk(2, dim=1)
    labels = torch.from_numpy(np.random.default_rng(6).integers(0, V, T)).cuda()
    labels[::9] = -100
    order = torch.argsort(chosen.reshape(-1), stable=True)      # rows sorted by expert
    token = order // 2
    weight = p.reshape(-1)[order]
    sizes = torch.bincount(chosen.reshape(-1), minlength=E)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), sizes.cumsum(0)])
    bounds = offsets.tolist()
    assert 0 in sizes.tolist()

    rows = X[token]
    y1 = t2sp_amd.gemm_grouped(rows, W1, offsets)
    mask = (y1 > 0).float()
    a = y1 * mask
    y2 = t2sp_amd.gemm_grouped(a, W2, offsets)
    back = torch.argsort(order)                                 # row of (token, choice)
    pair = (y2 * weight[:, None])[back].reshape(T, 2, D)
    H = pair[:, 0] + pair[:, 1]
    loss, lse = t2sp_amd.xent(H, Wv, labels)
    valid = labels >= 0
    dloss = valid.float() / int(valid.sum())
    dH, dWv = t2sp_amd.xent_grad(H, Wv, labels, lse, dloss)
    dy2 = dH[token] * weight[:, None]
    dW2 = t2sp_amd.gemm_grouped_wgrad(a, dy2, offsets)
    dy1 = t2sp_amd.gemm_grouped(dy2, W2, offsets, opb=1) * mask
    dW1 = t2sp_amd.gemm_grouped_wgrad(rows, dy1, offsets)
    drows = t2sp_amd.gemm_grouped(dy1, W1, offsets, opb=1)

    # the same in float64 with bounds
    w = weight.double()[:, None]
    b_rows = Bounded(rows)
    b_y1 = by_group(lambda e, s: b_rows.rows(s).mm(Bounded(W1[e])), bounds)
    b_y1.check(y1)
    b_a = Bounded(b_y1.v * mask.double(), b_y1.e * mask.double())
    b_y2 = by_group(lambda e, s: b_a.rows(s).mm(Bounded(W2[e])), bounds)
    b_pair = b_y2.times(w).rows(back)
    v, e = b_pair.v.reshape(T, 2, D), b_pair.e.reshape(T, 2, D)
    hv = v[:, 0] + v[:, 1]
    b_H = Bounded(hv, (e[:, 0] + e[:, 1]) * (1 + U) + U * hv.abs())
    b_H.check(H)
    z = b_H.mm(Bounded(Wv).t())
    lse64 = torch.logsumexp(z.v, 1)
    span = z.v.max(1).values - z.v.min(1).values
    e_lse = z.e.max(1).values + 3 * (3 * span + 2) * U + V * U + 2 * U * (lse64.abs() + 1)
    at = (torch.arange(T, device="cuda"), labels.clamp(min=0))
    want = torch.where(valid, lse64 - z.v[at], torch.zeros_like(lse64))
    assert ((loss.double() - want).abs() <= e_lse + z.e[at] + U * (want.abs() + lse64.abs())).all()
    prob = torch.exp(z.v - lse64[:, None])
    hot = torch.zeros_like(prob)
    hot[at] = 1.0
    on = valid.double()[:, None]
    g = Bounded((prob - hot) * on, (prob * (z.e + e_lse[:, None] + (3 * (z.v - lse64[:, None]).abs() + 2) * U) * 1.01 + 2 * U * (prob + hot)) * on)
    b_dH = g.mm(Bounded(Wv))
    b_dH.e = b_dH.e + 4 * U * (g.v.abs() @ Wv.double().abs())   # (the parts of the reduction are joined)
    b_dH = b_dH.times(dloss.double()[:, None])
    b_dH.check(dH)
    top = float(dloss.max())
    b_dWv = g.t().mm(b_H.times(dloss.double()[:, None] / top))
    b_dWv.times(torch.tensor(top, dtype=torch.float64, device="cuda")).check(dWv)
    b_dy2 = b_dH.rows(token).times(w)
    for ex in range(E):
        s = slice(bounds[ex], bounds[ex + 1])
        b_a.rows(s).t().mm(b_dy2.rows(s)).check(dW2[ex])
    b_da = by_group(lambda ex, s: b_dy2.rows(s).mm(Bounded(W2[ex]).t()), bounds)
    b_dy1 = Bounded(b_da.v * mask.double(), b_da.e * mask.double())
    for ex in range(E):
        s = slice(bounds[ex], bounds[ex + 1])
        b_rows.rows(s).t().mm(b_dy1.rows(s)).check(dW1[ex])
    by_group(lambda ex, s: b_dy1.rows(s).mm(Bounded(W1[ex]).t()), bounds).check(drows)


def test_a_token_through_4_bit_experts_agrees_with_the_grouped_product():
    """The same experts once as 4-bit numbers, once as the float matrices they stand for (numbers, zero points and scales chosen
    such that (q - z) s is exact in float): gemv_w4 with ids and gemm_grouped agree within the sum of their bounds."""
    import torch
    E, N, K, group = 6, 50, 200, 32
    rng = np.random.default_rng(7)
    q = torch.from_numpy(rng.integers(0, 16, (E, N, K)).astype(np.uint8)).cuda()
    s = torch.from_numpy(rng.choice([0.25, 0.5, 0.125], (E, N, 7)).astype(np.float32)).cuda()
    z = torch.from_numpy(rng.integers(4, 12, (E, N, 7)).astype(np.float32)).cuda()
    of = torch.arange(K, device="cuda") // group
    W = (q.float() - z[:, :, of]) * s[:, :, of]
    x = normal((4, K), 8)
    ids = torch.tensor([0, 2, 2, 5], dtype=torch.int32).cuda()
    y4 = t2sp_amd.gemv_w4(x, t2sp_amd.pack_w4(q, s, z, group=group), ids=ids)
    offsets = torch.tensor([0, 1, 1, 3, 3, 3, 4], dtype=torch.int32).cuda()
    yg = t2sp_amd.gemm_grouped(x, W, offsets, opb=1)
    for m, e in enumerate(ids.tolist()):
        want = W[e].double() @ x[m].double()
        mag = W[e].double().abs() @ x[m].double().abs()
        wide = (s[e][:, of].double() * (16 + q[e].double() + 16 + z[e][:, of].double())) @ x[m].double().abs()
        assert ((yg[m].double() - want).abs() <= (K + 1) * U * mag).all()
        assert ((y4[m].double() - want).abs() <= (K + 8) * U * wide).all()


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_entries_on_host_arrays_give_the_device_results(dtype):
    import torch
    rng = np.random.default_rng(9)
    half = dtype == np.float16
    dev = lambda a: torch.from_numpy(a).cuda()
    X, W, dY = (rng.standard_normal(s).astype(dtype) for s in ((40, 24), (3, 24, 17), (40, 17)))
    off = np.array([2, 2, 30, 38], np.int64)
    Y = np.full((40, 17), 3.0, dtype)
    assert t2sp_amd.gemm_grouped(X, W, off, out=Y) is Y
    want = t2sp_amd.gemm_grouped(dev(X), dev(W), dev(off)).cpu().numpy()
    assert (Y[2:38] == want[2:38]).all() and (Y[:2] == 3).all() and (Y[38:] == 3).all()
    Wt = np.ascontiguousarray(W.transpose(0, 2, 1))
    assert (t2sp_amd.gemm_grouped(X, Wt, off, opb=1)[2:38] == t2sp_amd.gemm_grouped(dev(X), dev(Wt), dev(off), opb=1).cpu().numpy()[2:38]).all()
    assert (t2sp_amd.gemm_grouped_wgrad(X, dY, off) == t2sp_amd.gemm_grouped_wgrad(dev(X), dev(dY), dev(off)).cpu().numpy()).all()
    if half:                                                    # float results of half operands
        Yf = np.zeros((40, 17), np.float32)
        t2sp_amd.gemm_grouped(X, W, off, out=Yf)
        assert (Yf[2:38].astype(np.float16) == want[2:38]).all()
    H, Wv = rng.standard_normal((21, 24)).astype(dtype), (rng.standard_normal((50, 24)) * 0.3).astype(dtype)
    lab = rng.integers(-1, 50, 21).astype(np.int32)
    loss, lse = t2sp_amd.xent(H, Wv, lab)
    tl, te = t2sp_amd.xent(dev(H), dev(Wv), dev(lab))
    assert (loss == tl.cpu().numpy()).all() and (lse == te.cpu().numpy()).all()
    d = rng.standard_normal(21).astype(np.float32)
    for a, b in zip(t2sp_amd.xent_grad(H, Wv, lab, lse, d), t2sp_amd.xent_grad(dev(H), dev(Wv), dev(lab), te, dev(d))):
        assert (a == b.cpu().numpy()).all()
    q, s, z = rng.integers(0, 16, (3, 20, 70)).astype(np.uint8), rng.random((3, 20, 3)).astype(dtype), rng.random((3, 20, 3)).astype(dtype)
    x, ids = rng.standard_normal((4, 70)).astype(dtype), np.array([2, 0, 9, 1], np.int32)
    for args, kw in (((q, s, z), dict(ids=ids)), ((q[0], s[0]), {})):
        host = t2sp_amd.gemv_w4(x, t2sp_amd.pack_w4(*args, group=32), **kw)
        on_device = t2sp_amd.gemv_w4(dev(x), t2sp_amd.pack_w4(*map(dev, args), group=32), **{k: dev(v) for k, v in kw.items()})
        assert (host == on_device.cpu().numpy()).all()
    assert t2sp_amd.last_kernel_ns() > 0


def test_device_buffers_through_the_entries():
    """halide_buffer_t with device memory of bfloat16 elements (type code 4)."""
    import torch
    from t2sp_amd.buffer import HalideBuffer
    X, W = normal((30, 64), 10).bfloat16(), normal((2, 64, 40), 11).bfloat16()
    off = torch.tensor([0, 13, 30], dtype=torch.int32).cuda()
    Y = torch.zeros((30, 40), dtype=torch.bfloat16, device="cuda")
    b = [HalideBuffer.wrap(t) for t in (X, W, off, Y)]
    torch.cuda.synchronize()
    assert t2sp_amd.lib().gemm_grouped(0, *[x.ref for x in b]) == 0
    assert torch.equal(Y, t2sp_amd.gemm_grouped(X, W, off))


def test_streams_and_threads_at_once():
    """Calls of every operator in flight on several streams, from several threads, each against its own plain result."""
    import torch
    sets = []
    for i in range(4):
        X, W = normal((300 + 41 * i, 65), 20 + i).bfloat16(), normal((3, 65, 72), 30 + i).bfloat16()
        T = X.shape[0]
        off = torch.tensor([0, 100, 100 + i, T], dtype=torch.int32).cuda()
        H, Wv = normal((90 + i, 70), 40 + i).half(), normal((500 + i, 70), 50 + i, 0.2).half()
        lab = torch.from_numpy(np.random.default_rng(i).integers(-1, 500, 90 + i)).cuda()
        d = (lab >= 0).float()
        w4 = t2sp_amd.pack_w4(torch.from_numpy(np.random.default_rng(i).integers(0, 16, (100, 65)).astype(np.uint8)).cuda(),
                              normal((100, 3), 60 + i).bfloat16(), group=32)

        def run(X=X, W=W, off=off, H=H, Wv=Wv, lab=lab, d=d, w4=w4):
            loss, lse = t2sp_amd.xent(H, Wv, lab)
            return (t2sp_amd.gemm_grouped(X, W, off), t2sp_amd.gemm_grouped_wgrad(X, X, off), loss, *t2sp_amd.xent_grad(H, Wv, lab, lse, d),
                    t2sp_amd.gemv_w4(X[:20], w4))
        sets.append((run, run()))
    torch.cuda.synchronize()
    failed = []

    def work(run, want):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got = run()
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(want, got)):
                        failed.append("differs")
        except Exception as e:                                  # reported by the main thread
            failed.append(repr(e))
    threads = [threading.Thread(target=work, args=s) for s in sets]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


@pytest.mark.parametrize("cus,xcds", [(1, 1), (3, 8), (38, 1), (304, 8), (64, 4)])
def test_planned_for_other_machines(cus, xcds):
    """Launches planned for other numbers of CUs and dies (a partitioned device) cover every tile: values against float64."""
    import torch
    L = t2sp_amd.lib()
    X, W, dY = normal((1200, 136), 70), normal((5, 136, 520), 71), normal((1200, 520), 72)
    bounds = [0, 700, 700, 830, 831, 1190]
    off = torch.tensor(bounds, dtype=torch.int32).cuda()
    Hh, Wv = normal((300, 64), 73).bfloat16(), normal((1000, 64), 74, 0.2).bfloat16()
    lab = torch.arange(300).cuda()
    want = t2sp_amd.xent(Hh, Wv, lab)[0]
    L.t2sp_set_machine(cus, xcds)
    try:
        for half in (False, True):
            x, w, d = (t.bfloat16() if half else t for t in (X, W, dY))
            Y, dW = t2sp_amd.gemm_grouped(x, w, off, out_dtype=torch.float32), t2sp_amd.gemm_grouped_wgrad(x, d, off, out_dtype=torch.float32)
            by_group(lambda e, s: Bounded(x[s]).mm(Bounded(w[e])), bounds).check(Y[:1190])
            for e in range(5):
                s = slice(bounds[e], bounds[e + 1])
                Bounded(x[s]).t().mm(Bounded(d[s])).check(dW[e])
        loss, lse = t2sp_amd.xent(Hh, Wv, lab)
        assert torch.allclose(loss, want, rtol=0, atol=1e-5)     # (sums of 1000 terms near 1, in another order)
        dH, _ = t2sp_amd.xent_grad(Hh, Wv, lab, lse, torch.full((300,), 1 / 300, device="cuda"))
        assert torch.isfinite(dH.float()).all()
    finally:
        L.t2sp_set_machine(0, 0)


def test_driver_in_cpp_prints_success(tmp_path):
    """tests/drivers/gemm_grouped-run.cpp: the C++ interface with host buffers (built by `make -C tests/drivers`)."""
    import os
    import subprocess
    exe = os.path.join(os.path.dirname(os.path.abspath(__file__)), "drivers", "bin", "gemm_grouped-run")
    assert os.path.exists(exe), "build the drivers first: make -C tests/drivers"
    p = subprocess.run([exe], capture_output=True, text=True, timeout=100, cwd=str(tmp_path))
    print(p.stdout, p.stderr)
    assert p.returncode == 0 and p.stdout.strip().splitlines()[-1] == "Success"
