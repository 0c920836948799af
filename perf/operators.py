"""The products of a language model's layers, as cases to time: what each operator of this kind in t2sp_amd does, in
plain torch (own = False) and through the framework's entry points (own = True).

  grouped  rows sorted by the expert they were routed to, each expert's rows times that expert's matrix: forward ("fwd"),
           gradient of the rows ("dx") and gradient of the matrices ("dw")
  xent     cross entropy of a softmax over a vocabulary, from hidden states and the output matrix: the loss alone
           ("loss"), or the loss with the gradients of both ("step")
  w4       a few rows times a matrix of 4-bit numbers with a scale (and maybe a zero point) for each group of inputs;
           with `experts` > 0 each row picks its own matrix
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORED = -100


def listed():
    return [
        # a prompt batch through a layer of experts: 8192 tokens, two experts each, popular and unpopular ones
        dict(name="grouped_prompt_bf16", op="grouped", dir="fwd", dtype="bf16", T=16384, E=16, K=2048, N=4096, opb=0, skew=0.5),
        # the gradient of the matrices of that layer
        dict(name="grouped_dw_bf16", op="grouped", dir="dw", dtype="bf16", T=16384, E=16, K=2048, N=4096, opb=0, skew=0.5),
        # one new token that goes to eight of 64 experts: latency, and eight matrices to read
        dict(name="grouped_token_bf16", op="grouped", dir="fwd", dtype="bf16", T=8, E=64, K=2048, N=1024, opb=1, skew=0.0),
        # a decoding batch: a handful of rows for each expert, some experts without any
        dict(name="grouped_batch_bf16", op="grouped", dir="fwd", dtype="bf16", T=256, E=32, K=4096, N=2048, opb=0, skew=0.7),
        # the gradient of the rows, at sizes that no tile or vector divides
        dict(name="grouped_dx_odd_fp16", op="grouped", dir="dx", dtype="fp16", T=2999, E=5, K=1000, N=1365, opb=0, skew=0.3),
        # the framework's own type, at its smallest benchmark's extents
        dict(name="grouped_fp32", op="grouped", dir="fwd", dtype="fp32", T=2048, E=8, K=1024, N=1024, opb=0, skew=0.3),
        # a training step's last layer over a large vocabulary
        dict(name="xent_step_bf16", op="xent", dir="step", dtype="bf16", T=8192, D=4096, V=128000),
        # the loss of a held-out batch
        dict(name="xent_loss_bf16", op="xent", dir="loss", dtype="bf16", T=2048, D=2048, V=32000),
        # a short ragged batch, an odd vocabulary, a width off the vector grid
        dict(name="xent_step_odd_fp16", op="xent", dir="step", dtype="fp16", T=777, D=1022, V=50001),
        # one token through a square projection
        dict(name="w4_token_bf16", op="w4", dtype="bf16", M=1, N=4096, K=4096, group=128, zeros=False, experts=0),
        # sixteen sequences decoded together, through a wide projection with zero points
        dict(name="w4_batch_fp16", op="w4", dtype="fp16", M=16, N=16384, K=4096, group=64, zeros=True, experts=0),
        # one token through the eight experts it was routed to
        dict(name="w4_experts_bf16", op="w4", dtype="bf16", M=8, N=2048, K=4096, group=128, zeros=True, experts=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """An extent of a model's width: mostly a multiple of 64, sometimes of 8, sometimes any number."""
    n = _log(rng, lo, hi)
    step = rng.choice((64, 64, 64, 8, 1))
    return max(step, n // step * step)


def draw(rng):
    op = rng.choice(("grouped", "grouped", "xent", "w4"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "grouped":
        return dict(op=op, dir=rng.choice(("fwd", "fwd", "dx", "dw")), dtype=dtype, T=_log(rng, 1, 8192), E=_log(rng, 1, 64),
                    K=_width(rng, 64, 4096), N=_width(rng, 64, 4096), opb=rng.choice((0, 1)), skew=round(rng.uniform(0.0, 1.2), 2))
    if op == "xent":
        return dict(op=op, dir=rng.choice(("loss", "step")), dtype=dtype, T=_log(rng, 1, 4096), D=_width(rng, 64, 4096),
                    V=_log(rng, 500, 64000))
    return dict(op=op, dtype=dtype, M=_log(rng, 1, 64), N=_width(rng, 64, 16384), K=_width(rng, 64, 16384),
                group=rng.choice((32, 64, 128)), zeros=rng.choice((False, True)), experts=rng.choice((0, 0, 8)))


def _shares(case):
    """The probability that a row goes to each expert, the popular ones first."""
    p = np.arange(1, case["E"] + 1, dtype=np.float64) ** -case["skew"]
    return p / p.sum()


def _normal(gen, shape, std, dtype):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["op"] == "grouped":
        T, E, K, N = case["T"], case["E"], case["K"], case["N"]
        counts = rng.multinomial(T, rng.permutation(_shares(case)))
        bounds = np.concatenate([[0], np.cumsum(counts)])
        s["bounds"] = [int(b) for b in bounds]
        s["offsets"] = torch.tensor(bounds, dtype=torch.int32, device="cuda")
        if case["dir"] in ("fwd", "dw"):
            s["X"] = _normal(gen, (T, K), 1.0, dt)
        if case["dir"] in ("dx", "dw"):
            s["dY"] = _normal(gen, (T, N), 1.0, dt)
        if case["dir"] != "dw":           # W[e] is K x N, stored as it is or (opb) transposed
            s["W"] = _normal(gen, (E, N, K) if case["opb"] else (E, K, N), K ** -0.5, dt)
    elif case["op"] == "xent":
        T, D, V = case["T"], case["D"], case["V"]
        s["H"] = _normal(gen, (T, D), 1.0, dt)
        s["W"] = _normal(gen, (V, D), 2.0 * D ** -0.5, dt)
        labels = rng.integers(0, V, T)
        labels[rng.random(T) < 0.06] = IGNORED          # padding and prompt tokens that carry no loss
        s["labels"] = torch.tensor(labels, dtype=torch.int64, device="cuda")
        valid = labels != IGNORED
        s["dloss"] = torch.tensor(valid / max(int(valid.sum()), 1), dtype=torch.float32, device="cuda")   # of the mean
    else:
        M, N, K, G = case["M"], case["N"], case["K"], case["group"]
        E = case["experts"]
        lead = (E,) if E else ()
        s["x"] = _normal(gen, (M, K), 1.0, dt)
        s["q"] = torch.randint(0, 16, lead + (N, K), generator=gen, device="cuda", dtype=torch.uint8)   # the 4-bit numbers
        groups = -(-K // G)
        s["scales"] = ((0.5 + torch.rand(lead + (N, groups), generator=gen, device="cuda")) * (0.2 * K ** -0.5)).to(dt)
        s["zeros"] = (torch.rand(lead + (N, groups), generator=gen, device="cuda") * 6 + 5).to(dt) if case["zeros"] else None
        s["picked"] = [int(i) for i in rng.permutation(max(E, M))[:M] % E] if E else None
        s["ids"] = torch.tensor(s["picked"], dtype=torch.int32, device="cuda") if E else None
        if own:                                         # the weights in the layout that the kernel reads, made once
            import t2sp_amd
            s["w4"] = t2sp_amd.pack_w4(s["q"], s["scales"], s["zeros"], group=G)
    return s


# ---------------------------------------------------------------------------------------------- the plain forms
def _plain_grouped(s):
    case, b = s["case"], s["bounds"]
    dt = DTYPES[case["dtype"]]
    T, E, K, N = case["T"], case["E"], case["K"], case["N"]
    if case["dir"] == "dw":
        dW = torch.zeros((E, K, N), dtype=dt, device="cuda")
        for e in range(E):
            if b[e + 1] > b[e]:
                dW[e] = (s["X"][b[e]:b[e + 1]].float().t() @ s["dY"][b[e]:b[e + 1]].float()).to(dt)
        return dW
    src = s["X"] if case["dir"] == "fwd" else s["dY"]
    out = torch.empty((T, N if case["dir"] == "fwd" else K), dtype=dt, device="cuda")
    for e in range(E):
        if b[e + 1] > b[e]:
            W = s["W"][e].float()
            if bool(case["opb"]) == (case["dir"] == "fwd"):
                W = W.t()
            out[b[e]:b[e + 1]] = (src[b[e]:b[e + 1]].float() @ W).to(dt)
    return out


def _plain_xent(s):
    H, W, labels = s["H"].float(), s["W"].float(), s["labels"]
    valid = labels != IGNORED
    target = torch.where(valid, labels, torch.zeros_like(labels))
    z = H @ W.t()
    top = z.max(dim=1).values
    e = torch.exp(z - top[:, None])
    total = e.sum(dim=1)
    rows = torch.arange(H.shape[0], device=H.device)
    loss = torch.where(valid, torch.log(total) + top - z[rows, target], torch.zeros_like(top))
    if s["case"]["dir"] == "loss":
        return loss
    g = e / total[:, None]
    g[rows, target] -= 1.0
    g = g * torch.where(valid, s["dloss"], torch.zeros_like(top))[:, None]
    dt = s["H"].dtype
    return loss, (g @ W).to(dt), (g.t() @ H).to(dt)


def _plain_w4(s):
    case = s["case"]
    K, G = case["K"], case["group"]
    x = s["x"].float()

    def matrix(q, scales, zeros):
        of = torch.arange(K, device="cuda") // G
        z = zeros.float()[:, of] if zeros is not None else 8.0
        return (q.float() - z) * scales.float()[:, of]

    if not case["experts"]:
        return (x @ matrix(s["q"], s["scales"], s["zeros"]).t()).to(s["x"].dtype)
    y = torch.empty((case["M"], case["N"]), dtype=s["x"].dtype, device="cuda")
    for r, e in enumerate(s["picked"]):
        z = s["zeros"][e] if s["zeros"] is not None else None
        y[r] = (matrix(s["q"][e], s["scales"][e], z) @ x[r]).to(y.dtype)
    return y


# ---------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    import t2sp_amd
    case = s["case"]
    if case["op"] == "grouped":
        if case["dir"] == "dw":
            return t2sp_amd.gemm_grouped_wgrad(s["X"], s["dY"], s["offsets"])
        if case["dir"] == "fwd":
            return t2sp_amd.gemm_grouped(s["X"], s["W"], s["offsets"], opb=case["opb"])
        return t2sp_amd.gemm_grouped(s["dY"], s["W"], s["offsets"], opb=1 - case["opb"])
    if case["op"] == "xent":
        loss, lse = t2sp_amd.xent(s["H"], s["W"], s["labels"])
        if case["dir"] == "loss":
            return loss
        dH, dW = t2sp_amd.xent_grad(s["H"], s["W"], s["labels"], lse, s["dloss"])
        return loss, dH, dW
    return t2sp_amd.gemv_w4(s["x"], s["w4"], ids=s["ids"])


def run(state):
    if own:
        return _own(state)
    return {"grouped": _plain_grouped, "xent": _plain_xent, "w4": _plain_w4}[state["case"]["op"]](state)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "grouped":
        T, E, K, N = case["T"], case["E"], case["K"], case["N"]
        active = float(np.sum(1.0 - (1.0 - _shares(case)) ** T))        # experts with at least one row, on average
        matrices = E if case["dir"] == "dw" else active                 # (a gradient of zeros is written too)
        return dict(bytes=size * (T * K + T * N + matrices * K * N) + 4 * (E + 1), flops=2.0 * T * K * N)
    if case["op"] == "xent":
        T, D, V = case["T"], case["D"], case["V"]
        if case["dir"] == "loss":
            return dict(bytes=size * (T * D + V * D) + 12 * T, flops=2.0 * T * D * V)
        return dict(bytes=2 * size * (T * D + V * D) + 16 * T, flops=6.0 * T * D * V)
    M, N, K = case["M"], case["N"], case["K"]
    matrices = min(case["experts"], M) if case["experts"] else 1
    groups = -(-K // case["group"])
    side = N * groups * size * (2 if case["zeros"] else 1)
    return dict(bytes=matrices * (N * K / 2.0 + side) + size * (M * K + M * N), flops=2.0 * M * N * K)


# ---------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "grouped":
        offs = s["offsets"].cpu().numpy()
        pieces = []
        for e, (lo, hi) in enumerate(zip(offs[:-1], offs[1:])):
            lo, hi = int(lo), int(hi)
            if case["dir"] == "dw":
                pieces.append(torch.mm(s["X"][lo:hi].double().transpose(0, 1), s["dY"][lo:hi].double()))
                continue
            if hi == lo:
                continue
            K_by_N = s["W"][e].double().transpose(0, 1) if case["opb"] else s["W"][e].double()
            pieces.append(torch.mm(s["X"][lo:hi].double(), K_by_N) if case["dir"] == "fwd"
                          else torch.mm(s["dY"][lo:hi].double(), K_by_N.transpose(0, 1)))
        return torch.stack(pieces) if case["dir"] == "dw" else torch.cat(pieces)
    if case["op"] == "xent":
        T, step = case["T"], 1024
        W = s["W"].double()
        losses, dHs, dW = [], [], None
        for lo in range(0, T, step):
            h, lab = s["H"][lo:lo + step].double(), s["labels"][lo:lo + step]
            keep = (lab >= 0).double()
            hot = torch.zeros((h.shape[0], case["V"]), dtype=torch.float64, device="cuda")
            hot.scatter_(1, lab.clamp(min=0)[:, None], 1.0)
            z = torch.mm(h, W.transpose(0, 1))
            lse = torch.logsumexp(z, dim=1)
            losses.append(keep * (lse - (z * hot).sum(dim=1)))
            if case["dir"] == "step":
                d = (torch.exp(z - lse[:, None]) - hot) * (keep * s["dloss"][lo:lo + step].double())[:, None]
                dHs.append(torch.mm(d, W))
                part = torch.mm(d.transpose(0, 1), h)
                dW = part if dW is None else dW.add_(part)
        loss = torch.cat(losses)
        return loss if case["dir"] == "loss" else (loss, torch.cat(dHs), dW)
    M, N, K, G = case["M"], case["N"], case["K"], case["group"]
    y = torch.zeros((M, N), dtype=torch.float64, device="cuda")
    for g in range(-(-K // G)):
        lo, hi = g * G, min(K, g * G + G)
        x = s["x"][:, lo:hi].double()
        for r in range(M) if case["experts"] else (slice(None),):
            at = (s["ids"][r].item(),) if case["experts"] else ()
            q = s["q"][at + (slice(None), slice(lo, hi))].double()
            z = s["zeros"][at + (slice(None), g)].double() if case["zeros"] else torch.full((N,), 8.0, dtype=torch.float64, device="cuda")
            term = torch.mm(x[r:r + 1] if case["experts"] else x, (q - z[:, None]).transpose(0, 1))
            y[r] += (term * s["scales"][at + (slice(None), g)].double())[0 if case["experts"] else slice(None)]
    return y
