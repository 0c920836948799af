"""GPU tests of the products with 4-bit weights (pack_w4, gemv_w4) against float64.

Tolerance.  The kernel sums x (16 + q) and x over the inputs of a group (products exact in float; float rows of x enter as
three bfloat16 pieces whose sum is x up to 2^-24 |x|), takes (16 + z) times the second from the first, and adds s times that.
With u = 2^-24 and n = K terms: |dy| <= sum over groups |s| * ((K + 8) u * (sum |x| (16 + q) + (16 + z) sum |x|)), and half a
step of the result's type.  That covers partial sums by several waves: any order of the K terms and ceil(K / 32) groups."""
import numpy as np
import pytest

import t2sp_amd

pytestmark = pytest.mark.gpu
TYPES = ["float32", "float16", "bfloat16"]


def dt(name):
    import torch
    return getattr(torch, name)


def weights(shape, group, dtype, zeros, seed):
    import torch
    g = torch.Generator().manual_seed(seed)
    K = shape[-1]
    q = torch.randint(0, 16, shape, generator=g, dtype=torch.uint8).cuda()
    side = tuple(shape[:-1]) + (-(-K // group),)
    s = ((torch.rand(side, generator=g) - 0.3) * 0.1).to(dt(dtype)).cuda()
    z = (torch.rand(side, generator=g) * 15).to(dt(dtype)).cuda() if zeros else None
    return q, s, z


def rows(M, K, dtype, seed):
    import torch
    return torch.randn((M, K), generator=torch.Generator().manual_seed(seed)).to(dt(dtype)).cuda()


def close(y, x, q, s, z, group):
    import torch
    K = q.shape[1]
    of = torch.arange(K, device="cuda") // group
    zz = z.double()[:, of] if z is not None else torch.full(q.shape, 8.0, dtype=torch.float64, device="cuda")
    ss, qq, xx = s.double()[:, of], q.double() % 16, x.double()
    want = xx @ ((qq - zz) * ss).t()
    bound = (K + 8) * 2.0 ** -24 * (xx.abs() @ (ss.abs() * (16 + qq + 16 + zz)).t())
    t = y.dtype
    if t != torch.float32:
        bound = bound + torch.finfo(t).eps / 2 * (want.abs() + bound) + torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
    err = (y.double() - want).abs()
    assert torch.isfinite(y.double()).all()
    assert (err <= bound).all(), float((err / bound.clamp(min=1e-300)).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,N,K,group", [(1, 16, 128, 128), (1, 1, 1, 32), (2, 5, 33, 32), (3, 100, 257, 64), (16, 33, 1000, 32), (17, 64, 512, 128),
                                         (31, 40, 96, 256), (33, 130, 2050, 64), (64, 48, 384, 32), (65, 16, 4096, 128), (200, 20, 160, 32),
                                         (1, 512, 5000, 8192)])
def test_product(dtype, zeros, M, N, K, group):
    q, s, z = weights((N, K), group, dtype, zeros, 1)
    x = rows(M, K, dtype, 2)
    w = t2sp_amd.pack_w4(q, s, z, group=group)
    close(t2sp_amd.gemv_w4(x, w), x, q, s, z, group)


@pytest.mark.parametrize("dtype", TYPES)
def test_every_number_at_every_place(dtype):
    """Integers that every type holds: the product is exact, so each number's place in the layout shows."""
    import torch
    N, K, group = 48, 300, 32
    q = (torch.arange(N * K).reshape(N, K) * 7 % 16).to(torch.uint8).cuda()
    s = torch.ones((N, 10), dtype=dt(dtype), device="cuda")
    w = t2sp_amd.pack_w4(q, s, torch.zeros_like(s), group=group)
    for k0 in range(0, K, 60):
        x = torch.zeros((60, K), dtype=dt(dtype), device="cuda")
        x[torch.arange(60), torch.arange(k0, k0 + 60)] = 1.0
        assert torch.equal(t2sp_amd.gemv_w4(x, w), q[:, k0:k0 + 60].t().to(dt(dtype)))


@pytest.mark.parametrize("dtype", TYPES)
def test_upper_bits_and_strided_arguments(dtype):
    import torch
    q0, s0, z0 = weights((70, 500), 64, dtype, True, 3)
    q0 |= 0xA0                                               # (only the low four bits are numbers)
    q, s, z = q0[1:60, 3:453], s0[1:60, :], z0[1:60, :]
    big = rows(9, 480, dtype, 4)
    w = t2sp_amd.pack_w4(q, s, z, group=64) if s.shape[1] == -(-450 // 64) else t2sp_amd.pack_w4(q, s[:, :8], z[:, :8], group=64)
    for d in (0, 1, 8):
        x = big[:, d:d + 450]
        out = torch.full((9, 80), 7.0, dtype=dt(dtype), device="cuda")
        t2sp_amd.gemv_w4(x, w, out=out[:, 5:64])
        close(out[:, 5:64], x, q, s[:, :8], z[:, :8], 64)
        assert (out[:, :5] == 7).all() and (out[:, 64:] == 7).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("zeros", [False, True])
def test_a_matrix_for_each_row(dtype, zeros):
    import torch
    E, N, K, group = 5, 40, 300, 32
    q, s, z = weights((E, N, K), group, dtype, zeros, 5)
    x = rows(9, K, dtype, 6)
    w = t2sp_amd.pack_w4(q, s, z, group=group)
    ids = torch.tensor([4, 0, 0, 2, -1, 3, 5, 1, 4], dtype=torch.int32).cuda()
    y = t2sp_amd.gemv_w4(x, w, ids=ids)
    for m, e in enumerate(ids.tolist()):
        if 0 <= e < E:
            close(y[m:m + 1], x[m:m + 1], q[e], s[e], z[e] if zeros else None, group)
        else:
            assert (y[m] == 0).all()


def test_what_lies_behind_a_row_reaches_nothing():
    import torch
    q, s, z = weights((20, 130), 64, "bfloat16", False, 7)
    big = torch.full((4, 256), float("nan"), dtype=torch.bfloat16, device="cuda")
    big[:, :130] = rows(4, 130, "bfloat16", 8)
    w = t2sp_amd.pack_w4(q, s, group=64)
    close(t2sp_amd.gemv_w4(big[:, :130], w), big[:, :130], q, s, None, 64)
    big[2, 5] = float("inf")
    y = t2sp_amd.gemv_w4(big[:, :130], w)
    assert torch.isfinite(y[[0, 1, 3]].float()).all() and not torch.isfinite(y[2].float()).any()


def test_no_rows():
    import torch
    q, s, _ = weights((20, 64), 64, "float16", False, 9)
    assert t2sp_amd.gemv_w4(torch.empty((0, 64), dtype=torch.float16, device="cuda"), t2sp_amd.pack_w4(q, s, group=64)).shape == (0, 20)


def test_float_rows_of_any_size():
    """Three bfloat16 pieces hold a float: rows of very large and very small values."""
    import torch
    q, s, _ = weights((64, 256), 128, "float32", False, 10)
    w = t2sp_amd.pack_w4(q, s, group=128)
    for scale in (2.0 ** 90, 2.0 ** -90, 1.0 / 3.0):
        x = rows(3, 256, "float32", 11) * scale
        close(t2sp_amd.gemv_w4(x, w), x, q, s, None, 128)


def test_on_a_side_stream_and_in_a_graph():
    import torch
    q, s, z = weights((4, 100, 700), 64, "bfloat16", True, 12)
    w, w0 = t2sp_amd.pack_w4(q, s, z, group=64), t2sp_amd.pack_w4(q[0], s[0], z[0], group=64)
    x, ids = rows(6, 700, "bfloat16", 13), torch.tensor([0, 3, 1, 1, 2, 0], dtype=torch.int32).cuda()
    want = (t2sp_amd.gemv_w4(x, w, ids=ids), t2sp_amd.gemv_w4(x, w0))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = (t2sp_amd.gemv_w4(x, w, ids=ids), t2sp_amd.gemv_w4(x, w0))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = (t2sp_amd.gemv_w4(x, w, ids=ids), t2sp_amd.gemv_w4(x, w0))
    for _ in range(3):
        for r in res:
            r.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, res))
    ids.copy_(torch.tensor([3, 3, 3, 3, 3, 3], dtype=torch.int32))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(res[0], t2sp_amd.gemv_w4(x, w, ids=ids))
