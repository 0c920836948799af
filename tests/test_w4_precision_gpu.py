"""GPU tests of the products with 4-bit weights beyond the bounds of test_w4_gpu.py: rows whose elements have one sign, rows
that are not finite or very large, and every form that a launch may take."""
import numpy as np
import pytest

import t2sp_amd
import test_products_plans as plans
from test_grouped_forms_gpu import on_full_card
from test_w4_gpu import TYPES, close, dt, rows, weights

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def exact(x, q, s, z, group):
    import torch
    of = torch.arange(q.shape[1], device="cuda") // group
    zz = z.double()[:, of] if z is not None else 8.0
    return x.double() @ ((q.double() - zz) * s.double()[:, of]).t()


@pytest.mark.parametrize("M", [1, 16, 40])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_float_rows_of_one_sign(M, zeros, group):
    """As exact as a direct product in float.  Per result 4096 / 8 inputs a wave: its own sum over groups (of partial sums that grow
    towards it, since x > 0 and q - 8 has a mean) rounds 4 to 16 times by at most u of its part, the join of eight waves by
    u (2 + ... + 8) / 8 of the result at worst, 2u typically (independent roundings of u / sqrt(3)); inside a group the sums are of
    128 / 4096 of the inputs and add less than u in the root of the mean square over the groups: 4u in norm.  Zero points between 0
    and 15 turn the groups' signs about: sums of 128 x (z - 8) against a result that grows with the root of the number of
    groups, twice that."""
    import torch
    K, N = 4096, 256
    q, s, z = weights((N, K), group, "float32", zeros, 1)
    s = s.abs() + 0.01
    x = 1.0 + 0.1 * rows(M, K, "float32", 2)
    y = t2sp_amd.gemv_w4(x, t2sp_amd.pack_w4(q, s, z, group=group))
    want = exact(x, q, s, z, group)
    close(y, x, q, s, z, group)
    assert float((y.double() - want).norm() / want.norm()) <= (8 if zeros else 4) * U


def same_kind(y, x, q, s, z, group):
    """y against the definition, with its infinities and NaN; finite values within the bound of test_w4_gpu.py (which covers a
    sum in the order of the inputs too)."""
    import torch
    of = torch.arange(q.shape[1], device="cuda") // group
    zz = z.double()[:, of] if z is not None else 8.0
    w = (q.double() - zz) * s.double()[:, of]
    want = torch.stack([(row[None, :] * w).sum(1) for row in x.double()])
    top = torch.finfo(y.dtype).max
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    infinite = torch.isinf(want)
    assert torch.equal(y.double()[infinite], want[infinite])
    finite = torch.isfinite(want) & (want.abs() < top / 2)
    xx = torch.where(torch.isfinite(x.double()), x.double(), torch.zeros_like(x.double())).abs()
    bound = (q.shape[1] + 8) * U * (xx @ (s.double()[:, of].abs() * (16 + q.double() + 16 + zz)).t())
    if y.dtype != torch.float32:
        bound = bound + torch.finfo(y.dtype).eps / 2 * (want.abs() + bound) + torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps / 2
    assert ((y.double() - want).abs() <= bound)[finite].all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,N,K,group", [(1, 41, 304, 32), (20, 48, 304, 64), (50, 33, 300, 128), (3, 16, 40, 32)])
def test_rows_with_infinities(dtype, zeros, M, N, K, group):
    import torch
    q, s, z = weights((N, K), group, dtype, zeros, 3)
    x = rows(M, K, dtype, 4)
    w = t2sp_amd.pack_w4(q, s, z, group=group)
    plain = t2sp_amd.gemv_w4(x, w)
    x[M // 2, 7] = float("inf")
    x[M - 1, K - 1] = float("-inf")
    if M > 3:
        x[3, 5], x[3, 6] = float("inf"), float("-inf")
        x[4, 9], x[5, 11] = float("nan"), float("nan")
        x[5, 12] = float("inf")
    y = t2sp_amd.gemv_w4(x, w)
    same_kind(y, x, q, s, z, group)
    rest = torch.isfinite(x.float()).all(1)
    assert torch.equal(y[rest], plain[rest])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,K", [(1, 256), (18, 250), (40, 256)])
def test_rows_near_the_largest_number(dtype, zeros, M, K):
    """x (16 + q) leaves float's range, the result does not."""
    import torch
    q, s, z = weights((50, K), 64, dtype, zeros, 5)
    x = rows(M, K, dtype, 6)
    x[::2] *= 2.0 ** 121
    x[0, 3] = torch.finfo(dt(dtype)).max
    if dtype == "float32":
        x[M - 1, 4] = float(np.finfo(np.float32).max)        # rounds to infinity as a bfloat16
    y = t2sp_amd.gemv_w4(x, t2sp_amd.pack_w4(q, s, z, group=64))
    same_kind(y, x, q, s, z, 64)


@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_with_a_matrix_for_each_row(dtype):
    import torch
    E, N, K, group = 4, 40, 160, 32
    q, s, z = weights((E, N, K), group, dtype, True, 7)
    x = rows(6, K, dtype, 8)
    x[1, 3], x[2, 4], x[4, 5], x[5, 6] = float("inf"), float("nan"), float("-inf"), float("inf")
    ids = torch.tensor([0, 3, 1, 2, 3, -1], dtype=torch.int32).cuda()
    y = t2sp_amd.gemv_w4(x, t2sp_amd.pack_w4(q, s, z, group=group), ids=ids)
    for m, e in enumerate(ids.tolist()):
        if e >= 0:
            same_kind(y[m:m + 1], x[m:m + 1], q[e], s[e], z[e], group)
        else:
            assert (y[m] == 0).all()


@pytest.mark.parametrize("case", range(len(plans.W4)))
@pytest.mark.parametrize("zeros", [False, True])
def test_every_form_of_the_product(case, zeros):
    """Matrices whose last tiles are partial and whose last workgroup has tiles behind the last one."""
    import torch
    mt, nt, types, M, N, K, group = plans.W4[case]
    for dtype in types:
        assert plans.w4_form(on_full_card(), dtype, 0, M, N, K, group) == (mt, nt)
        q, s, z = weights((N, K), group, dtype, zeros, 9)
        x = rows(M, K, dtype, 10)
        out = torch.full((M + 1, N + 9), 7.0, dtype=dt(dtype), device="cuda")
        w = t2sp_amd.pack_w4(q, s, z, group=group)
        t2sp_amd.gemv_w4(x, w, out=out[:M, 3:N + 3])
        close(out[:M, 3:N + 3], x, q, s, z, group)
        assert (out[:, :3] == 7).all() and (out[:, N + 3:] == 7).all() and (out[M] == 7).all()
        x[M - 1, 1] = float("inf")
        y = t2sp_amd.gemv_w4(x, w)
        assert torch.equal(y[:M - 1], out[:M - 1, 3:N + 3])
        same_kind(y[M - 1:, -40:], x[M - 1:], q[-40:], s[-40:], None if z is None else z[-40:], group)
