"""GPU tests of the products with 4-bit weights beyond the bounds of test_w4_gpu.py: rows whose elements have one sign, rows
that are not finite or very large, and every form that a launch may take."""
import numpy as np
import pytest

import t2sp_amd
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
