"""GPU tests of rows that lie far apart: the last hidden states of sequences, views of one row."""
import pytest

import t2sp_amd
from test_grouped_gpu import TYPES, make, offs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B", [1, 3])
def test_last_token_of_each_sequence(dtype, B):
    """Rows 9 MB apart (18 MB for floats), off and on the vector grid."""
    import torch
    for K in (4096, 4090):
        hidden = make((B, 1152, K), dtype, 1)
        x = hidden[:, -1]
        assert x.stride(0) * x.element_size() > 1 << 23
        q = torch.randint(0, 16, (40, K), generator=torch.Generator().manual_seed(2), dtype=torch.uint8).cuda()
        w = t2sp_amd.pack_w4(q, make((40, -(-K // 128)), dtype, 3), group=128)
        assert torch.equal(t2sp_amd.gemv_w4(x, w), t2sp_amd.gemv_w4(x.contiguous(), w))
        W, off = make((1, K, 24), dtype, 4), offs([B])
        assert torch.equal(t2sp_amd.gemm_grouped(x, W, off), t2sp_amd.gemm_grouped(x.contiguous(), W, off))
        V, lab = make((50, K), dtype, 5, 0.02), torch.arange(B, device="cuda")
        for a, b in zip(t2sp_amd.xent(x, V, lab), t2sp_amd.xent(x.contiguous(), V, lab)):
            assert torch.equal(a, b)


def test_one_row_of_any_stride():
    """A stride beyond every limit, which a single row (or matrix) does not use."""
    import torch
    K, far = 64, 1 << 40
    x0, W0 = make((1, K), "bfloat16", 6), make((1, K, 8), "bfloat16", 7)
    x, W = torch.as_strided(x0, (1, K), (far, 1)), torch.as_strided(W0, (1, K, 8), (far, 8, 1))
    off = offs([1])
    assert torch.equal(t2sp_amd.gemm_grouped(x, W, off), t2sp_amd.gemm_grouped(x0, W0, off))
    assert torch.equal(t2sp_amd.gemm_grouped_wgrad(x, x, off), t2sp_amd.gemm_grouped_wgrad(x0, x0, off))
    q = torch.ones((16, K), dtype=torch.uint8, device="cuda")
    w = t2sp_amd.pack_w4(q, make((16, 1), "bfloat16", 8), group=64)
    assert torch.equal(t2sp_amd.gemv_w4(x, w), t2sp_amd.gemv_w4(x0, w))


def test_rows_that_overlap_are_refused():
    import torch
    x, W, off = make((1, 64), "bfloat16", 9).expand(4, 64), make((1, 64, 8), "bfloat16", 10), offs([4])
    with pytest.raises(t2sp_amd.T2spError) as e:
        t2sp_amd.gemm_grouped(x, W, off)
    assert e.value.code == -8
