"""GPU tests of the cross entropy in every form that a launch may take (the tables of test_products_plans.py); tolerances as
derived in test_xent_gpu.py."""
import pytest

import t2sp_amd
import test_products_plans as plans
from test_grouped_forms_gpu import on_full_card
from test_xent_gpu import check, dt, labels_for, make, mean_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case,dtype", [(i, t) for i, case in enumerate(plans.XENT) for t in case[2]])
def test_every_form_of_the_cross_entropy(case, dtype):
    import torch
    tile, grad, _, T, V, D = plans.XENT[case]
    assert plans.xent_form(on_full_card(), dtype, T, V, D)[:2] == (tile, grad)
    H, W, lab = make((T, D), dtype, 1), make((V, D), dtype, 2, 2.0 * D ** -0.5), labels_for(T, V, 3)
    lab[0], lab[T - 1] = V - 1, 0                            # the last word of the last tile, the first of the first
    d = mean_of(lab, V)
    loss, lse, dH, dW = check(H, W, lab, d)
    if dtype != "float32":
        check(H, W, lab, d, out_dtype=torch.float32)
        rH, rW = t2sp_amd.xent_grad(H, W, lab, lse, d, rounded=True)
        eps = torch.finfo(dt(dtype)).eps
        for a, b in ((rH, dH), (rW, dW)):
            assert float((a.double() - b.double()).norm() / b.double().norm()) < eps
