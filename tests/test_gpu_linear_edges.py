"""GPU tests of fused_linear at its edges: batches without rows and infinite weights."""
import pytest
import torch

from compactwarprnntloss_b200 import fused_linear

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("act", [None, "tanh"])
@pytest.mark.parametrize("n_in,n_out", [(2048, 40), (40, 2048), (4096, 4096)])
def test_no_rows_and_a_long_sum(n_in, n_out, act):
    x = torch.zeros(0, n_in, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    w = torch.ones(n_out, n_in, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    b = torch.ones(n_out, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    y = fused_linear(x, w, b, activation=act)
    assert y.shape == (0, n_out)
    y.sum().backward()
    assert x.grad.shape == x.shape and not w.grad.any() and not b.grad.any()
