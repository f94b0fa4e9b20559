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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["relu", "tanh", "silu"])
@pytest.mark.parametrize("M,N,K", [(70, 64, 64), (33, 40, 72), (300, 264, 136), (5, 40, 72)])
def test_an_infinite_weight_leaves_the_sums_over_rows_finite(M, N, K, act, dtype):
    """Every z of a column with an infinite weight is infinite, its slope 0 or 1: the gradients of bias and weight are sums
    over the rows that there are, whatever stands behind the last one in a tile. (db: one rounding of dz in two parts below
    2^-15 each, M additions, one rounding.)"""
    g = torch.Generator().manual_seed(M)
    x = torch.rand(M, K, generator=g).add(0.1).to(dtype)
    w = (torch.randn(N, K, generator=g) * K ** -0.5).to(dtype)
    w[3, 5], w[N - 1, 0] = float("inf"), float("-inf")
    b = torch.randn(N, generator=g).to(dtype)
    dy = torch.randn(M, N, generator=g).to(dtype)
    leaves = [t.to(DEV).requires_grad_(True) for t in (w, b)]
    y = fused_linear(x.to(DEV), *leaves, activation=act)
    dw, db = torch.autograd.grad([y], leaves, [dy.to(DEV)])
    z = (x.double() @ w.double().t() + b.double()).requires_grad_(True)
    a = {"relu": torch.relu, "tanh": torch.tanh, "silu": lambda v: v.clamp(-104, 104) * torch.sigmoid(v)}[act](z)
    dz, = torch.autograd.grad(a, z, dy.double())
    dz = dz.detach()
    if act == "silu":  # the slope's limits
        dz[:, 3], dz[:, N - 1] = dy[:, 3].double(), 0.0
    eps = torch.finfo(dtype).eps / 2
    zerr = (K / 16 + 8) * 2.0 ** -21 * (x.double().abs() @ w.double().abs().t() + b.double().abs())
    zerr[~torch.isfinite(z.detach())] = 0.0
    near = (z.detach().abs() <= zerr) if act == "relu" else torch.zeros_like(dz, dtype=torch.bool)
    delta = 2.0 ** -15 * dz.abs() + dy.double().abs() * (zerr + 2.0 ** -20 + near) + torch.finfo(dtype).smallest_normal * 2.0 ** -10
    want = dz.sum(0)
    bound = eps * want.abs() + 1.01 * delta.sum(0) + M * 2.0 ** -24 * dz.abs().sum(0) + torch.finfo(dtype).smallest_normal
    assert bool(((db.double().cpu() - want).abs() <= bound).all()), (db, want)
    want = dz.t() @ x.double()
    bound = eps * want.abs() + 1.01 * delta.t() @ x.double() + (M / 16 + 8) * 2.0 ** -21 * dz.abs().t() @ x.double()
    assert bool(((dw.double().cpu() - want).abs() <= bound + torch.finfo(dtype).smallest_normal).all())
