"""GPU tests of distill_loss under an upstream gradient that is not 1, a loss scale above all: the gradient computed in the
forward call against the one computed late and against the 64-bit oracle.

Tolerance: the late pass carries the factor in float, so a gradient element is off by its terms' errors
(tests/rowops_bounds.py) and one rounding to its type, at whatever scale."""
import numpy as np
import pytest
import torch

from compactwarprnntloss_b200 import distill_loss
from tests import rowops_bounds as rb
from tests import rowops_oracle as ro

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64}
NODES = 314340.0  # lattice nodes that the mean is over


def _case(seed, R, V, K, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, V, generator=g, dtype=torch.float64) * 2.0
    t = x + 0.7 * torch.randn(R, V, generator=g, dtype=torch.float64)
    val, idx = torch.log_softmax(t, 1).topk(K, 1)
    return x.to(DT[dtype]), val.to(torch.float64 if dtype == "f64" else torch.float32), idx.int()


def _grad(x, val, idx, factor, eager, **kw):
    leaf = x.detach().clone().requires_grad_(True)
    loss = distill_loss(leaf, val, idx, eager_grad=eager, mean_denominator=NODES, **kw)
    g, = torch.autograd.grad([loss], [leaf], [torch.full_like(loss, factor)])
    return g


# registers with several rows and one row a warp, a CTA a row, a warp a row, and runs of rows
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("V,n,K", [(129, 40, 2), (1024, 40, 2), (1000, 9, 20), (9001, 6, 5), (4000, 4741, 3), (24, 303109, 2)])
def test_a_loss_scale_reaches_a_float16_gradient_before_its_rounding(V, n, K, tail):
    m = min(n, 40)
    x, val, idx = _case(V, m, V, K, "f16")
    times = lambda t: t.repeat((n + m - 1) // m, 1)[:n].contiguous().to(DEV)
    xd, vd, idd = times(x), times(val), times(idx)
    for factor in (65536.0, 1.0, 0.5, -3.0, 0.0):
        late = _grad(xd, vd, idd, factor, False, tail=tail)
        eager = _grad(xd, vd, idd, factor, True, tail=tail)
        assert torch.equal(eager, late)
        _, want, _, mag = ro.distill(x.double().numpy(), val.double().numpy(), idx.numpy(), None, tail, 1.0)
        want, mag = want * factor / NODES, mag * abs(factor) / NODES
        bound = ro.HALF_STEP["float16"] * np.abs(want) + 2 * (rb.sum_error(V, 2) + rb.term_error(2)) * mag + ro.TINY["float16"]
        assert (np.abs(eager[:m].double().cpu().numpy() - want) <= bound).all()
    # a token of probability 1e-3 at that scale: 3e-9, nothing in float16, before it is scaled
    assert int((_grad(xd, vd, idd, 65536.0, True, tail=tail) != 0).sum()) > 1.2 * int((_grad(xd, vd, idd, 1.0, True, tail=tail) != 0).sum())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f64"])
def test_other_types_round_once_more(dtype):
    x, val, idx = _case(3, 30, 500, 4, dtype)
    args = (x.to(DEV), val.to(DEV), idx.to(DEV))
    late, eager = _grad(*args, 65536.0, False).double(), _grad(*args, 65536.0, True).double()
    half = ro.HALF_STEP[str(DT[dtype]).split(".")[1]]
    assert bool(((late - eager).abs() <= 2.1 * half * late.abs()).all())


def test_factors_that_are_not_finite():
    x, val, idx = (t.to(DEV) for t in _case(4, 20, 300, 3, "f16"))
    for factor in (float("inf"), float("nan")):
        late, eager = _grad(x, val, idx, factor, False), _grad(x, val, idx, factor, True)
        assert torch.equal(torch.nan_to_num(late, 7.0), torch.nan_to_num(eager, 7.0))


def test_a_loss_scale_that_changes_between_replays():
    """Loss and gradient in one graph, the loss scale a tensor of the program's, as a gradient scaler keeps it."""
    x, val, idx = (t.to(DEV) for t in _case(5, 60, 700, 3, "f16"))
    scale = torch.full((), 65536.0, device=DEV)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    leaf = x.clone()

    def step():
        y = leaf.detach().requires_grad_(True)
        loss = distill_loss(y, val, idx, mean_denominator=NODES)
        return torch.autograd.grad([loss], [y], [scale])[0]

    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        g = step()
    for seed, factor in ((6, 65536.0), (7, 1.0), (8, 1.0), (9, 1024.0)):
        new = _case(seed, 60, 700, 3, "f16")[0].to(DEV)
        leaf.copy_(new)
        scale.fill_(factor)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(g, _grad(new, val, idx, factor, False))


def test_logits_that_changed_before_backward_are_refused():
    x, val, idx = (t.to(DEV) for t in _case(10, 20, 300, 3, "f16"))
    leaf = x.clone().requires_grad_(True)
    y = leaf * 1.0
    loss = distill_loss(y, val, idx)
    with torch.no_grad():
        y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        (65536.0 * loss).backward()
