"""GPU tests of token_scores' gradient on rows whose logits are all -inf, under upstream gradients that are not finite: what a
logsumexp or a product with -inf hands back. It is zero, as for any other upstream gradient, and the other rows' is untouched."""
import pytest
import torch

from compactwarprnntloss_b200 import token_scores

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64}


@pytest.mark.parametrize("V,dtype", [(12, "f32"), (130, "f16"), (1024, "bf16"), (5000, "f32"), (70001, "f16"), (200, "f64")])
def test_an_empty_row_has_no_gradient_whatever_comes_from_above(V, dtype):
    g = torch.Generator().manual_seed(V)
    x = torch.randn(6, V, generator=g).to(DT[dtype]).to(DEV)
    x[2] = float("-inf")
    x[5] = float("-inf")
    t = torch.randint(0, V, (6, 2), generator=g, dtype=torch.int32).to(DEV)

    def grad(bad):
        leaf = x.clone().requires_grad_(True)
        s = token_scores(leaf, t, top_k=3, entropy=True)
        up = [torch.ones_like(o) for o in (s.log_probs, s.entropy, s.top_log_probs)]
        if bad is not None:
            for u in up:
                u[2] = bad
        return torch.autograd.grad([s.log_probs, s.entropy, s.top_log_probs], [leaf], up)[0]

    want = grad(None)
    assert not want[2].any() and not want[5].any()
    for bad in (float("nan"), float("inf"), float("-inf")):
        assert torch.equal(grad(bad), want)


def test_logsumexp_over_the_targets_of_an_empty_row():
    x = torch.randn(3, 50, device=DEV)
    x[1] = float("-inf")
    leaf = x.requires_grad_(True)
    lp = token_scores(leaf, torch.tensor([[1, 2]] * 3, dtype=torch.int32, device=DEV)).log_probs
    torch.logsumexp(lp, 1)[[0, 2]].sum().backward(retain_graph=True)
    assert bool(torch.isfinite(leaf.grad).all())
    leaf.grad = None
    (lp * torch.tensor([[1.0], [float("nan")], [1.0]], device=DEV)).nansum().backward()
    assert bool(torch.isfinite(leaf.grad).all()) and not leaf.grad[1].any()
