"""GPU tests of distill_loss with its forward and its backward captured in graphs of their own."""
import pytest
import torch

from compactwarprnntloss_b200 import distill_loss

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_backward_in_a_graph_of_its_own_is_replayed_by_itself(dtype):
    """Every replay of the backward graph gives the gradient for the upstream gradient of that moment, however often it
    is replayed for one replay of the forward graph."""
    g = torch.Generator(DEV).manual_seed(1)
    x = torch.randn(50, 300, generator=g, device=DEV).to(dtype)
    val, idx = torch.log_softmax(torch.randn(50, 300, generator=g, device=DEV), 1).topk(3, 1)
    idx = idx.int()
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = x.clone().requires_grad_(True)
        up = torch.ones((), device=DEV)
        torch.autograd.grad([distill_loss(leaf, val, idx, reduction="sum")], [leaf], [up])
    side.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first, stream=side):
        loss = distill_loss(leaf, val, idx, reduction="sum")
    with torch.cuda.graph(second, stream=side, pool=first.pool()):
        got, = torch.autograd.grad([loss], [leaf], [up])
    for seed, factors in ((2, (0.5, 0.5, 1.0, -2.0)), (3, (1.0, 4.0, 4.0))):
        with torch.no_grad():
            leaf.copy_(torch.randn(50, 300, generator=g, device=DEV).to(dtype))
        torch.cuda.synchronize()
        first.replay()
        for factor in factors:
            up.fill_(factor)
            torch.cuda.synchronize()
            second.replay()
            torch.cuda.synchronize()
            other = leaf.detach().clone().requires_grad_(True)
            want, = torch.autograd.grad([distill_loss(other, val, idx, reduction="sum", eager_grad=False)], [other],
                                        [torch.full((), factor, device=DEV)])
            assert torch.equal(got, want), (seed, factor)
