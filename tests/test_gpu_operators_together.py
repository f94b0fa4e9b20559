"""GPU tests of the operators around the lattice in a run, as a program uses them: a captured training step of hidden layer,
output layer, scores and distillation through autograd, and the same step from several host threads at once. Each replay and
each thread gives the bits of a call on its own."""
import threading

import pytest
import torch

from compactwarprnntloss_b200 import distill_loss, fused_linear, token_scores

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _inputs(seed, dtype, rows=700, H=96, V=520):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)
    x, w1, w2, b2 = make(rows, H), make(H, H) * 0.1, make(V, H) * 0.1, make(V)
    teacher, t = make(rows, V), torch.randint(0, V, (rows, 2), generator=g, dtype=torch.int32).to(DEV)
    return x, w1, w2, b2, teacher, t


def _step(x, w1, w2, b2, teacher, t):
    leaves = [v.detach().requires_grad_(True) for v in (x, w1, w2, b2)]
    h = fused_linear(leaves[0], leaves[1], None, leaves[0], activation="silu")
    logits = fused_linear(h, leaves[2], leaves[3])
    with torch.no_grad():
        best = token_scores(teacher, top_k=8)
    s = token_scores(logits, t, entropy=True)
    loss = distill_loss(logits, best.top_log_probs, best.top_indices) - 0.1 * s.log_probs.mean() - 0.01 * s.entropy.mean()
    return [loss.detach(), *torch.autograd.grad([loss], leaves)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_captured_training_step(dtype):
    static = _inputs(1, dtype)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(*static)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = _step(*static)
    for seed in (2, 3):
        new = _inputs(seed, dtype)
        for dst, src in zip(static, new):
            dst.copy_(src)
        torch.cuda.synchronize()
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, _step(*new)):
                assert torch.equal(a, b) and bool(torch.isfinite(a).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_threads_at_once(dtype):
    data = [_inputs(seed, dtype) for seed in range(10, 14)]
    want = [_step(*d) for d in data]
    torch.cuda.synchronize()
    bad = []

    def work(d, expected):
        try:
            stream = torch.cuda.Stream(DEV)
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got = _step(*d)
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, expected)):
                        bad.append("values")
        except Exception as e:  # a thread's exception would go unseen
            bad.append(repr(e))

    threads = [threading.Thread(target=work, args=a) for a in zip(data, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
