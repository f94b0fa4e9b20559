"""GPU tests of fused_linear in threads that have made no CUDA call of their own: the driver has no context bound to them. Each
runs in a process of its own, as any earlier call may have bound one to autograd's thread. (Values are compared by one rounding of the
largest: y is below 1, dx below 64, db below 256; 2^-8 of these and as much again.)"""
import subprocess
import sys
import textwrap

import pytest

pytestmark = pytest.mark.gpu

HEAD = """
import threading, torch
from compactwarprnntloss_b200 import fused_linear
g = torch.Generator().manual_seed(1)
x, w, b = (torch.randn(s, generator=g).to(torch.%s).cuda() for s in ((260, 64), (256, 64), (256,)))
dy = torch.ones(260, 256, dtype=x.dtype, device="cuda")
torch.cuda.synchronize()
"""
FORWARD = """
got = []
def call():
    got.append(fused_linear(x, w, b, activation="tanh"))
t = threading.Thread(target=call); t.start(); t.join()
assert len(got) == 1
torch.cuda.synchronize()
want = torch.tanh(x.double() @ w.double().t() + b.double())
assert float((got[0].double() - want).abs().max()) < 2 * 2.0 ** -8
"""
BACKWARD = """
leaves = [t.requires_grad_(True) for t in (x, w, b)]
y = fused_linear(*leaves, activation="tanh")
grads = torch.autograd.grad([y], leaves, [dy])
z = (x.detach().double() @ w.detach().double().t() + b.detach().double())
dz = 1 - torch.tanh(z) ** 2
assert float((grads[0].double() - dz @ w.detach().double()).abs().max()) < 2 * 64 * 2.0 ** -8
assert float((grads[2].double() - dz.sum(0)).abs().max()) < 2 * 256 * 2.0 ** -8
"""


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("body", [FORWARD, BACKWARD], ids=["forward", "backward"])
def test_a_thread_without_a_context(body, dtype):
    code = textwrap.dedent(HEAD % dtype + body)
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
