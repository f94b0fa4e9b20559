"""CPU-side checks of the row operators' and the linear layers' argument checks and host plans."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from compactwarprnntloss_b200 import capi, distill_loss, fused_linear, token_scores

ONE = ctypes.c_void_p(256)  # never followed: the call is refused first, or has no rows


def _rows(**kw):
    d = dict(n_rows=10, x_stride=64, grad_stride=64, temperature=1.0, V=64, dtype=capi.F16, n_list=2, top_k=0)
    d.update(kw)
    return ctypes.byref(capi.Rows(**d))


@pytest.mark.parametrize("upstream,row_loss,loss,grad", [(None, None, None, ONE), (ONE, ONE, None, ONE), (ONE, None, ONE, ONE),
                                                         (ONE, None, None, None)])
def test_a_gradient_is_made_anew_from_a_factor_and_into_a_gradient_only(upstream, row_loss, loss, grad):
    call = capi.lib().cwrnnt_distill
    for stride in (capi.UPSTREAM_UNLESS_ONE,):
        assert call(_rows(), 1, ONE, ONE, ONE, None, upstream, stride, 1.0, ONE, 1 << 20, row_loss, loss, grad, None) == 1
    assert call(_rows(n_rows=0), 1, None, None, None, None, None, capi.UPSTREAM_UNLESS_ONE, 1.0, None, 0, None, None, None,
                None) == 0
    assert call(_rows(), 1, ONE, ONE, ONE, None, ONE, -2, 1.0, ONE, 1 << 20, None, None, ONE, None) == 1


def test_tangents_are_refused():
    """A dual tensor does not require a gradient: without a check its tangent would be dropped without a word. (Whether the
    tensors are on a GPU is looked at later.)"""
    x, t = torch.randn(4, 9), torch.zeros(4, 2, dtype=torch.int32)
    a, w = torch.randn(4, 8).bfloat16(), torch.randn(6, 8).bfloat16()
    b, r = torch.randn(6).bfloat16(), torch.randn(4, 6).bfloat16()
    with fwAD.dual_level():
        dual = lambda v: fwAD.make_dual(v, torch.ones_like(v))
        calls = [lambda: token_scores(dual(x), t), lambda: token_scores(dual(x), entropy=True),
                 lambda: distill_loss(dual(x), torch.zeros(4, 2), t),
                 lambda: distill_loss(dual(x), torch.zeros(4, 2), t, reduction="none", eager_grad=False),
                 lambda: fused_linear(dual(a), w), lambda: fused_linear(a, dual(w)),
                 lambda: fused_linear(a, w, dual(b)), lambda: fused_linear(a, w, b, dual(r), activation="tanh")]
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="CUDA"):  # no tangent: the next check
            token_scores(x, t)


@pytest.mark.parametrize("n_in", [1, 64, 640, 1984, 1985, 2048, 20000])
@pytest.mark.parametrize("n_out", [1, 48, 1024, 2048, 50257])
def test_layers_without_rows_have_a_workspace(n_in, n_out):
    """No rows are no tiles; how a long sum is split over few tiles is not to divide by their number."""
    L = capi.lib()
    for act in range(4):
        p = ctypes.byref(capi.Linear(0, n_in, n_in, n_out, n_in, n_out, capi.BF16, act))
        for which in range(3):
            assert L.cwrnnt_linear_workspace_bytes(p, which) >= 256
        assert L.cwrnnt_linear_forward(p, None, None, None, None, None, 0, None, None) == 0
        assert L.cwrnnt_linear_backward(p, None, None, None, None, None, 0, None, None, None, None) == 0
