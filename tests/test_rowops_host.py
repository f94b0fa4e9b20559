"""CPU-side checks of the operators on rows of logits: the C ABI refuses bad descriptions, null pointers and workspaces
before any launch, and the Python entry points refuse what they cannot take."""
import ctypes

import pytest
import torch

from compactwarprnntloss_b200 import capi, distill_loss, token_scores


def _rows(**kw):
    d = dict(n_rows=10, x_stride=64, grad_stride=64, temperature=1.0, V=64, dtype=capi.F32, n_list=2, top_k=0)
    d.update(kw)
    return ctypes.byref(capi.Rows(**d))


BAD = [dict(n_rows=-1), dict(n_rows=2 ** 31), dict(V=0), dict(V=-3), dict(x_stride=63), dict(dtype=4), dict(dtype=-1),
       dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")),
       dict(n_list=-1), dict(n_list=33), dict(top_k=-1), dict(top_k=33), dict(V=8, top_k=9)]


@pytest.mark.parametrize("bad", BAD)
def test_bad_descriptions_are_refused(bad):
    L = capi.lib()
    one = ctypes.c_void_p(256)  # never followed: the description is refused first
    assert L.cwrnnt_token_scores(_rows(**bad), one, one, one, one, one, one, one, None) == 1
    assert L.cwrnnt_token_scores_backward(_rows(**bad), one, one, one, one, one, one, one, one, one, None) == 1
    assert L.cwrnnt_distill(_rows(**bad), 1, one, one, one, None, None, 0, 1.0, one, 1 << 20, one, one, one, None) == 1
    assert L.cwrnnt_distill_workspace_bytes(_rows(**bad)) < 0


def test_missing_pointers_and_workspaces_are_refused():
    L = capi.lib()
    one = ctypes.c_void_p(256)
    assert L.cwrnnt_token_scores(None, one, one, one, one, one, one, one, None) == 1
    assert L.cwrnnt_token_scores(_rows(), None, one, one, None, None, None, None, None) == 1       # x
    assert L.cwrnnt_token_scores(_rows(), one, None, one, None, None, None, None, None) == 1       # targets
    assert L.cwrnnt_token_scores(_rows(), one, one, None, None, None, None, None, None) == 1       # log_probs
    assert L.cwrnnt_token_scores(_rows(n_list=0, top_k=3), one, None, None, None, one, None, None, None) == 1
    assert L.cwrnnt_token_scores(_rows(n_list=0, top_k=3), one, None, None, None, None, one, None, None) == 1
    back = L.cwrnnt_token_scores_backward
    assert back(_rows(), one, one, None, None, None, one, None, None, one, None) == 1              # lse
    assert back(_rows(), one, one, None, one, None, one, None, None, None, None) == 1              # grad_x
    assert back(_rows(), one, None, None, one, None, one, None, None, one, None) == 1              # targets
    assert back(_rows(), one, one, None, one, None, None, one, None, one, None) == 1               # entropy
    assert back(_rows(grad_stride=63), one, one, None, one, None, one, None, None, one, None) == 1
    assert back(_rows(n_list=0, top_k=2), one, None, None, one, None, None, None, one, one, None) == 1
    d = L.cwrnnt_distill
    assert d(_rows(), 1, None, one, one, None, None, 0, 1.0, one, 1 << 20, one, one, one, None) == 1
    assert d(_rows(), 1, one, None, one, None, None, 0, 1.0, one, 1 << 20, one, one, one, None) == 1
    assert d(_rows(), 1, one, one, None, None, None, 0, 1.0, one, 1 << 20, one, one, one, None) == 1
    assert d(_rows(), 2, one, one, one, None, None, 0, 1.0, one, 1 << 20, one, one, one, None) == 1
    assert d(_rows(), 1, one, one, one, None, None, 2, 1.0, one, 1 << 20, one, one, one, None) == 1
    assert d(_rows(n_list=0), 1, one, one, one, None, None, 0, 1.0, one, 1 << 20, one, one, one, None) == 1
    assert d(_rows(grad_stride=1), 1, one, one, one, None, None, 0, 1.0, one, 1 << 20, one, one, one, None) == 1
    n = L.cwrnnt_distill_workspace_bytes(_rows())
    assert n >= 8 * 10
    assert d(_rows(), 1, one, one, one, None, None, 0, 1.0, None, n, one, one, one, None) == 2
    assert d(_rows(), 1, one, one, one, None, None, 0, 1.0, one, n - 1, one, one, one, None) == 2
    assert d(_rows(), 1, one, one, one, None, None, 0, 1.0, ctypes.c_void_p(260), n, one, one, one, None) == 2


def test_no_rows_is_no_work():
    L = capi.lib()
    assert L.cwrnnt_token_scores(_rows(n_rows=0), None, None, None, None, None, None, None, None) == 0
    assert L.cwrnnt_token_scores_backward(_rows(n_rows=0), None, None, None, None, None, None, None, None, None, None) == 0
    assert L.cwrnnt_distill(_rows(n_rows=0), 1, None, None, None, None, None, 0, 1.0, None, 0, None, None, None, None) == 0


def test_python_entry_points_refuse_what_they_cannot_take():
    x = torch.zeros(4, 9)
    t = torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(AssertionError):
        token_scores(x)                                   # nothing asked for
    with pytest.raises(AssertionError):
        token_scores(x, t.long())                         # int64 targets
    with pytest.raises(AssertionError):
        token_scores(x, t[:3])                            # another number of rows
    with pytest.raises(RuntimeError, match="CUDA"):
        token_scores(x, t)                                # not on a GPU
    v = torch.zeros(4, 2)
    for bad in (dict(teacher=v.double()), dict(teacher=v[:, :1]), dict(indices=t.long()), dict(weight=torch.zeros(3)),
                dict(weight=torch.zeros(4, dtype=torch.float64)), dict(reduction="max"),
                dict(teacher=torch.zeros(4, 33), indices=torch.zeros(4, 33, dtype=torch.int32)),
                dict(teacher=torch.zeros(4, 0), indices=torch.zeros(4, 0, dtype=torch.int32))):
        kw = dict(teacher=v, indices=t)
        kw.update(bad)
        with pytest.raises(AssertionError):
            distill_loss(x, kw.pop("teacher"), kw.pop("indices"), **kw)
    with pytest.raises(RuntimeError, match="CUDA"):
        distill_loss(x, v, t)


def _linear(**kw):
    d = dict(n_rows=64, x_stride=32, w_stride=32, g_stride=48, n_in=32, n_out=48, dtype=capi.BF16, activation=0)
    d.update(kw)
    return ctypes.byref(capi.Linear(**d))


LINEAR_BAD = [dict(n_rows=-1), dict(n_rows=2 ** 31), dict(n_in=0), dict(n_out=0), dict(n_in=2 ** 25), dict(x_stride=31),
              dict(w_stride=31), dict(x_stride=2 ** 39), dict(dtype=capi.F32), dict(dtype=capi.F64), dict(dtype=9),
              dict(activation=-1), dict(activation=4)]


@pytest.mark.parametrize("bad", LINEAR_BAD)
def test_bad_linear_layers_are_refused(bad):
    L = capi.lib()
    one = ctypes.c_void_p(256)
    assert L.cwrnnt_linear_workspace_bytes(_linear(**bad), 0) < 0
    assert L.cwrnnt_linear_forward(_linear(**bad), one, one, one, one, one, 1 << 40, one, None) == 1
    assert L.cwrnnt_linear_backward(_linear(**bad), one, one, one, one, one, 1 << 40, one, one, one, None) == 1


def test_linear_pointers_and_workspaces():
    L = capi.lib()
    one, odd = ctypes.c_void_p(256), ctypes.c_void_p(264)
    n, m = L.cwrnnt_linear_workspace_bytes(_linear(), 0), L.cwrnnt_linear_workspace_bytes(_linear(), 1)
    assert n >= 256 and m >= 256
    assert L.cwrnnt_linear_workspace_bytes(_linear(x_stride=33), 0) >= 64 * 32 * 2  # a copy of x
    f, b = L.cwrnnt_linear_forward, L.cwrnnt_linear_backward
    assert f(None, one, one, None, None, one, n, one, None) == 1
    assert f(_linear(), None, one, None, None, one, n, one, None) == 1
    assert f(_linear(), one, None, None, None, one, n, one, None) == 1
    assert f(_linear(), one, one, None, None, one, n, None, None) == 1
    assert f(_linear(), odd, one, None, None, one, n, one, None) == 1      # off a 16-byte boundary
    assert f(_linear(), one, odd, None, None, one, n, one, None) == 1
    assert f(_linear(), one, one, None, odd, one, 1 << 40, one, None) == 1
    assert L.cwrnnt_linear_workspace_bytes(_linear(), 3) < 0 and L.cwrnnt_linear_workspace_bytes(_linear(), -1) < 0
    assert L.cwrnnt_linear_workspace_bytes(_linear(n_out=47), 2) >= 64 * 48 * 2  # a copy of the residual
    assert f(_linear(), one, one, None, None, None, n, one, None) == 2
    assert f(_linear(), one, one, None, None, odd, n, one, None) == 2
    assert f(_linear(), one, one, None, None, one, n - 1, one, None) == 2
    assert b(_linear(g_stride=47), one, one, None, one, one, m, one, one, one, None) == 1
    assert b(_linear(), one, one, None, None, one, m, one, one, one, None) == 1
    assert b(_linear(), one, one, None, odd, one, m, one, one, one, None) == 1
    assert b(_linear(), one, one, None, one, one, m - 1, one, one, one, None) == 2
    assert f(_linear(n_rows=0), None, None, None, None, None, 0, None, None) == 0
    assert b(_linear(n_rows=0), None, None, None, None, None, 0, None, None, None, None) == 0


def test_fused_linear_refuses_what_it_cannot_take():
    from compactwarprnntloss_b200 import fused_linear
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(6, 8, dtype=torch.bfloat16)
    for args, kw in (((x.float(), w.float()), {}), ((x.double(), w.double()), {}), ((x, w[:, :7]), {}),
                     ((x, w, torch.zeros(5)), {}), ((x, w, None, torch.zeros(4, 5)), {}), ((x, w), dict(activation="gelu"))):
        with pytest.raises(AssertionError):
            fused_linear(*args, **kw)
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_linear(x, w)


def test_every_linear_layer_has_a_workspace():
    """The plans of all sizes are host arithmetic: both passes, widths and lengths around every tile and split."""
    L = capi.lib()
    sizes = (1, 7, 8, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 640, 1000, 1024, 4096, 20000)
    for m in (1, 16, 17, 128, 129, 256, 1000, 9001, 40009, 314340, 2 ** 31 - 1024):
        for n in sizes:
            for k in sizes:
                for act in (0, 2):
                    p = ctypes.byref(capi.Linear(m, k, k, n, k, n, capi.BF16, act))
                    f, b = L.cwrnnt_linear_workspace_bytes(p, 0), L.cwrnnt_linear_workspace_bytes(p, 1)
                    assert f >= 256 and b >= 256 and f % 256 == 0 and b % 256 == 0
