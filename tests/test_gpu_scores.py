"""GPU tests of token_scores against the 64-bit oracle: every type, row sizes on both sides of every kernel shape,
misaligned and strided rows, masks, ties, and the gradient against the formula and against differences.

Tolerances (tests/rowops_oracle.py derives the constants): a log-probability x/tau - lse is put together in double from
a sum good to SUM32, and rounded to float once; the entropy ln s - t/s carries that error of s and of t, the latter
weighed by sum p |ln p|; a gradient carries it per term, is rounded to the row's type once, and the same terms in 64
bits give its magnitude."""
import numpy as np
import pytest
import torch

from compactwarprnntloss_b200 import token_scores
from tests import rowops_oracle as ro

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64}


def _logits(seed, R, V, dtype, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(R, V, generator=g, dtype=torch.float64) * spread).to(dtype)


def _sum_error(dtype):
    return ro.SUM64 if dtype == torch.float64 else ro.SUM32


def _bound(name, want, mag, coef):
    flush, err = (0.0, ro.SUM64) if name == "float64" else (ro.FLUSH32, ro.SUM32)
    return ro.HALF_STEP[name] * np.abs(want) + 2 * err * mag + flush * coef + ro.TINY[name]


def _check(x, targets, k, tau, got, grads=None):
    """`got`: TokenScores for device rows equal to the CPU tensor x; grads: (upstream three, gradient)."""
    x64 = x.double().numpy()
    t = None if targets is None else targets.numpy()
    lps, ent, top, idx = ro.scores(x64, t, k, tau)
    err, unit = _sum_error(x.dtype), (2.0 ** -53 if x.dtype == torch.float64 else 2.0 ** -24)
    if targets is not None:
        np.testing.assert_allclose(got.log_probs.detach().double().cpu().numpy(), lps, atol=err, rtol=2 * unit)
    if got.entropy is not None:
        np.testing.assert_allclose(got.entropy.detach().double().cpu().numpy(), ent, atol=err, rtol=2 * err)
    if k:
        np.testing.assert_array_equal(got.top_indices.cpu().numpy(), idx)
        np.testing.assert_allclose(got.top_log_probs.detach().double().cpu().numpy(), top, atol=err, rtol=2 * unit)
    if grads is not None:
        (g_lp, g_ent, g_top), gx = grads
        want, mag, coef = ro.scores_grad(x64, t, idx, *(None if g is None else g.double().numpy()
                                                  for g in (g_lp, g_ent, g_top)), tau)
        name = str(x.dtype).split(".")[1]
        bound = _bound(name, want, mag, coef)
        off = np.abs(gx.double().cpu().numpy() - want)
        assert gx.dtype == x.dtype and (off <= bound).all(), (off - bound).max()


def _run(x, targets, k, entropy, tau=1.0, seed=0):
    xd = x.to(DEV).requires_grad_(True)
    got = token_scores(xd, None if targets is None else targets.to(DEV), top_k=k, entropy=entropy, temperature=tau)
    g = torch.Generator().manual_seed(seed + 77)
    ct = torch.float64 if x.dtype == torch.float64 else torch.float32
    up = [None if o is None else torch.randn(o.shape, generator=g, dtype=ct)
          for o in (got.log_probs, got.entropy, got.top_log_probs)]
    pairs = [(o, u) for o, u in zip((got.log_probs, got.entropy, got.top_log_probs), up) if o is not None]
    gx, = torch.autograd.grad([o for o, _ in pairs], [xd], [u.to(DEV) for _, u in pairs])
    _check(x, targets, k, tau, got, (up, gx))
    with torch.no_grad():  # the same without a graph
        again = token_scores(xd, None if targets is None else targets.to(DEV), top_k=k, entropy=entropy,
                             temperature=tau)
    for a, b in zip(got, again):
        assert a is None and b is None or torch.equal(a, b)


def _targets(seed, R, V, P):
    g = torch.Generator().manual_seed(seed)
    t = torch.randint(0, V, (R, P), generator=g, dtype=torch.int32)
    if P > 1:
        t[::3, 1] = -1
        t[1::3, 1] = t[1::3, 0]  # the same token twice
    return t


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16", "f64"])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 31, 64, 127, 128, 136, 257, 512, 513, 1000, 1024, 1032, 2048, 2049, 4096,
                               4100, 9001, 33000])
def test_every_row_size(dtype, V):
    R = 5 if V > 2048 else 37
    k = min(V, 8)
    _run(_logits(V, R, V, DT[dtype]), _targets(V, R, V, 2), k, True)


@pytest.mark.parametrize("k", [1, 2, 3, 4, 5, 8, 16, 17, 31, 32])
@pytest.mark.parametrize("V,dtype", [(32, "f16"), (128, "f16"), (255, "f32"), (1024, "bf16"), (4096, "bf16"),
                                     (5001, "f16"), (300, "f64")])
def test_every_list_length(k, V, dtype):
    _run(_logits(k, 9, V, DT[dtype]), None, k, False)
    _run(_logits(k, 3, V, DT[dtype]), _targets(k, 3, V, 32), k, True, tau=1.7)


@pytest.mark.parametrize("k", [2, 4, 8, 16, 32])
@pytest.mark.parametrize("dtype", ["f16", "f32", "f64"])
def test_rows_of_about_as_many_vectors_as_entries_wanted(k, dtype):
    """Fewer vectors than entries: every entry is a candidate, and the largest may all lie in one vector."""
    per = 16 // torch.empty(0, dtype=DT[dtype]).element_size()
    for V in {max(k, (k + d) * per + e) for d in (-1, 0, 1) for e in (-1, 0, 1)}:
        x = _logits(V, 11, V, DT[dtype])
        x[1] = x[1].sort(descending=True)[0]
        x[2] = x[2].sort()[0]
        _run(x, None, k, True)


@pytest.mark.parametrize("V,dtype", [(40, "f16"), (128, "bf16"), (1024, "f32"), (1023, "bf16"), (4096, "f16"),
                                     (6000, "f32"), (20011, "bf16")])
def test_equal_entries_go_to_the_lowest_index(V, dtype):
    g = torch.Generator().manual_seed(V)
    x = torch.randint(-2, 3, (7, V), generator=g).to(DT[dtype])  # five values only
    x[1] = 3.0                                                    # constant rows
    x[2] = 0.0
    x[3, ::2] = -0.0                                              # -0 equals 0
    x[4, :] = torch.arange(V).to(DT[dtype])                       # ascending, equal where the type runs out of steps
    _run(x, None, min(V, 32), True)
    _run(x, None, 3, False)


@pytest.mark.parametrize("V,dtype", [(12, "f32"), (128, "f16"), (1024, "bf16"), (1031, "f16"), (8200, "f32"),
                                     (200, "f64")])
def test_masks_infinities_and_nan(V, dtype):
    x = _logits(3, 12, V, DT[dtype])
    ninf = float("-inf")
    x[0] = ninf                              # nothing left
    x[1] = torch.finfo(DT[dtype]).min        # the type's lowest value everywhere
    x[2, 1:] = ninf                          # one entry left
    x[3, : V // 2] = ninf
    x[4, V // 3:] = torch.finfo(DT[dtype]).min
    x[5, V - 1] = float("nan")
    x[6, 0] = float("inf")
    x[7, 0], x[7, 3], x[7, 5] = float("nan"), float("inf"), float("nan")
    x[8] = float("nan")
    x[9, 1:] = torch.finfo(DT[dtype]).min
    x[9, 0] = torch.finfo(DT[dtype]).max
    k = min(V, 6)
    t = _targets(5, 12, V, 2)
    t[3, 0] = V // 2
    xd = x.to(DEV).requires_grad_(True)
    got = token_scores(xd, t.to(DEV), top_k=k, entropy=True)
    with np.errstate(over="ignore"):
        lps, ent, top, idx = ro.scores(x.double().numpy(), t.numpy(), k, 1.0)
    np.testing.assert_array_equal(got.top_indices.cpu().numpy(), idx)
    err = _sum_error(x.dtype)
    with np.errstate(over="ignore"):  # ln p of the lowest value beside the highest is beyond the type: -inf
        ct = np.float64 if dtype == "f64" else np.float32
        lps, top = lps.astype(ct), top.astype(ct)
    np.testing.assert_allclose(got.log_probs.detach().double().cpu().numpy(), lps, atol=err, rtol=err)
    np.testing.assert_allclose(got.entropy.detach().double().cpu().numpy(), ent, atol=err, rtol=2 * err)
    np.testing.assert_allclose(got.top_log_probs.detach().double().cpu().numpy(), top, atol=err, rtol=err)
    gx, = torch.autograd.grad([got.log_probs.sum(), got.entropy.sum()], [xd])
    gx = gx.double().cpu().numpy()
    ones = np.ones
    want, mag, coef = ro.scores_grad(x.double().numpy(), t.numpy(), idx, ones(t.shape), ones(12), None, 1.0)
    name = str(x.dtype).split(".")[1]
    for r in range(12):
        if np.isnan(ent[r]):
            assert np.isnan(gx[r]).all()
        else:
            bound = _bound(name, want[r], mag[r], coef[r])
            assert (np.abs(gx[r] - want[r]) <= bound).all(), r
    assert (gx[0] == 0).all()


def test_a_target_outside_the_row_gives_nan_and_no_gradient():
    x = _logits(1, 4, 50, torch.float32).to(DEV).requires_grad_(True)
    t = torch.tensor([[50, 1], [2, 3], [2147483647, -1], [-5, 4]], dtype=torch.int32, device=DEV)
    got = token_scores(x, t).log_probs
    nan = torch.isnan(got).cpu()
    assert nan.tolist() == [[True, False], [False, False], [True, False], [False, False]]
    assert float(got[2, 1].detach()) == 0.0 and float(got[3, 0].detach()) == 0.0
    gx, = torch.autograd.grad([got], [x], [torch.ones_like(got)])
    assert torch.isfinite(gx).all() and not gx[2].any()


@pytest.mark.parametrize("V,dtype", [(96, "bf16"), (1024, "f32"), (1030, "f16"), (5000, "bf16"), (64, "f64")])
def test_strided_and_misaligned_rows(V, dtype):
    wide = _logits(2, 11, V + 13, DT[dtype])
    dev = wide.to(DEV)
    t = _targets(2, 11, V, 2)
    for start in (0, 1, 5, 8):
        view = dev[:, start:start + V].detach().requires_grad_(True)
        assert not view.is_contiguous()
        got = token_scores(view, t.to(DEV), top_k=4, entropy=True)
        up = [torch.ones(o.shape, dtype=o.dtype) for o in (got.log_probs, got.entropy, got.top_log_probs)]
        gx, = torch.autograd.grad([got.log_probs, got.entropy, got.top_log_probs], [view], [u.to(DEV) for u in up])
        _check(wide[:, start:start + V], t, 4, 1.0, got, (up, gx))
    flat = dev.reshape(-1)[3:3 + 10 * V].view(10, V)  # contiguous, base not on a 16-byte boundary
    _check(flat.cpu(), t[:10], 4, 1.0, token_scores(flat, t[:10].to(DEV), top_k=4, entropy=True))
    turned = _logits(4, V, 6, DT[dtype]).to(DEV).t()  # columns contiguous, rows not: copied
    _check(turned.cpu().contiguous(), t[:6], 2, 1.0, token_scores(turned, t[:6].to(DEV), top_k=2))
    same = dev[:1, :V].expand(5, V)                   # one row five times
    _check(same.cpu().contiguous(), t[:5], 2, 1.0, token_scores(same, t[:5].to(DEV), top_k=2))


def test_leading_axes_empty_batches_and_single_targets():
    x = _logits(1, 24, 70, torch.float32)
    t = _targets(1, 24, 70, 3)
    got = token_scores(x.view(2, 3, 4, 70).to(DEV), t.view(2, 3, 4, 3).to(DEV), top_k=5, entropy=True)
    assert got.log_probs.shape == (2, 3, 4, 3) and got.entropy.shape == (2, 3, 4) and got.top_indices.shape == (2, 3, 4, 5)
    flat = token_scores(x.to(DEV), t.to(DEV), top_k=5, entropy=True)
    for a, b in zip(got, flat):
        assert torch.equal(a.reshape(b.shape), b)
    one = token_scores(x.to(DEV), t[:, 0].contiguous().to(DEV), top_k=5, entropy=True).log_probs
    assert one.shape == (24,) and torch.equal(one, flat.log_probs[:, 0])
    row = token_scores(x[0].to(DEV), top_k=5).top_indices  # a single row without a batch axis
    assert row.shape == (5,) and torch.equal(row, flat.top_indices[0])
    none = token_scores(x[:0].to(DEV).requires_grad_(True), t[:0].to(DEV), top_k=2, entropy=True)
    assert none.log_probs.shape == (0, 3) and none.entropy.shape == (0,) and none.top_indices.shape == (0, 2)
    none.log_probs.sum().backward()


def test_only_what_has_an_upstream_gradient_counts():
    x = _logits(8, 6, 300, torch.float32)
    xd = x.to(DEV).requires_grad_(True)
    t = _targets(8, 6, 300, 2)
    got = token_scores(xd, t.to(DEV), top_k=3, entropy=True)
    idx = got.top_indices.cpu().numpy()
    for which in range(3):
        o = (got.log_probs, got.entropy, got.top_log_probs)[which]
        u = torch.ones(o.shape)
        gx, = torch.autograd.grad([o], [xd], [u.to(DEV)], retain_graph=True)
        up = [None, None, None]
        up[which] = u.double().numpy()
        want, mag, coef = ro.scores_grad(x.double().numpy(), t.numpy(), idx, *up, 1.0)
        assert (np.abs(gx.double().cpu().numpy() - want) <= _bound("float32", want, mag, coef)).all()


def test_gradient_against_differences():
    x = _logits(5, 3, 41, torch.float64).to(DEV)
    t = _targets(5, 3, 41, 2).to(DEV)
    w = torch.tensor([0.7, -1.3], dtype=torch.float64, device=DEV)

    def value(y):
        s = token_scores(y, t, top_k=3, entropy=True, temperature=1.4)
        return (s.log_probs * w).sum() + 0.6 * s.entropy.sum() + (s.top_log_probs ** 2).sum()

    leaf = x.clone().requires_grad_(True)
    gx, = torch.autograd.grad(value(leaf), [leaf])
    h = 1e-5  # third derivatives of a few units: h^2 = 1e-10, rounding 1e-14 / h = 1e-9
    for r, j in [(0, 0), (0, 40), (1, int(t[1, 0])), (2, 17)]:
        up, down = x.clone(), x.clone()
        up[r, j] += h
        down[r, j] -= h
        assert abs(float((value(up) - value(down)) / (2 * h)) - float(gx[r, j])) < 1e-7


def test_captured_and_replayed_on_new_contents():
    x = torch.zeros(40, 1000, dtype=torch.bfloat16, device=DEV)
    t = torch.zeros(40, 2, dtype=torch.int32, device=DEV)
    x.copy_(_logits(1, 40, 1000, torch.bfloat16))
    side = torch.cuda.Stream(DEV)
    with torch.cuda.stream(side):
        token_scores(x, t, top_k=9, entropy=True)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = token_scores(x, t, top_k=9, entropy=True)
    for seed in (2, 3):
        new, nt = _logits(seed, 40, 1000, torch.bfloat16), _targets(seed, 40, 1000, 2)
        x.copy_(new)
        t.copy_(nt)
        graph.replay()
        torch.cuda.synchronize()
        _check(new, nt, 9, 1.0, got)


def test_results_repeat_bit_for_bit():
    x = _logits(11, 64, 4096, torch.bfloat16).to(DEV)
    x[:, ::2] = x[:, 1::2]
    a = token_scores(x, top_k=32, entropy=True)
    b = token_scores(x, top_k=32, entropy=True)
    for u, v in zip(a, b):
        assert u is None and v is None or torch.equal(u, v)


def test_rows_beyond_32_bit_offsets():
    """A matrix of more than 2^31 elements: its last rows against the oracle."""
    V, R = 32768, 65552
    x = torch.zeros(R, V, dtype=torch.float16, device=DEV)
    tail = _logits(6, 4, V, torch.float16)
    x[-4:] = tail.to(DEV)
    got = token_scores(x, top_k=3, entropy=True)
    last = type(got)(*(None if v is None else v[-4:] for v in got))
    _check(tail, None, 3, 1.0, last)
    assert got.top_indices[:-4].cpu().tolist() == [[0, 1, 2]] * (R - 4)


def test_not_differentiable_twice():
    x = _logits(9, 4, 60, torch.float32).to(DEV).requires_grad_(True)
    g, = torch.autograd.grad(token_scores(x, entropy=True).entropy.sum(), [x], create_graph=True)
    assert torch.isfinite(g).all()
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
