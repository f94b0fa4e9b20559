"""GPU tests of token_scores and distill_loss on rows with large finite values: masks of -1e9 to -1e30 in the place of
-inf, logits of 1e10, and values on both sides of the border between the two ways in which the kernels form their terms.
Loss and gradient, every type, rows in registers, a warp and a CTA a row, against the 64-bit oracle.

Tolerances: tests/rowops_bounds.py. A log-probability (x - max) / tau - ln s is off by the sum's error, by two roundings of
its own size (temperatures are powers of two, so 1 / tau is exact) and by logf's two steps of ln s <= ln V. An entropy
ln s - ln2 t / s carries the error of s and of t; t's terms are those of s times d. A divergence adds entries
q (ln q - ln p) of these and is rounded once. What lies below the smallest normal number is held to a fixed step: single
precision flushes a term there (2^-126), double rounds it by 2^-1075 at most, and either error is multiplied by the term's
coefficient. The oracle's coefficients allow for |ln p| of 100; a double's term that is not zero has 745 at most. The
oracle itself rounds g p by 2^-1075 before it multiplies by ln p + H and 1 / tau: 753 2^-1075 / tau."""
import math

import numpy as np
import pytest
import torch

from compactwarprnntloss_b200 import distill_loss, token_scores
from tests import rowops_bounds as rb
from tests import rowops_oracle as ro

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64}
MASKS = {"f32": [-1e7, -11629078.0, -1.2e7, -1e9, -1e10, -1e12, -1e30, 1e10], "bf16": [-1e7, -1e10, -1e30, 1e10],
         "f16": [-3e4, -65504.0, 6e4], "f64": [-1e10, -1e16, -1e20, -1e30, 1e20]}
ROWS = 9


def _rows(V, dtype, mask, seed=0):
    """[9, V]: the kinds of rows that a mask of that value leaves."""
    g = torch.Generator().manual_seed(seed + V)
    t = DT[dtype]
    x = (torch.randn(ROWS, V, generator=g, dtype=torch.float64) * 2.0).to(t)
    m = torch.tensor(mask, dtype=torch.float64).to(t)
    x[0] = m                                             # nothing but the mask
    keep = x[1, V // 2].clone()
    x[1] = m
    x[1, V // 2] = keep                                  # one token left
    alive = torch.randperm(V, generator=g)[:10]
    keep = x[2, alive].clone()
    x[2] = m
    x[2, alive] = keep                                   # ten
    x[3, torch.rand(V, generator=g) < 0.5] = m           # half of them
    step = torch.randint(0, 4, (V,), generator=g).double()
    x[4] = (m.double() * (1 + step * torch.finfo(t).eps)).to(t)  # values next to the mask's
    x[5, : V - V // 8] = m                               # what a warp or lane sees first is masked
    x[6] = m
    x[6, V // 3:] = float("-inf")                        # the mask beside -inf
    x[7, 1::2] = m
    x[7, 0::2] = m * 0.5                                 # two large values
    return x                                             # x[8]: an ordinary row


def _scores_check(x, targets, k, tau, got, up, gx):
    size, V = x.element_size(), x.size(1)
    x64, t = x.double().numpy(), targets.numpy()
    lps, ent, top, idx = ro.scores(x64, t, k, tau)
    err, unit = rb.sum_error(V, size), 2.0 ** -53 if size == 8 else 2.0 ** -24
    lse = err + 3 * unit * math.log(V)
    np.testing.assert_array_equal(got.top_indices.cpu().numpy(), idx)
    np.testing.assert_allclose(got.log_probs.detach().double().cpu().numpy(), lps, atol=lse, rtol=2 * unit)
    np.testing.assert_allclose(got.top_log_probs.detach().double().cpu().numpy(), top, atol=lse, rtol=2 * unit)
    off = np.abs(got.entropy.detach().double().cpu().numpy() - ent)
    assert (off <= 3 * err * (1 + math.log(V)) + 4 * unit * math.log(V)).all(), off
    want, mag, coef = ro.scores_grad(x64, t, idx, *(u.double().numpy() for u in up), tau)
    name = str(x.dtype).split(".")[1]
    bound = ro.HALF_STEP[name] * np.abs(want) + 2 * (err + rb.term_error(size)) * mag + ro.TINY[name]
    bound += 8 * 2.0 ** -1074 * coef + 377 * 2.0 ** -1074 / tau if size == 8 else ro.FLUSH32 * coef
    off = np.abs(gx.double().cpu().numpy() - want)
    assert (off <= bound).all(), [(r, (off - bound)[r].max()) for r in range(len(off)) if not (off <= bound)[r].all()]


def _distill_check(x, val, idx, tail, tau, rows, gx):
    size, V = x.element_size(), x.size(1)
    err, unit = rb.sum_error(V, size), 2.0 ** -53 if size == 8 else 2.0 ** -24
    loss, grad, lmag, gmag = ro.distill(x.double().numpy(), val.double().numpy(), idx.numpy(), None, tail, tau)
    got = rows.detach().double().cpu().numpy()
    fine = np.isfinite(loss)  # (a listed token that the student rules out: an infinite divergence)
    np.testing.assert_array_equal(got[~fine], loss[~fine])
    assert (np.abs(got - loss)[fine] <= ((2 * err + 2.0 ** -31) * lmag + unit * np.abs(loss))[fine]).all(), (got, loss)
    name = str(x.dtype).split(".")[1]
    bound = ro.HALF_STEP[name] * np.abs(grad) + 2 * (err + rb.term_error(size)) * gmag + ro.TINY[name]
    # what is flushed has a coefficient of Q <= 1 and, in the rest class, as much again, over tau
    bound += (2.0 ** -1073 if size == 8 else 2 * ro.FLUSH32) / tau
    off = np.abs(gx.double().cpu().numpy() - grad)
    assert (off <= bound).all(), [(r, (off - bound)[r].max()) for r in range(len(off)) if not (off <= bound)[r].all()]


def _times(t, n):
    """The rows over and over, n of them."""
    return t.repeat((n + t.size(0) - 1) // t.size(0), *([1] * (t.dim() - 1)))[:n].contiguous()


def _same_rows(full, n):
    """Repetitions at the same place between two 16-byte boundaries (every 8th at the latest) are the same, bit for bit;
    returns the first."""
    period = full[:8 * ROWS]
    want = period if n <= 8 * ROWS else _times(period, n)
    assert torch.equal(torch.isnan(full), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(full), torch.nan_to_num(want))
    return full[:ROWS]


# (V, type, rows): registers, a CTA a row, and with rows enough a warp a row, aligned and not
SHAPES = [(12, "f32", 9), (128, "f16", 9), (1000, "bf16", 9), (1031, "f32", 9), (300, "f64", 9), (9001, "f32", 9),
          (20000, "bf16", 9), (5000, "f16", 9), (3001, "f64", 9), (2500, "f32", 4741), (2501, "f32", 4741),
          (4096, "bf16", 4741), (4097, "f16", 4741)]


@pytest.mark.parametrize("V,dtype,n", SHAPES)
def test_scores_of_masked_rows(V, dtype, n):
    for mask in MASKS[dtype]:
        for tau in (1.0, 2.0 ** -7):
            x = _rows(V, dtype, mask)
            g = torch.Generator().manual_seed(1)
            t = torch.randint(0, V, (ROWS, 2), generator=g, dtype=torch.int32)
            t[:, 0] = V // 2
            ct = torch.float64 if dtype == "f64" else torch.float32
            up = [torch.randn(s, generator=g, dtype=ct) for s in ((ROWS, 2), (ROWS,), (ROWS, 4))]
            xd = _times(x, n).to(DEV).requires_grad_(True)
            got = token_scores(xd, _times(t, n).to(DEV), top_k=4, entropy=True, temperature=tau)
            gx, = torch.autograd.grad([got.log_probs, got.entropy, got.top_log_probs], [xd], [_times(u, n).to(DEV) for u in up])
            first = type(got)(*(_same_rows(v.detach(), n) for v in got))
            _scores_check(x, t, 4, tau, first, up, _same_rows(gx, n))


@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("V,dtype,n", SHAPES)
def test_divergences_of_masked_rows(V, dtype, n, tail):
    for mask in MASKS[dtype]:
        for tau in (1.0, 2.0 ** -7):
            x = _rows(V, dtype, mask)
            ct = torch.float64 if dtype == "f64" else torch.float32
            g = torch.Generator().manual_seed(2)
            idx = torch.stack([torch.randperm(V, generator=g)[:3] for _ in range(ROWS)]).to(torch.int32)
            idx[1, 0] = V // 2 if V // 2 not in idx[1].tolist() else idx[1, 0]
            # an ordinary row whose unlisted tokens are all masked
            keep = x[8, idx[8].long()].clone()
            x[8] = torch.tensor(mask, dtype=torch.float64).to(DT[dtype])
            x[8, idx[8].long()] = keep
            val = torch.log(torch.tensor([[0.5, 0.3, 0.1]] * ROWS, dtype=ct))
            xd = _times(x, n).to(DEV).requires_grad_(True)
            args = (_times(val, n).to(DEV), _times(idx, n).to(DEV))
            rows = distill_loss(xd, *args, tail=tail, temperature=tau, reduction="none")
            gx, = torch.autograd.grad([rows], [xd], [torch.ones_like(rows)])
            _distill_check(x, val, idx, tail, tau, _same_rows(rows.detach(), n), _same_rows(gx, n))
            assert not bool(torch.isnan(distill_loss(xd.detach(), *args, tail=tail, temperature=tau)))
