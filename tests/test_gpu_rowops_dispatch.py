"""GPU tests of token_scores and distill_loss with batches so large that other kernels take them than a few rows get: a warp a
row, runs of rows, shared memory beyond its default. Every row, last runs that are not full among them, against the same
definitions in 64 bits of torch on the same GPU. Tolerances: tests/rowops_bounds.py; a float log-probability
(x - max) / tau - ln s takes two roundings of its own and logf's, a divergence's steps are double (2^-33) and it is rounded once."""
import math

import pytest
import torch

from compactwarprnntloss_b200 import distill_loss, token_scores
from tests import rowops_bounds as rb
from tests import rowops_oracle as ro

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64}

# rows, V, type, entries: a warp a row from 148 * 32 rows on (aligned, not, the shortest and the longest of them); runs of rows
# from 148 * 32 * (256 / lanes) on, for 32, 16, 8 and 4 lanes a row
LARGE = [(4739, 4096, "bf16", 5), (4739, 2500, "f32", 32), (4741, 2501, "f32", 3), (4737, 2057, "f16", 1),
         (4736 + 5, 16377, "f16", 16), (4739, 700, "f64", 4),
         (37894, 60, "f16", 32), (37893, 97, "f32", 32), (37891, 300, "bf16", 20), (37890, 33, "f64", 5),
         (75781, 80, "bf16", 16), (75779, 51, "f32", 9), (151557, 64, "f16", 8), (151555, 43, "f32", 7),
         (303109, 24, "f32", 2), (303111, 37, "bf16", 4)]


def _rows(seed, n, V, dtype):
    g = torch.Generator(DEV).manual_seed(seed)
    x = torch.randn(n, V, generator=g, device=DEV) * 2.0
    x[torch.rand(n, V, generator=g, device=DEV) < 0.02] = float("-inf")
    x[n // 2] = float("-inf")
    return x.to(DT[dtype]), g


def _within(name, got, want, bound):
    off = (got.double() - want).abs()
    ok = (off <= bound) | (got.double() == want)
    assert bool(ok.all()), (name, int((~ok).sum()), (~ok).nonzero()[:3].tolist())


@pytest.mark.parametrize("n,V,dtype,k", LARGE)
def test_scores_of_large_batches(n, V, dtype, k):
    x, g = _rows(n, n, V, dtype)
    size, ct = x.element_size(), torch.float64 if dtype == "f64" else torch.float32
    t = torch.randint(0, V, (n, 2), generator=g, device=DEV, dtype=torch.int32)
    t[::5, 1] = -1
    leaf = x.clone().requires_grad_(True)
    s = token_scores(leaf, t, top_k=min(k, V), entropy=True)
    outs = (s.log_probs, s.entropy, s.top_log_probs)
    up = [torch.randn(o.shape, generator=g, device=DEV, dtype=ct) for o in outs]
    gx, = torch.autograd.grad(outs, [leaf], up)

    empty = (x == float("-inf")).all(1)
    z = x.double()
    lp = torch.log_softmax(z, 1)
    lp[empty] = float("-inf")
    p = lp.exp()
    first = torch.sort(z, dim=1, descending=True, stable=True)[1][:, :min(k, V)]
    lse = rb.sum_error(V, size) + 3 * (2.0 ** -53 if size == 8 else 2.0 ** -24) * math.log(V)
    unit = 2.0 ** -53 if size == 8 else 2.0 ** -24
    at = t.clamp(min=0).long()
    want = torch.where(t >= 0, lp.gather(1, at), 0.0)
    _within("log_probs", s.log_probs.detach(), want, lse + 2 * unit * want.abs().nan_to_num(posinf=0.0))
    assert torch.equal(s.top_indices.long(), first)
    want = lp.gather(1, first)
    _within("top", s.top_log_probs.detach(), want, lse + 2 * unit * want.abs().nan_to_num(posinf=0.0))
    seen = lp.masked_fill(p == 0, 0.0)
    ent = -(p * seen).sum(1)
    _within("entropy", s.entropy.detach(), ent, 3 * rb.sum_error(V, size) * (1 + math.log(V)) + 4 * unit * math.log(V))

    u_lp = torch.where(t >= 0, up[0].double(), 0.0)
    total, mass = u_lp.sum(1) + up[2].double().sum(1), u_lp.abs().sum(1) + up[2].double().abs().sum(1)
    want, mag = torch.zeros_like(z), torch.zeros_like(z)
    want.scatter_add_(1, at, u_lp).scatter_add_(1, first, up[2].double())
    mag.scatter_add_(1, at, u_lp.abs()).scatter_add_(1, first, up[2].double().abs())
    ge = up[1].double()[:, None]
    want -= p * (total[:, None] + ge * (seen + ent[:, None]))
    mag += p * (mass[:, None] + ge.abs() * (seen.abs() + ent[:, None]))
    want[empty], mag[empty] = 0.0, 0.0
    name = str(DT[dtype]).split(".")[1]
    bound = ro.HALF_STEP[name] * want.abs() + 2 * (rb.sum_error(V, size) + rb.term_error(size)) * mag + ro.TINY[name]
    _within("gradient", gx, want, bound + ro.FLUSH32 * (mass[:, None] + 200 * ge.abs()))


@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("n,V,dtype,k", LARGE)
def test_divergences_of_large_batches(n, V, dtype, k, tail):
    x, g = _rows(n + 1, n, V, dtype)
    size, ct = x.element_size(), torch.float64 if dtype == "f64" else torch.float32
    k = min(k, V)
    near = x.double().clamp(min=-30.0) + 0.7 * torch.randn(n, V, generator=g, device=DEV, dtype=torch.float64)
    val, idx = torch.log_softmax(near, 1).topk(k, 1)
    val, idx = val.to(ct), idx.int()
    if k > 2:
        idx[::7, 2] = -1
    weight = torch.rand(n, generator=g, device=DEV, dtype=ct)
    weight[::6] = 0.0
    leaf = x.clone().requires_grad_(True)
    rows = distill_loss(leaf, val, idx, weight=weight, tail=tail, reduction="none")
    gx, = torch.autograd.grad([rows], [leaf], [torch.ones_like(rows)])
    total = distill_loss(x, val, idx, weight=weight, tail=tail, reduction="sum")

    empty = (x == float("-inf")).all(1)
    z = x.double()
    lp = torch.log_softmax(z, 1)
    p = lp.exp()
    used = idx >= 0
    at = idx.clamp(min=0).long()
    a = torch.where(used, val.double(), float("-inf"))
    lq = a if tail else torch.log_softmax(a, 1)
    q = lq.exp()
    picked = lp.gather(1, at)
    each = torch.where(q > 0, q * (lq - picked), 0.0)
    emag = torch.where(q > 0, q * (lq.abs() + picked.abs() + 1.0), 0.0)
    D, mag = each.sum(1), emag.sum(1)
    Q = q.sum(1)
    grad, gmag = torch.zeros_like(z), torch.zeros_like(z)
    grad.scatter_add_(1, at, -q)
    gmag.scatter_add_(1, at, q)
    if tail:
        listed = torch.zeros_like(z, dtype=torch.int32).scatter_add_(1, at, used.int()) > 0
        other = torch.where(listed, float("-inf"), lp)
        some = (other > float("-inf")).any(1)
        left = torch.where(some, (1.0 - Q).clamp(min=0.0), 0.0)
        lr = torch.where(some, torch.logsumexp(other, 1), 0.0)
        D = D + torch.where(left > 0, left * (left.log() - lr), 0.0)
        mag = mag + torch.where(left > 0, left * (left.log().abs() + lr.abs() + 1.0), 0.0)
        Q = Q + left
        rest = torch.where(some[:, None], left[:, None] * (other - lr[:, None]).exp(), 0.0)
        grad -= rest
        gmag += rest
    grad += Q[:, None] * p
    gmag += Q[:, None] * p
    w = weight.double()
    D, mag, grad, gmag = w * D, w * mag, w[:, None] * grad, w[:, None] * gmag
    out = empty | (weight == 0)
    D[out], mag[out], grad[out], gmag[out] = 0.0, 0.0, 0.0, 0.0
    unit = 2.0 ** -53 if size == 8 else 2.0 ** -24
    infinite = torch.isinf(D)  # a listed token that the student rules out
    loss_bound = ((2 * rb.sum_error(V, size) + 2.0 ** -31) * mag + unit * D.abs()).masked_fill(infinite, 0.0)
    _within("row losses", rows.detach(), D, loss_bound)
    if not bool(infinite.any()):
        assert abs(float(total) - float(D.sum())) <= float(loss_bound.sum()) + unit * abs(float(D.sum()))
    name = str(DT[dtype]).split(".")[1]
    bound = ro.HALF_STEP[name] * grad.abs() + 2 * (rb.sum_error(V, size) + rb.term_error(size)) * gmag + ro.TINY[name]
    _within("gradient", gx, grad, bound + 2 * ro.FLUSH32)


# ------------------------------------------------------------------------------------ sums that are exact

@pytest.mark.parametrize("n,V,dtype", [(9, 100, "f32"), (9, 128, "f16"), (9, 1024, "bf16"), (9, 2048, "f16"), (9, 5001, "f32"),
                                       (9, 30000, "bf16"), (4739, 2501, "f32"), (4739, 4096, "bf16"), (37894, 60, "f16")])
def test_sums_of_powers_of_two(n, V, dtype):
    """At the temperature 1 / ln 2 whole logits have powers of two for terms, and their sums fit 24 bits: what is left are ex2
    (2^-22 for a term, and as much for each of the eight raises to a new maximum and for the undone shift), logf (2^-23 of
    ln s) and the last roundings. A thirtieth of what rows of any values may be off by."""
    g = torch.Generator(DEV).manual_seed(V)
    x = torch.randint(-8, 1, (n, V), generator=g, device=DEV).double()
    x[0] = 0.0
    x[1, 1:] = float("-inf")
    x[2] -= 40.0
    x = x.to(DT[dtype])
    tau = 1.4426950408889634
    t = torch.randint(0, V, (n, 2), generator=g, device=DEV, dtype=torch.int32)
    s = token_scores(x, t, top_k=3, entropy=True, temperature=tau)
    lp = torch.log_softmax(x.double() / tau, 1)
    ex2, unit = 10 * 2.0 ** -22, 2.0 ** -24
    want = lp.gather(1, t.long())
    _within("log_probs", s.log_probs, want, ex2 + 2 * unit * math.log(V) + 4 * unit * want.abs().nan_to_num(posinf=0.0))
    p = lp.exp()
    ent = -(p * lp.masked_fill(p == 0, 0.0)).sum(1)
    _within("entropy", s.entropy, ent, 2 * ex2 * (1 + math.log(V)) + 4 * unit * math.log(V))
    idx = torch.stack([torch.zeros(n, device=DEV), torch.full((n,), V - 1.0, device=DEV)], 1).int()
    val = torch.log(torch.tensor([[0.25, 0.125]] * n, device=DEV))
    rows = distill_loss(x, val, idx, tail=False, temperature=tau, reduction="none")
    q = torch.softmax(val.double() / tau, 1)
    each = q * (q.log() - lp.gather(1, idx.long()))
    want = each.sum(1)
    _within("divergence", rows, want, ex2 + 2.0 ** -30 * each.abs().sum(1).nan_to_num(posinf=0.0) + unit * want.abs().nan_to_num(posinf=0.0))
