"""GPU tests of distill_loss with values that a diverged teacher hands over: NaN and +inf. The row's loss and gradient are
NaN, those of the other rows are untouched bit for bit, and an unused slot's value is never looked at."""
import pytest
import torch

from compactwarprnntloss_b200 import distill_loss

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64}


def _call(x, val, idx, weight, tail, reduction="none"):
    leaf = x.clone().requires_grad_(True)
    out = distill_loss(leaf, val, idx, weight=weight, tail=tail, reduction=reduction)
    gx, = torch.autograd.grad([out], [leaf], [torch.ones_like(out)])
    return out.detach(), gx


@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("K", [1, 3, 16, 32])
# registers, a CTA a row, a warp a row
@pytest.mark.parametrize("V,dtype,n", [(40, "f16", 12), (300, "f32", 12), (1024, "bf16", 12), (100, "f64", 12),
                                       (9000, "f32", 12), (4000, "f64", 12), (3000, "f32", 4740)])
def test_a_nan_in_the_teacher_is_a_nan_in_its_row(V, dtype, n, K, tail):
    g = torch.Generator().manual_seed(V + K)
    ct = torch.float64 if dtype == "f64" else torch.float32
    x = torch.randn(n, V, generator=g).to(DT[dtype]).to(DEV)
    idx = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(12)]).repeat(n // 12, 1).int().to(DEV)
    val = torch.log_softmax(torch.randn(n, K + 1, generator=g, dtype=ct), 1)[:, :K].contiguous().to(DEV)
    weight = torch.ones(n, dtype=ct, device=DEV)
    weight[5] = 0.0
    x[8] = float("-inf")
    clean, clean_g = _call(x, val, idx, weight, tail)
    assert bool(torch.isfinite(clean).all())
    nan = float("nan")
    val[0, 0] = nan
    val[1, K - 1] = nan
    val[2] = nan
    val[5, 0] = nan                        # a row of weight 0 is not read
    val[6, 0], idx[6, 0] = nan, -1         # a slot that is not used
    val[8, 0] = nan                        # the student has nothing: NaN all the same
    val[9, K // 2] = float("inf")
    rows, gx = _call(x, val, idx, weight, tail)
    bad = [0, 1, 2, 8] + ([] if tail else [9])
    keep = [r for r in range(n) if r not in (0, 1, 2, 6, 8, 9)]
    assert bool(torch.isnan(rows[bad]).all()) and bool(torch.isnan(gx[bad]).all())
    assert torch.equal(rows[keep], clean[keep]) and torch.equal(gx[keep], clean_g[keep])
    assert bool(torch.isfinite(rows[6])) and bool(torch.isfinite(gx[6]).all())
    assert not bool(torch.isfinite(rows[9]))
    total, _ = _call(x, val, idx, weight, tail, "mean")
    assert bool(torch.isnan(total))
