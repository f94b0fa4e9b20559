"""GPU tests of fused_linear's gradients against bounds that a lost second part of dz or a lost block of rows does not pass
(tests/linear_bounds.py; tests/test_linear_bounds_host.py shows it), and of the epilogues that small and split products
take: few rows, and parts that are joined, with every activation."""
import pytest
import torch

from compactwarprnntloss_b200 import fused_linear
from tests import linear_bounds as lb

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _check(x, w, b, r, dy, act, dtype):
    leaves = [None if t is None else t.to(DEV).requires_grad_(True) for t in (x, w, b, r)]
    y = fused_linear(*leaves, activation=act)
    some = [t for t in leaves if t is not None]
    got = iter(torch.autograd.grad([y], some, [dy.to(DEV)]))
    dx, dw, db, dr = [None if t is None else next(got) for t in leaves]
    want, _ = lb.expect(x, w, b, r, dy, act, dtype)
    for name, v in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        if v is not None:
            assert lb.outside(v, want[name]) == 0, name
    if r is not None:
        assert torch.equal(dr.cpu(), dy)
    # each gradient by itself, from the same kernels
    for i, (leaf, alone) in enumerate(zip(leaves[:3], (dx, dw, db))):
        if leaf is None:
            continue
        one = [None if t is None else t.detach().requires_grad_(t is leaf) for t in leaves]
        again, = torch.autograd.grad([fused_linear(*one, activation=act)], [one[i]], [dy.to(DEV)])
        assert torch.equal(again, alone)


@pytest.mark.parametrize("act", ["tanh", "silu"])
@pytest.mark.parametrize("M,N,K,dtype,xs,ws,ds", lb.TWO_PART_CASES)
def test_both_parts_of_dz_count(M, N, K, dtype, xs, ws, ds, act):
    _check(*lb.case(M + N, M, N, K, dtype, xs, ws, ds), act, dtype)


@pytest.mark.parametrize("act", [None, "relu", "tanh", "silu"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M", [1, 3, 8, 9, 16])
def test_few_rows(M, dtype, act):
    for N, K in ((64, 128), (41, 67), (8, 2000), (2000, 9), (1024, 640)):
        _check(*lb.case(M + N, M, N, K, dtype), act, dtype)
    _check(*lb.case(M, M, 96, 80, dtype, 2.0 ** -6, 2.0 ** 6, 2.0 ** -15, residual=False), act, dtype)


@pytest.mark.parametrize("act", [None, "relu", "tanh", "silu"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
# z from parts, aligned and not; dx from parts (a long row of dz); dw from parts (many rows), the first ones of dz's low part
# only; one of more columns than a tile has
@pytest.mark.parametrize("M,N,K", [(100, 96, 9000), (60, 33, 2100), (64, 5000, 40), (30, 4003, 24), (9001, 130, 40),
                                   (20000, 64, 72), (150, 300, 2300)])
def test_parts_of_long_sums(M, N, K, dtype, act):
    _check(*lb.case(M + K, M, N, K, dtype), act, dtype)
    if act in ("tanh", "silu"):
        _check(*lb.case(M + K, M, N, K, dtype, 2.0 ** -6, 2.0 ** 6, 2.0 ** -15, residual=False), act, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("act", [None, "relu", "silu"])
def test_sums_over_rows_in_every_order(dtype, act):
    """Column sums by pieces of 32 rows, folded and joined, and by runs of rows."""
    for M, N, K in ((20000, 64, 24), (40009, 40, 16), (8193, 300, 16), (5000, 257, 9)):
        _check(*lb.case(M, M, N, K, dtype, residual=False), act, dtype)


@pytest.mark.parametrize("dtype,scales", [("bf16", (1.0, 1.0, 1.0)), ("f16", (1.0, 1.0, 1.0)),
                                          ("f16", (2.0 ** -6, 2.0 ** 6, 2.0 ** -15))])
def test_tiles_that_two_ctas_share(dtype, scales):
    """All three gradient products by tiles of 256 x 256, dW's in parts."""
    _check(*lb.case(1, 19001, 640, 512, dtype, *scales), "tanh", dtype)
