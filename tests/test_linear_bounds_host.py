"""CPU checks of the bounds that the linear layers' gradients are tested with: 64-bit products of a dz that keeps both of its
parts pass, of a dz rounded once do not, and neither does a column sum that lacks a block of rows."""
import numpy as np
import pytest
import torch

from tests import linear_bounds as lb


def _rounded(v, dtype):
    return torch.from_numpy(v).to(lb.DT[dtype]).double().numpy()


@pytest.mark.parametrize("act", ["tanh", "silu"])
@pytest.mark.parametrize("M,N,K,dtype,xs,ws,ds", lb.TWO_PART_CASES)
def test_the_bounds_tell_one_part_from_two(M, N, K, dtype, xs, ws, ds, act):
    x, w, b, r, dy = lb.case(M + N, M, N, K, dtype, xs, ws, ds)
    want, dz = lb.expect(x, w, b, r, dy, act, dtype)
    x64, w64 = x.double().numpy(), w.double().numpy()
    high = _rounded(dz, dtype)
    shift = 2.0 ** 11 if dtype == "f16" else 1.0
    both = high + _rounded((dz - high) * shift, dtype) / shift
    bad = {}
    for name, part in (("both", both), ("high", high)):
        got = {"dx": _rounded(part @ w64, dtype), "dw": _rounded(part.T @ x64, dtype), "db": _rounded(part.sum(0), dtype)}
        bad[name] = sum(lb.outside(torch.from_numpy(v), want[k]) for k, v in got.items())
    assert bad["both"] == 0
    assert bad["high"] > 0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("act", [None, "silu"])
def test_the_bounds_miss_no_block_of_rows(act, dtype):
    M, N, K = 20000, 64, 24
    x, w, b, r, dy = lb.case(5, M, N, K, dtype)
    want, dz = lb.expect(x, w, b, r, dy, act, dtype)
    assert lb.outside(torch.from_numpy(_rounded(dz.sum(0), dtype)), want["db"]) == 0
    for first in (0, 6400, 19968):
        part = dz.copy()
        part[first:first + 32] = 0.0
        assert lb.outside(torch.from_numpy(_rounded(part.sum(0), dtype)), want["db"]) > 0
