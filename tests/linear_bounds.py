"""Cases of a linear layer and 64-bit gradients with error bounds that one lost part of dz, a lost block of rows or a wrong
epilogue does not pass.

Products: tests/test_gpu_linear.py, (n/16 + 8) 2^-21 of the sum of the absolute products for n of them. dz = dy act'(z) goes
into its products in two parts: float16 loses 2^-22 of it or 2^-36 where that is less, bfloat16 2^-16 (relu's dz is dy or
zero: nothing). z's error moves the slope by less than itself; the slope is put together from ex2, rcp (2^-22 each, the
exponent's roundings as much for each unit of z) and a few roundings: tanh s (1 + |z| / 4) 2^-20, silu, whose 1 - s is a
difference, sigma (2 + |z|) (1 + |z| / 8) 2^-20. A column sum adds, one after the other, at most 64 of a piece of 32 rows in
two parts, or a 2048th of the rows and both parts (two times 5 at 20 000); 5 pieces, 16 and 8 joined sums: below 140."""
import numpy as np
import torch

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}
TWO_PARTS = {"f16": (2.0 ** -22, 2.0 ** -36), "bf16": (2.0 ** -16, 2.0 ** -133)}


def case(seed, M, N, K, dtype, x_scale=1.0, w_scale=1.0, dy_scale=1.0, residual=True):
    """x, weight, bias, residual, dy on the CPU; z of the order of x_scale * w_scale."""
    g = torch.Generator().manual_seed(seed)
    make = lambda shape, scale: (torch.randn(shape, generator=g, dtype=torch.float64) * scale).to(DT[dtype])
    return (make((M, K), x_scale), make((N, K), w_scale * K ** -0.5), make((N,), x_scale * w_scale),
            make((M, N), 1.0) if residual else None, make((M, N), dy_scale))


def _err(n):
    return (n / 16 + 8) * 2.0 ** -21


def _f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _activate(act, z):
    """act(z), its slope, the slope's error"""
    if act == "relu":
        return np.maximum(z, 0), (z > 0).astype(np.float64), np.zeros_like(z)
    if act == "tanh":
        s = 1 / np.cosh(np.minimum(np.abs(z), 300)) ** 2
        return np.tanh(z), s, s * (1 + np.abs(z) / 4) * 2.0 ** -20
    if act == "silu":
        s = 1 / (1 + np.exp(-z))
        return z * s, s * (1 + z * (1 - s)), s * (2 + np.abs(z)) * (1 + np.abs(z) / 8) * 2.0 ** -20
    return z, np.ones_like(z), np.zeros_like(z)


def expect(x, w, b, r, dy, act, dtype):
    """{name: (value, bound)} of y, dx, dw, db."""
    x, w, b, r, dy = map(_f64, (x, w, b, r, dy))
    (M, K), N = x.shape, w.shape[0]
    eps, tiny = EPS[dtype], TINY[dtype]
    ax, aw = np.abs(x), np.abs(w)
    z = x @ w.T + (0 if b is None else b)
    zerr = _err(K) * (ax @ aw.T + (0 if b is None else np.abs(b)))
    a, s, serr = _activate(act, z)
    y = a + (0 if r is None else r)
    dz = dy * s
    delta, parts = np.zeros_like(dz), 1
    if act not in (None, "none"):
        delta = np.abs(dy) * (zerr + serr)
    if act in ("tanh", "silu"):
        rel, least = TWO_PARTS[dtype]
        delta, parts = delta + rel * np.abs(dz) + least, 2
    if act == "relu":
        delta = np.abs(dy) * (np.abs(z) <= zerr)
    adz = np.abs(dz)
    out = {"y": (y, eps * np.abs(y) + 1.1 * zerr + 2.0 ** -20 * (np.abs(a) + np.abs(y)) + tiny)}
    want = dz @ w
    out["dx"] = (want, eps * np.abs(want) + 1.01 * (delta @ aw + _err(parts * N) * (adz @ aw)) + tiny)
    want = dz.T @ x
    out["dw"] = (want, eps * np.abs(want) + 1.01 * (delta.T @ ax + _err(parts * M) * (adz.T @ ax)) + tiny)
    want = dz.sum(0)
    out["db"] = (want, eps * np.abs(want) + 1.01 * (delta.sum(0) + 140 * 2.0 ** -24 * adz.sum(0)) + tiny)
    return out, dz


def outside(got, value_bound):
    """How many elements of `got` lie outside."""
    value, bound = value_bound
    return int((~(np.abs(_f64(got) - value) <= bound)).sum())


# the second part of dz counts in these: (M, N, K, dtype, scales of x, weight and dy)
TWO_PART_CASES = [(M, N, K, dtype) + scales
                  for M, N, K in ((260, 256, 32), (1000, 328, 16), (333, 200, 40), (9001, 130, 40), (12, 96, 32))
                  for dtype, scales in (("bf16", (1.0, 1.0, 1.0)), ("bf16", (1.0, 1.0, 1e-6)), ("f16", (1.0, 1.0, 1.0)),
                                        ("f16", (2.0 ** -6, 2.0 ** 6, 2.0 ** -15)), ("f16", (2.0 ** 7, 2.0 ** -7, 2.0 ** -15)))]
