"""GPU tests of fused_linear against 64-bit products: sizes on both sides of every tile and split, types, strides,
activations, residuals, gradients, graphs and the joint's whole chain.

Tolerances. A tensor-core sum of `n` products adds groups of 16 to a float: each of the n/16 additions, and the
alignment inside a group, loses at most 2^-21 of the sum of the absolute products (one unit of the last place of a float
and as much for the truncated low bits), a few more for joining parts and the bias: err(n) = (n/16 + 8) 2^-21 of that
magnitude. Activations are good to 2^-20. Every output is rounded to its type once; dz is rounded before the two
products it goes into (the tensor cores take it in that type, at best in two parts), which their bounds carry entry by
entry. act' is
Lipschitz with a constant below 1 (tanh: 0.77, silu: 0.5); relu's jumps where z is within its error of zero."""
import ctypes

import numpy as np
import pytest
import torch

from compactwarprnntloss_b200 import capi, compact_joint, fused_linear, transducer_loss
from tests import rowops_oracle as ro

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DT = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}


def _rand(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale).to(DT[dtype])


def _case(seed, M, N, K, dtype, bias=True, residual=True):
    g = torch.Generator().manual_seed(seed)
    return (_rand(g, (M, K), dtype), _rand(g, (N, K), dtype, K ** -0.5), _rand(g, (N,), dtype) if bias else None,
            _rand(g, (M, N), dtype) if residual else None, _rand(g, (M, N), dtype))


def _err(n):
    return (n / 16 + 8) * 2.0 ** -21


def _act(name, z):
    if name == "relu":
        return np.maximum(z, 0), (z > 0).astype(np.float64)
    if name == "tanh":
        return np.tanh(z), 1 / np.cosh(z) ** 2
    if name == "silu":
        s = 1 / (1 + np.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    return z, np.ones_like(z)


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _check(x, w, b, r, dy, act, dtype, y, grads):
    """CPU tensors in; device results `y` and (dx, dw, db, dr), each None where not asked for."""
    x, w, b, r, dy = map(_np, (x, w, b, r, dy))
    eps, tiny = EPS[dtype], TINY[dtype]
    (M, K), N = x.shape, w.shape[0]
    z = x @ w.T + (0 if b is None else b)
    zerr = _err(K) * (np.abs(x) @ np.abs(w).T + (0 if b is None else np.abs(b)))
    a, s = _act(act, z)
    want = a + (0 if r is None else r)
    off = np.abs(_np(y) - want)
    bound = eps * np.abs(want) + 1.1 * zerr + 2.0 ** -20 * (np.abs(a) + np.abs(want)) + tiny
    assert (off <= bound).all(), ("y", (off - bound).max())
    if grads is None:
        return
    dx, dw, db, dr = grads
    dz = dy * s
    delta = np.zeros_like(dz)
    if act not in (None, "none"):
        delta = eps * np.abs(dz) + np.abs(dy) * (zerr + 2.0 ** -20 * np.abs(s)) + tiny
        if act == "relu":
            delta += np.abs(dy) * (np.abs(z) <= zerr)
    if dx is not None:
        want = dz @ w
        bound = eps * np.abs(want) + (1 + eps) * (delta @ np.abs(w)) + _err(N) * (np.abs(dz) @ np.abs(w)) * 1.01 + tiny
        off = np.abs(_np(dx) - want)
        assert (off <= bound).all(), ("dx", (off - bound).max())
    if dw is not None:
        want = dz.T @ x
        bound = eps * np.abs(want) + (1 + eps) * (delta.T @ np.abs(x)) + _err(M) * (np.abs(dz).T @ np.abs(x)) * 1.01 + tiny
        off = np.abs(_np(dw) - want)
        assert (off <= bound).all(), ("dw", (off - bound).max())
    if db is not None:
        want = dz.sum(0)
        bound = eps * np.abs(want) + (1 + eps) * delta.sum(0) + 1.01 * M * 2.0 ** -24 * np.abs(dz).sum(0) + tiny
        off = np.abs(_np(db) - want)
        assert (off <= bound).all(), ("db", (off - bound).max())
    if dr is not None:
        np.testing.assert_array_equal(_np(dr), dy)


def _run(x, w, b, r, dy, act, dtype):
    leaves = [None if t is None else t.to(DEV).requires_grad_(True) for t in (x, w, b, r)]
    y = fused_linear(leaves[0], leaves[1], leaves[2], leaves[3], activation=act)
    assert y.dtype == DT[dtype] and y.shape == dy.shape
    some = [t for t in leaves if t is not None]
    got = iter(torch.autograd.grad([y], some, [dy.to(DEV)]))
    grads = [None if t is None else next(got) for t in leaves]
    _check(x, w, b, r, dy, act, dtype, y, grads)
    with torch.no_grad():
        assert torch.equal(fused_linear(*leaves, activation=act), y)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(128, 256, 64), (128, 32, 64), (1, 1, 1), (1, 8, 8), (8, 1024, 640), (2, 7, 3),
                                   (127, 33, 65), (129, 64, 63), (128, 128, 128), (300, 200, 72), (257, 264, 100),
                                   (1000, 640, 512), (513, 1001, 641), (640, 96, 1000), (50, 8, 2000), (3, 2000, 9)])
def test_every_size(M, N, K, dtype):
    _run(*_case(M + N + K, M, N, K, dtype), None, dtype)


@pytest.mark.parametrize("act", ["relu", "tanh", "silu"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(130, 256, 64), (77, 40, 96), (260, 129, 31)])
def test_activations(act, M, N, K, dtype):
    x, w, b, r, dy = _case(M, M, N, K, dtype)
    x[0] *= 30.0   # far out, where tanh is flat
    x[1] *= 1e-3   # where it is the identity
    _run(x, w, b, r, dy, act, dtype)
    _run(x, w, None, None, dy, act, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(20000, 64, 72), (9001, 130, 40), (4100, 640, 512), (100, 96, 9000), (1, 40, 16000)])
def test_long_sums_are_split_and_joined(M, N, K, dtype):
    """Sums over many rows (the weight's gradient) or a long input, in parts."""
    _run(*_case(M + K, M, N, K, dtype), "tanh" if K < 1000 else None, dtype)


def test_many_tiles_of_every_width():
    """More tiles than SMs, so that every CTA carries several: both halves of TMEM, all phases of the ring."""
    for N, K in ((512, 640), (128, 200), (64, 64), (32, 1024), (24, 8)):
        M = 148 * 128 * 5 + 37
        g = torch.Generator(DEV).manual_seed(N)
        x = torch.randn(M, K, generator=g, device=DEV).bfloat16()
        w = (torch.randn(N, K, generator=g, device=DEV) * K ** -0.5).bfloat16()
        y = fused_linear(x, w)
        want = x.double() @ w.double().t()
        bound = 2.0 ** -8 * want.abs() + _err(K) * (x.double().abs() @ w.double().abs().t()) + 2.0 ** -134
        assert bool(((y.double() - want).abs() <= bound).all()), (N, K)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_strided_and_misaligned_matrices(dtype):
    M, N, K = 200, 72, 80
    x, w, b, r, dy = _case(3, M, N, K, dtype)
    for x_room, x_at, w_room, w_at in ((16, 8, 8, 0), (24, 3, 5, 5), (1, 0, 1, 1), (0, 0, 0, 0)):
        xw = torch.zeros(M, K + x_room, dtype=DT[dtype], device=DEV)
        ww = torch.zeros(N, K + w_room, dtype=DT[dtype], device=DEV)
        xv, wv = xw[:, x_at:x_at + K], ww[:, w_at:w_at + K]
        xv.copy_(x), wv.copy_(w)
        leaves = [xv.detach().requires_grad_(True), wv.detach().requires_grad_(True),
                  b.to(DEV).requires_grad_(True), r.to(DEV).requires_grad_(True)]
        y = fused_linear(*leaves, activation="silu")
        _check(x, w, b, r, dy, "silu", dtype, y, torch.autograd.grad([y], leaves, [dy.to(DEV)]))
    # a transposed weight, an upstream gradient with its own strides, one row for all
    wt = w.t().contiguous().to(DEV).t().requires_grad_(True)
    xl = x.to(DEV).requires_grad_(True)
    y = fused_linear(xl, wt, b.to(DEV))
    wide = torch.zeros(M, N + 9, dtype=DT[dtype], device=DEV)
    wide[:, 1:1 + N] = dy.to(DEV)
    dx, dw = torch.autograd.grad([y], [xl, wt], [wide[:, 1:1 + N]], retain_graph=True)
    _check(x, w, b, None, dy, None, dtype, y, (dx, dw, None, None))
    dx, = torch.autograd.grad([y], [xl], [dy[:1].to(DEV).expand(M, N)], retain_graph=True)
    _check(x, w, b, None, dy[:1].expand(M, N).contiguous(), None, dtype, y, (dx, None, None, None))
    (y.float().sum() * 2).backward()  # an expanded scalar from autograd itself
    _check(x, w, b, None, torch.full((M, N), 2.0), None, dtype, y, (xl.grad, wt.grad, None, None))


def test_leading_axes_and_empty_batches():
    x, w, b, r, dy = _case(5, 24, 40, 16, "bf16")
    a = fused_linear(x.view(2, 3, 4, 16).to(DEV), w.to(DEV), b.to(DEV), r.view(2, 3, 4, 40).to(DEV))
    assert a.shape == (2, 3, 4, 40)
    assert torch.equal(a.view(24, 40), fused_linear(x.to(DEV), w.to(DEV), b.to(DEV), r.to(DEV)))
    assert fused_linear(x[0].to(DEV), w.to(DEV)).shape == (40,)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x[:0], w, b)]
    y = fused_linear(*leaves, activation="tanh")
    assert y.shape == (0, 40)
    y.sum().backward()
    assert leaves[0].grad.shape == (0, 16) and not leaves[1].grad.any() and not leaves[2].grad.any()


def test_only_the_gradients_asked_for():
    x, w, b, r, dy = _case(6, 150, 48, 56, "bf16")
    for which in range(4):
        leaves = [t.to(DEV).requires_grad_(i == which) for i, t in enumerate((x, w, b, r))]
        y = fused_linear(*leaves, activation="tanh")
        got = [None] * 4
        got[which], = torch.autograd.grad([y], [leaves[which]], [dy.to(DEV)])
        _check(x, w, b, r, dy, "tanh", "bf16", y, got)


def test_infinities_and_nan_stay_in_their_rows():
    x, w, b, r, dy = _case(7, 140, 64, 64, "bf16")
    x[3, 5], x[130, 0] = float("inf"), float("nan")
    y = fused_linear(x.to(DEV), w.to(DEV), b.to(DEV))
    bad = ~torch.isfinite(y)
    assert bad[3].all() and bad[130].all() and not bad[[i for i in range(140) if i not in (3, 130)]].any()
    for act in ("relu", "tanh", "silu"):
        assert torch.isnan(fused_linear(x.to(DEV), w.to(DEV), activation=act)[130]).all()


def test_rows_behind_the_last_and_beside_the_matrix_stay_as_they_were():
    """The C ABI on buffers with room around them: nothing outside [n_rows, n_out] is written."""
    M, N, K = 130, 40, 24
    x, w, b, _, _ = _case(8, M, N, K, "f16")
    x, w, b = (t.to(DEV) for t in (x, w, b))
    buf = torch.full((M * N + 4096,), 7.0, dtype=torch.float16, device=DEV)
    p = capi.Linear(M, K, K, N, K, N, capi.F16, 0)
    L = capi.lib()
    n = L.cwrnnt_linear_workspace_bytes(ctypes.byref(p), 0)
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    capi.check(L.cwrnnt_linear_forward(ctypes.byref(p), x.data_ptr(), w.data_ptr(), b.data_ptr(), None, ws.data_ptr(), n,
                                       buf.data_ptr(), None))
    torch.cuda.synchronize()
    assert bool((buf[M * N:] == 7.0).all())
    _check(x, w, b, None, None, None, "f16", buf[:M * N].view(M, N), None)


def test_captured_and_replayed_on_new_contents():
    M, N, K = 500, 200, 120
    x, w, b, r, dy = (t.to(DEV) for t in _case(9, M, N, K, "bf16"))
    side = torch.cuda.Stream(DEV)

    def step():
        p = capi.Linear(M, K, K, N, K, N, capi.BF16, 2)
        L, st = capi.lib(), torch.cuda.current_stream().cuda_stream
        y, gx, gw, gb = torch.empty_like(r), torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
        n = max(L.cwrnnt_linear_workspace_bytes(ctypes.byref(p), 1), L.cwrnnt_linear_workspace_bytes(ctypes.byref(p), 2))
        ws = torch.empty(n, dtype=torch.uint8, device=DEV)
        capi.check(L.cwrnnt_linear_forward(ctypes.byref(p), x.data_ptr(), w.data_ptr(), b.data_ptr(), r.data_ptr(),
                                           ws.data_ptr(), n, y.data_ptr(), st))
        capi.check(L.cwrnnt_linear_backward(ctypes.byref(p), x.data_ptr(), w.data_ptr(), b.data_ptr(), dy.data_ptr(),
                                            ws.data_ptr(), n, gx.data_ptr(), gw.data_ptr(), gb.data_ptr(), st))
        return y, gx, gw, gb

    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y, gx, gw, gb = step()
    for seed in (10, 11):
        new = _case(seed, M, N, K, "bf16")
        for dst, src in zip((x, w, b, r, dy), new):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        _check(*new, "tanh", "bf16", y, (gx, gw, gb, None))


def test_results_repeat_bit_for_bit_on_other_streams():
    x, w, b, r, dy = (t.to(DEV) for t in _case(12, 6000, 200, 96, "bf16"))

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
        y = fused_linear(*leaves, activation="silu")
        return [y.detach(), *torch.autograd.grad([y], leaves, [dy])]

    first = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    got = []
    for s in streams:  # two at once
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    for other in got:
        for a, c in zip(first, other):
            assert torch.equal(a, c)


def test_joint_linear_loss_chain(oracle):
    """enc / pred -> compact_joint -> a hidden layer -> the output layer -> transducer_loss, gradients of both weights:
    against the same chain in double, with every tensor between the operators rounded as the operators round it."""
    from tests.helpers import ragged_case
    case = ragged_case(31, 3, (4, 9), (1, 4), V=24)
    rng = np.random.default_rng(4)
    lx, ly, y = (torch.as_tensor(case[k]).to(DEV) for k in ("lx", "ly", "y"))
    H, V = 32, 24
    enc = torch.as_tensor(rng.standard_normal((3, int(lx.max()), H))).bfloat16().to(DEV)
    pred = torch.as_tensor(rng.standard_normal((3, int(ly.max()) + 1, H))).bfloat16().to(DEV)
    W1 = torch.as_tensor(rng.standard_normal((H, H)) * 0.2).bfloat16().to(DEV).requires_grad_(True)
    W2 = torch.as_tensor(rng.standard_normal((V, H)) * 0.3).bfloat16().to(DEV).requires_grad_(True)
    b2 = torch.as_tensor(rng.standard_normal(V) * 0.1).bfloat16().to(DEV).requires_grad_(True)
    h = compact_joint(enc, pred, lx, ly, "tanh")
    h2 = fused_linear(h, W1, None, h, activation="silu")
    logits = fused_linear(h2, W2, b2)
    h2.retain_grad(), logits.retain_grad()
    loss = transducer_loss(logits, lx, y, ly, fused_log_softmax=True)
    loss.backward()
    _check(h.cpu(), W1.cpu(), None, h.cpu(), h2.grad.cpu(), "silu", "bf16", h2, (None, W1.grad, None, None))
    _check(h2.cpu(), W2.cpu(), b2.cpu(), None, logits.grad.cpu(), None, "bf16", logits, (h2.grad, W2.grad, b2.grad, None))
    costs, _ = oracle.fused(_np(logits), case["lx"], case["ly"], case["y"], 0, weights=np.full(3, 1.0 / 3))
    assert abs(float(loss.detach()) - costs.mean()) <= 1e-5 * abs(costs.mean())


def test_not_differentiable_twice():
    x, w, b, r, _ = (t.to(DEV) for t in _case(13, 20, 16, 24, "bf16"))
    xl = x.requires_grad_(True)
    g, = torch.autograd.grad(fused_linear(xl, w, b, r, activation="tanh").float().sum(), [xl], create_graph=True)
    assert torch.isfinite(g).all()
    with pytest.raises(RuntimeError, match="twice"):
        g.float().sum().backward()
