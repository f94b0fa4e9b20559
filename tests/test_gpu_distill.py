"""GPU tests of distill_loss against the 64-bit oracle: both forms, every type and row size, masks, weights, repeated
and unused entries, reductions, the eager and the late gradient, differences, graphs, and a transducer distilled through
token_scores and analyse.

Tolerances: a row's divergence adds entries q (ln q - ln p) whose log-probabilities are good to SUM32 (derived in
tests/rowops_oracle.py), so it is off by that times their magnitude, and by one rounding to float; a gradient element
is off by SUM32 times the magnitudes of its terms and one rounding to the row's type."""
import numpy as np
import pytest
import torch

from compactwarprnntloss_b200 import distill_loss, token_scores
from tests import rowops_oracle as ro

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64}


def _case(seed, R, V, K, dtype, tail=True, spread=2.0, tau=1.0):
    """Student rows (CPU, dtype), the teacher's K best (values, int32 tokens) from logits near the student's."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, V, generator=g, dtype=torch.float64) * spread
    t = x + 0.7 * torch.randn(R, V, generator=g, dtype=torch.float64)
    val, idx = torch.log_softmax(t / tau, 1).topk(K, 1)
    ct = torch.float64 if dtype == torch.float64 else torch.float32
    return x.to(dtype), val.to(ct), idx.to(torch.int32)


def _check(x, val, idx, weight, tail, tau, rows, gx):
    x64 = x.double().numpy()
    loss, grad, lmag, gmag = ro.distill(x64, val.double().numpy(), idx.numpy(),
                                        None if weight is None else weight.double().numpy(), tail, tau)
    name = str(x.dtype).split(".")[1]
    err = ro.SUM64 if x.dtype == torch.float64 else ro.SUM32
    got = rows.detach().double().cpu().numpy()
    unit = 2.0 ** -53 if x.dtype == torch.float64 else 2.0 ** -24
    fine = np.isfinite(loss)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(loss))
    assert (np.abs(got[fine] - loss[fine]) <= 2 * err * lmag[fine] + unit * np.abs(loss[fine])).all()
    np.testing.assert_array_equal(got[~fine & ~np.isnan(loss)], loss[~fine & ~np.isnan(loss)])
    g = gx.double().cpu().numpy()
    np.testing.assert_array_equal(np.isnan(g), np.isnan(grad))
    ok = ~np.isnan(grad)
    bound = ro.HALF_STEP[name] * np.abs(grad) + 2 * err * gmag + ro.TINY[name]
    assert (np.abs(g - grad)[ok] <= bound[ok]).all(), np.nanmax(np.abs(g - grad) - bound)


def _run(x, val, idx, weight=None, tail=True, tau=1.0):
    xd = x.to(DEV).requires_grad_(True)
    w = None if weight is None else weight.to(DEV)
    rows = distill_loss(xd, val.to(DEV), idx.to(DEV), weight=w, tail=tail, temperature=tau, reduction="none")
    gx, = torch.autograd.grad([rows], [xd], [torch.ones_like(rows)])
    _check(x, val, idx, weight, tail, tau, rows, gx)
    # the summed loss with the gradient from the same pass
    total = distill_loss(xd, val.to(DEV), idx.to(DEV), weight=w, tail=tail, temperature=tau, reduction="sum")
    g2, = torch.autograd.grad(total, [xd])
    assert torch.equal(torch.nan_to_num(g2), torch.nan_to_num(gx))
    return rows, total


@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16", "f64"])
@pytest.mark.parametrize("V", [1, 2, 5, 32, 33, 128, 129, 256, 260, 512, 1000, 1024, 1026, 2048, 4096, 4104, 10007, 33000])
def test_every_row_size(dtype, V, tail):
    R = 4 if V > 2048 else 21
    K = min(V, 3)
    _run(*_case(V, R, V, K, DT[dtype]), tail=tail)


@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("K", [1, 2, 4, 5, 8, 9, 16, 17, 32])
@pytest.mark.parametrize("V,dtype", [(32, "bf16"), (128, "f16"), (1024, "f32"), (4096, "bf16"), (5003, "f16"),
                                     (90, "f64")])
def test_every_list_length(K, V, dtype, tail):
    g = torch.Generator().manual_seed(K)
    w = torch.rand(9, generator=g, dtype=torch.float64 if dtype == "f64" else torch.float32)
    w[::4] = 0.0
    _run(*_case(K, 9, V, K, DT[dtype], tau=2.0), weight=w, tail=tail, tau=2.0)


@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("V,dtype", [(40, "f16"), (128, "f32"), (1000, "bf16"), (4099, "f32"), (30, "f64")])
def test_unused_repeated_and_impossible_entries(V, dtype, tail):
    x, val, idx = _case(V, 10, V, 6, DT[dtype])
    idx[1, 2:] = -1                    # a shorter list
    idx[2] = -1                        # no entry at all
    idx[3, 1] = idx[3, 0]              # a token named twice
    idx[4] = idx[4, 0]                 # six times
    val[4] -= 3.0
    val[5, 1] = float("-inf")          # the teacher rules a listed token out
    val[6] = float("-inf")             # all of them
    idx[7, 5] = V                      # outside the row: that row's loss and gradient are NaN
    idx[8, 0] = 2147483647
    val[9] = -40.0                     # nearly everything is left to the rest
    rows, total = _run(x, val, idx, tail=tail)
    assert torch.isnan(rows[7:9]).all() and torch.isfinite(rows[[0, 1, 2, 3, 4, 5, 9]]).all()
    assert abs(float(rows[2])) <= ro.SUM32 and torch.isnan(total)


@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("V,dtype", [(24, "f32"), (128, "f16"), (1024, "bf16"), (1029, "f32"), (6000, "bf16"),
                                     (50, "f64")])
def test_masks_infinities_and_nan(V, dtype, tail):
    x, val, idx = _case(V + 1, 12, V, 4, DT[dtype])
    ct = val.dtype
    ninf = float("-inf")
    low = torch.finfo(DT[dtype]).min
    x[0] = ninf                                     # the student has nothing: no loss, no gradient
    keep = x[1].clone()
    x[1] = ninf                                     # only listed tokens are left: no class for the rest
    x[1, idx[1].long()] = keep[idx[1].long()]
    x[2, int(idx[2, 0])] = ninf                     # a listed token is impossible for the student: infinite loss
    x[3, int(idx[3, 1])] = float("nan")             # NaN at a listed token
    other = [j for j in range(V) if j not in idx[4].tolist()][0]
    x[4, other] = float("nan")                      # NaN elsewhere
    x[5, :] = low
    x[6, V // 2:] = low
    x[7, :] = float("nan")                          # masked by its weight
    x[8, 0] = float("inf")
    x[9, int(idx[9, 0])] = torch.finfo(DT[dtype]).max / 4  # the student is sure of a listed token
    w = torch.ones(12, dtype=ct)
    w[7] = 0.0
    w[10] = -0.5
    rows, _ = _run(x, val, idx, weight=w, tail=tail)
    assert float(rows[0]) == 0.0 and float(rows[7]) == 0.0
    assert float(rows[2]) == float("inf") and torch.isnan(rows[[3, 4, 8]]).all()


@pytest.mark.parametrize("V,dtype", [(96, "bf16"), (1024, "f32"), (1030, "f16"), (5000, "bf16")])
def test_strided_and_misaligned_rows(V, dtype):
    x, val, idx = _case(3, 9, V + 11, 5, DT[dtype])
    idx = idx.remainder(V)
    dev = x.to(DEV)
    for start in (0, 1, 8):
        view = dev[:, start:start + V].detach().requires_grad_(True)
        rows = distill_loss(view, val.to(DEV), idx.to(DEV), reduction="none")
        gx, = torch.autograd.grad([rows], [view], [torch.ones_like(rows)])
        _check(x[:, start:start + V], val, idx, None, True, 1.0, rows, gx)


def test_reductions_denominators_and_upstream_gradients():
    x, val, idx = _case(5, 50, 200, 4, torch.float32)
    w = torch.linspace(0.0, 2.0, 50)
    args = (val.to(DEV), idx.to(DEV))
    kw = dict(weight=w.to(DEV))
    loss, grad, lmag, gmag = ro.distill(x.double().numpy(), val.double().numpy(), idx.numpy(), w.numpy(), True, 1.0)
    up = np.linspace(-1.0, 1.0, 50)

    def grad_of(make, factor):
        for eager in (True, False):
            xd = x.to(DEV).requires_grad_(True)
            out = make(xd, eager)
            (3.0 * out).sum().backward() if factor is None else torch.autograd.backward([out], [factor])
            yield out.detach(), xd.grad.double().cpu().numpy()

    for reduction, denominator, divide in (("mean", 0, 50.0), ("mean", 7.5, 7.5), ("sum", 0, 1.0)):
        for out, g in grad_of(lambda xd, eager: distill_loss(xd, *args, **kw, reduction=reduction, eager_grad=eager,
                                                             mean_denominator=denominator), None):
            # the loss: the rows' errors, and one rounding
            assert abs(float(out) - loss.sum() / divide) <= (2 * ro.SUM32 * lmag.sum() + 2.0 ** -24 * abs(loss.sum())) / divide
            want = 3.0 * grad / divide
            # a gradient scaled after its rounding is rounded twice
            assert (np.abs(g - want) <= 2 * 2.0 ** -24 * np.abs(want) + 3.0 / divide * 2 * ro.SUM32 * gmag).all()
    for out, g in grad_of(lambda xd, eager: distill_loss(xd, *args, **kw, reduction=None, eager_grad=eager),
                          torch.as_tensor(up, dtype=torch.float32, device=DEV)):
        want = np.float32(up).astype(np.float64)[:, None] * grad
        assert (np.abs(g - want) <= 2.0 ** -24 * np.abs(want) + 2 * ro.SUM32 * np.abs(up)[:, None] * gmag).all()


def test_retained_graph_gives_the_gradient_again():
    x, val, idx = _case(6, 20, 1024, 2, torch.bfloat16)
    xd = x.to(DEV).requires_grad_(True)
    loss = distill_loss(xd, val.to(DEV), idx.to(DEV), reduction="sum")
    a, = torch.autograd.grad(loss, [xd], retain_graph=True)
    b, = torch.autograd.grad(loss, [xd])
    assert torch.equal(a, b)


def test_gradient_against_differences():
    x, val, idx = _case(7, 3, 40, 4, torch.float64)
    idx[2, 3] = idx[2, 0]
    args = (val.to(DEV), idx.to(DEV))
    for tail, tau in ((True, 1.0), (False, 1.8)):
        leaf = x.to(DEV).requires_grad_(True)
        gx, = torch.autograd.grad(distill_loss(leaf, *args, tail=tail, temperature=tau, reduction="sum"), [leaf])
        h = 1e-5  # third derivatives below one: h^2 = 1e-10, rounding 1e-15 / h = 1e-10
        for r, j in [(0, int(idx[0, 1])), (0, 39), (1, 0), (2, int(idx[2, 0]))]:
            up, down = x.clone(), x.clone()
            up[r, j] += h
            down[r, j] -= h
            f = [float(distill_loss(v.to(DEV), *args, tail=tail, temperature=tau, reduction="sum")) for v in (up, down)]
            assert abs((f[0] - f[1]) / (2 * h) - float(gx[r, j])) < 1e-8


def test_a_confident_student_keeps_the_digits_of_the_rest():
    """Listed tokens hold all but 1e-12 of the student's probability: ln p_rest and its gradient from the sums of the
    rest alone, not from one minus the listed ones."""
    V = 64
    x = torch.zeros(2, V)
    x[:, 0], x[:, 1] = 32.0, 31.0
    idx = torch.tensor([[0, 1]] * 2, dtype=torch.int32)
    val = torch.log(torch.tensor([[0.5, 0.3]] * 2))
    _run(x, val, idx)


@pytest.mark.parametrize("V,dtype", [(4096, "f16"), (40001, "f32"), (65536, "bf16")])
def test_a_rest_that_is_nearly_all_keeps_the_digits_of_its_logarithm(V, dtype):
    """The listed tokens hold a few V-ths of a flat student: -ln p_rest is about their share P of it, and a rest summed to
    SUM32 moves it by P SUM32 only. The listed ln p move by SUM32 (x / tau - max / tau is taken in double), each times its
    q. Beside these there are the double steps (an exponential and three logarithms to 2^-33 each) and one rounding."""
    x, _, idx = _case(21, 64, V, 2, DT[dtype], spread=0.1)
    val = torch.full((64, 2), 4.0 / V).log()
    rows = distill_loss(x.to(DEV), val.to(DEV), idx.to(DEV), reduction="none").double().cpu()
    want = torch.from_numpy(ro.distill(x.double().numpy(), val.double().numpy(), idx.numpy(), None, True, 1.0)[0])
    p = torch.softmax(x.double(), 1).gather(1, idx.long())
    bound = ro.SUM32 * (val.double().exp().sum(1) + p.sum(1)) + 2.0 ** -31 + 2.0 ** -24 * want.abs()
    assert ((rows - want).abs() <= bound).all(), ((rows - want).abs() / bound).max()


def test_empty_batches_and_leading_axes():
    x, val, idx = _case(8, 24, 60, 3, torch.float32)
    a = distill_loss(x.view(2, 3, 4, 60).to(DEV), val.view(2, 3, 4, 3).to(DEV), idx.view(2, 3, 4, 3).to(DEV), reduction="none")
    assert a.shape == (2, 3, 4)
    assert torch.equal(a.reshape(-1), distill_loss(x.to(DEV), val.to(DEV), idx.to(DEV), reduction="none"))
    e = x[:0].to(DEV).requires_grad_(True)
    for reduction in ("mean", "sum"):
        loss = distill_loss(e, val[:0].to(DEV), idx[:0].to(DEV), reduction=reduction)
        assert float(loss) == 0.0
        loss.backward()
    assert distill_loss(e, val[:0].to(DEV), idx[:0].to(DEV), reduction="none").shape == (0,)


def test_captured_and_replayed_on_new_contents():
    x0, v0, i0 = _case(9, 300, 1000, 3, torch.bfloat16)
    x, val, idx = x0.to(DEV), v0.to(DEV), i0.to(DEV)
    side = torch.cuda.Stream(DEV)
    with torch.cuda.stream(side):
        distill_loss(x, val, idx)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        loss = distill_loss(x, val, idx)
    for seed in (10, 11):
        nx, nv, ni = _case(seed, 300, 1000, 3, torch.bfloat16)
        x.copy_(nx), val.copy_(nv), idx.copy_(ni)
        graph.replay()
        torch.cuda.synchronize()
        want, _, lmag, _ = ro.distill(nx.double().numpy(), nv.double().numpy(), ni.numpy(), None, True, 1.0)
        assert abs(float(loss) - want.mean()) <= 2 * ro.SUM32 * lmag.mean() + 2.0 ** -24 * abs(want.mean())


def test_backward_captured_without_its_forward():
    """Every replay gives the gradient for the upstream gradient of that moment, not the last one's multiple."""
    x, val, idx = (t.to(DEV) for t in _case(22, 40, 300, 3, torch.float32))
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = x.clone().requires_grad_(True)
        loss = distill_loss(leaf, val, idx, reduction="sum")
        up = torch.full((), 2.0, device=DEV)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        g, = torch.autograd.grad([loss], [leaf], [up], retain_graph=True)
    other = x.clone().requires_grad_(True)
    want, = torch.autograd.grad(distill_loss(other, val, idx, reduction="sum"), [other])
    for factor in (2.0, 2.0, -0.5):
        up.fill_(factor)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(g, factor * want)


@pytest.mark.parametrize("V,dtype", [(1000, "bf16"), (9000, "f32")])
def test_two_streams_at_once(V, dtype):
    """Teacher's pass, loss and gradient on two streams that overlap: each the bits of a call on its own."""
    def step(x, teacher):
        t = token_scores(teacher, top_k=8)
        leaf = x.clone().requires_grad_(True)
        loss = distill_loss(leaf, t.top_log_probs, t.top_indices)
        g, = torch.autograd.grad(loss, [leaf])
        return t.top_log_probs, t.top_indices, loss.detach(), g

    data = [[_case(seed + k, 700, V, 1, DT[dtype])[0].to(DEV) for k in (0, 1)] for seed in (30, 40)]
    want = [step(*d) for d in data]
    streams = [torch.cuda.Stream(DEV) for _ in data]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, d in zip(streams, data):
            with torch.cuda.stream(s):
                got.append(step(*d))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_teacher_entries_from_token_scores():
    """The two operators together: the teacher's best tokens from token_scores are what distill_loss takes."""
    x, _, _ = _case(12, 33, 500, 1, torch.bfloat16)
    t, _, _ = _case(13, 33, 500, 1, torch.bfloat16)
    s = token_scores(t.to(DEV), top_k=7, temperature=1.5)
    val, idx = s.top_log_probs, s.top_indices
    rows, _ = _run(x, val.cpu(), idx.cpu(), tau=1.5)
    assert (rows > -1e-5).all()


def test_transducer_distilled_through_the_lattice():
    """Blank, label and the rest at every lattice node, weighted by the node posteriors of the student's own lattice:
    token_scores on the teacher's rows, analyse on the student's, distill_loss beside transducer_loss."""
    from compactwarprnntloss_b200 import analyse, transducer_loss
    from tests.helpers import ragged_case
    case = ragged_case(21, 3, (4, 9), (1, 5), V=40)
    lx, ly = torch.as_tensor(case["lx"]).to(DEV), torch.as_tensor(case["ly"]).to(DEV)
    y = torch.as_tensor(case["y"]).to(DEV)
    x = torch.as_tensor(case["x"]).to(DEV).requires_grad_(True)
    teacher = torch.as_tensor(case["x"]).to(DEV) + 0.5 * torch.randn(x.shape, generator=torch.Generator(DEV).manual_seed(1), device=DEV)
    nodes, weight = [], []
    post = analyse(x.detach(), lx, y, ly, fused_log_softmax=True).posteriors
    for n in range(3):
        T, U = int(lx[n]), int(ly[n])
        col = torch.full((T, U + 1, 2), -1, dtype=torch.int32)
        col[..., 0] = 0
        col[:, :U, 1] = y[n, :U].cpu()
        nodes.append(col.view(-1, 2))
        weight.append(post[n, :T, :U + 1].reshape(-1))
    nodes, weight = torch.cat(nodes).to(DEV), torch.cat(weight)
    lp = token_scores(teacher, nodes).log_probs
    loss = distill_loss(x, lp, nodes, weight=weight, reduction="sum")
    both = transducer_loss(x, lx, y, ly, fused_log_softmax=True) + loss
    both.backward()
    want, grad, lmag, gmag = ro.distill(x.detach().double().cpu().numpy(), lp.double().cpu().numpy(),
                                        nodes.cpu().numpy(), weight.double().cpu().numpy(), True, 1.0)
    assert abs(float(loss) - want.sum()) <= 2 * ro.SUM32 * lmag.sum() + 2.0 ** -24 * want.sum()
    from oracle import oracle as o
    _, dense = o.fused(case["x"], case["lx"], case["ly"], case["y"], 0, weights=np.full(3, 1.0 / 3))
    # the lattice's own gradient is good to 1e-5 (the parity tests' bound)
    assert (np.abs(x.grad.double().cpu().numpy() - (grad + dense)) <= 1e-5 + 2 * ro.SUM32 * gmag).all()


def test_not_differentiable_twice():
    x, val, idx = _case(14, 6, 50, 2, torch.float32)
    for reduction in ("mean", "none"):
        xd = x.to(DEV).requires_grad_(True)
        loss = distill_loss(xd, val.to(DEV), idx.to(DEV), reduction=reduction)
        g, = torch.autograd.grad(loss.sum(), [xd], create_graph=True)
        assert torch.isfinite(g).all()
        with pytest.raises(RuntimeError, match="twice"):
            g.sum().backward()
