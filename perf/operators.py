"""What the row operators around the transducer lattice are measured on: the joint's linear layer, the scores of its
logits rows, and distillation from a teacher's top entries.

Three operators of `compactwarprnntloss_b200`, each in the calls that a user makes (`own`) and in a plain form of
elementary torch operations in 32 bits:

  token_scores   log-probabilities of given tokens, entropy and the top alternatives of every row of logits, and the
                 gradient of all three
  distill_loss   cross entropy against a teacher's top entries, with or without a class for everything else, loss and
                 gradient
  fused_linear   act(x W^T + b) + residual, and its gradients

Sizes are those of the transducer workloads of this repository (a Conformer batch of 314 340 lattice nodes with 1 024
tokens, a 4 096-token one, ragged 128-token rows, a joint 640 wide) and generic text vocabularies.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one step of a beam search: the joint's rows of 16 hypotheses, eight alternatives each
        dict(name="scores_beam_step_bf16", op="scores", dtype="bf16", rows=16, V=1024, targets=0, top=8, entropy=False,
             grad=False, tau=1.0, padded=0),
        # confidence training on a whole Conformer lattice: blank and label of every node, entropy, and the gradient
        dict(name="scores_lattice_f32", op="scores", dtype="f32", rows=314340, V=1024, targets=2, top=0, entropy=True,
             grad=True, tau=1.0, padded=0),
        # a teacher's pass over a large vocabulary: its sixteen best tokens of every node, to be stored
        dict(name="scores_teacher_bf16", op="scores", dtype="bf16", rows=80003, V=4096, targets=1, top=16,
             entropy=True, grad=False, tau=1.0, padded=0),
        # scoring text with a language model's vocabulary of odd size (no row but the first is aligned)
        dict(name="scores_text_f16", op="scores", dtype="f16", rows=2051, V=50257, targets=1, top=20, entropy=True,
             grad=False, tau=1.0, padded=0),
        # rows shorter than a warp's load: the ragged workload's character vocabulary
        dict(name="scores_ragged_f16", op="scores", dtype="f16", rows=600011, V=128, targets=2, top=4, entropy=True,
             grad=False, tau=1.0, padded=0),
        # transducer distillation: blank, label and the rest at every node, weighted by the node posteriors
        dict(name="distill_lattice_bf16", op="distill", dtype="bf16", rows=314340, V=1024, K=2, tail=True, tau=1.0,
             weighted=True),
        # distillation from a teacher's stored top sixteen, renormalised, at a raised temperature
        dict(name="distill_top_bf16", op="distill", dtype="bf16", rows=40961, V=4096, K=16, tail=False, tau=2.0,
             weighted=False),
        # one short utterance
        dict(name="distill_short_f16", op="distill", dtype="f16", rows=33, V=129, K=3, tail=True, tau=1.0,
             weighted=True),
        # a text vocabulary in single precision
        dict(name="distill_text_f32", op="distill", dtype="f32", rows=2047, V=32003, K=32, tail=True, tau=1.0,
             weighted=False),
        # the joint's output layer in a decoding step
        dict(name="linear_step_bf16", op="linear", dtype="bf16", rows=8, N=1024, K=640, bias=True, act="none",
             residual=False, grad=False),
        # the joint's output layer over a whole Conformer lattice
        dict(name="linear_logits_bf16", op="linear", dtype="bf16", rows=314340, N=1024, K=640, bias=True, act="none",
             residual=False, grad=False),
        # a hidden layer in training: bias, tanh and residual, and all its gradients
        dict(name="linear_train_f16", op="linear", dtype="f16", rows=40009, N=640, K=512, bias=True, act="tanh",
             residual=True, grad=True),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["scores", "distill", "linear"])
    if op == "linear":
        N, K = _spread(rng, 1, 2048), _spread(rng, 1, 2048)
        if rng.random() < 0.5:
            N, K = -(-N // 8) * 8, -(-K // 8) * 8
        grad = rng.random() < 0.5
        rows = _spread(rng, 1, min(314340, 314340 * 1024 * 640 // (N * K * (4 if grad else 1))))
        return dict(op="linear", dtype=rng.choice(["bf16", "f16"]), rows=rows, N=N, K=K, bias=rng.random() < 0.8,
                    act=rng.choice(["none", "relu", "tanh", "silu"]), residual=rng.random() < 0.4, grad=grad)
    V = _spread(rng, 2, 70000)
    if rng.random() < 0.5:
        V = -(-V // 8) * 8
    grad = op == "distill" or rng.random() < 0.5
    rows = _spread(rng, 1, min(700000, 314340 * 1024 // ((2 if grad else 1) * V)))
    dtype = rng.choice(["bf16", "f16", "f32"])
    if op == "scores":
        top = min(V, rng.choice([0, 1, 2, 4, 8, 13, 20, 32]))
        targets = rng.choice([0, 1, 2, 5])
        return dict(op="scores", dtype=dtype, rows=rows, V=V, targets=targets, top=top,
                    entropy=rng.random() < 0.5 or not (top or targets), grad=grad,
                    tau=rng.choice([1.0, 1.0, 1.5]), padded=rng.choice([0, 0, V // 16]))
    return dict(op="distill", dtype=dtype, rows=rows, V=V, K=min(V, rng.choice([1, 2, 3, 8, 16, 27, 32])),
                tail=rng.random() < 0.5, tau=rng.choice([1.0, 1.0, 2.0]), weighted=rng.random() < 0.5)


def work(case):
    e, R = BYTES[case["dtype"]], case["rows"]
    if case["op"] == "scores":
        small = 8 * case["targets"] + 8 * case["top"] + 4 * case["entropy"]
        passes = 2 if case["grad"] else 1  # the row read once; in training its gradient written once
        return {"bytes": R * (case["V"] * e * passes + small), "flops": R * case["V"] * 4.0 * passes}
    if case["op"] == "distill":
        return {"bytes": R * (case["V"] * e * 2 + 8 * case["K"] + 4 * case["weighted"]), "flops": R * case["V"] * 8.0}
    N, K = case["N"], case["K"]
    moved = R * K + N * K + R * N + N * case["bias"] + R * N * case["residual"]
    if case["grad"]:
        moved += R * N + R * K + N * K + N * case["bias"]
    return {"bytes": moved * e, "flops": 2.0 * R * N * K * (3 if case["grad"] else 1)}


# ----------------------------------------------------------------------------------------------------------- inputs

def _normal(g, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, R = DTYPES[case["dtype"]], case["rows"]
    s = {"case": case}
    if case["op"] == "linear":
        N, K = case["N"], case["K"]
        s["x"] = _normal(g, (R, K), dtype)
        s["weight"] = _normal(g, (N, K), dtype, K ** -0.5)
        s["bias"] = _normal(g, (N,), dtype, 0.5) if case["bias"] else None
        s["residual"] = _normal(g, (R, N), dtype) if case["residual"] else None
        s["activation"] = case["act"]
        if case["grad"]:
            s["dy"] = _normal(g, (R, N), dtype)
            for name in ("x", "weight", "bias", "residual"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
        return s
    V = case["V"]
    x = torch.randn((R, V), generator=g, device="cuda", dtype=torch.float32).mul_(2.0)
    # a joint's rows: at a good part of the nodes the blank (token 0) stands out
    x[:, 0] += 8.0 * (torch.rand(R, generator=g, device="cuda") < 0.4)
    if case["op"] == "scores":
        if case["padded"]:
            x[:, V - case["padded"]:] = -math.inf  # a vocabulary padded to a round size
        s["x"] = x.to(dtype)
        P = case["targets"]
        live = V - case["padded"]
        t = torch.randint(0, live, (R, P), generator=g, device="cuda", dtype=torch.int32)
        if P >= 2:
            t[:, 0] = 0
            t[torch.rand(R, generator=g, device="cuda") < 0.02, 1] = -1  # the last column of a lattice has no label
        s["targets"] = t if P else None
        if case["grad"]:
            s["x"].requires_grad_(True)
            s["g_lp"] = _normal(g, (R, P), torch.float32) if P else None
            s["g_ent"] = _normal(g, (R,), torch.float32) if case["entropy"] else None
            s["g_top"] = _normal(g, (R, case["top"]), torch.float32) if case["top"] else None
        return s
    K = case["K"]
    teacher = x.add(torch.randn((R, V), generator=g, device="cuda"), alpha=0.7).div_(case["tau"])
    teacher -= torch.logsumexp(teacher, 1, keepdim=True)
    top, index = teacher.topk(K, 1)
    s["teacher"], s["index"] = top.contiguous(), index.to(torch.int32).contiguous()
    s["x"] = x.to(dtype).requires_grad_(True)
    s["weight"] = None
    if case["weighted"]:
        w = torch.rand(R, generator=g, device="cuda")
        s["weight"] = w * (w > 0.1)  # nodes that no alignment passes through weigh nothing
    return s


# -------------------------------------------------------------------------------------------------------- the calls

def run(s):
    case = s["case"]
    if own:
        return _run_own(case, s)
    with torch.no_grad():
        return {"scores": _scores, "distill": _distill, "linear": _linear}[case["op"]](case, s)


def _run_own(case, s):
    x = s["x"]
    if case["op"] == "scores":
        from compactwarprnntloss_b200 import token_scores
        r = token_scores(x, s["targets"], top_k=case["top"], entropy=case["entropy"], temperature=case["tau"])
        out = {"log_probs": r.log_probs, "entropy": r.entropy, "top": r.top_log_probs, "index": r.top_indices}
        if case["grad"]:
            pairs = [(r.log_probs, s["g_lp"]), (r.entropy, s["g_ent"]), (r.top_log_probs, s["g_top"])]
            pairs = [(o, d) for o, d in pairs if o is not None]
            out["grad"], = torch.autograd.grad([o for o, _ in pairs], [x], [d for _, d in pairs])
        return out
    if case["op"] == "distill":
        from compactwarprnntloss_b200 import distill_loss
        loss = distill_loss(x, s["teacher"], s["index"], weight=s["weight"], tail=case["tail"],
                            temperature=case["tau"], reduction="mean")
        grad, = torch.autograd.grad(loss, [x])
        return {"loss": loss, "grad": grad}
    from compactwarprnntloss_b200 import fused_linear
    y = fused_linear(x, s["weight"], s["bias"], s["residual"], activation=s["activation"])
    out = {"y": y}
    if case["grad"]:
        names = [n for n in ("x", "weight", "bias", "residual") if s[n] is not None]
        out.update(zip(names, torch.autograd.grad([y], [s[n] for n in names], [s["dy"]])))
    return out


# ------------------------------------------------------------------------------------------------------ plain forms

def _plain_log_probs(x, tau):
    z = x.float() / tau
    m = z.amax(1, keepdim=True)
    return z - (m + (z - m).exp().sum(1, keepdim=True).log())


def _scores(case, s):
    x, k = s["x"], case["top"]
    R, V = x.shape
    logp = _plain_log_probs(x, case["tau"])
    out = {"log_probs": None, "entropy": None, "top": None, "index": None}
    if s["targets"] is not None:
        t = s["targets"].long()
        picked = logp.gather(1, t.clamp(min=0))
        out["log_probs"] = torch.where(t >= 0, picked, torch.zeros_like(picked))
    p = logp.exp() if case["entropy"] or case["grad"] else None
    if case["entropy"]:
        plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
        out["entropy"] = -plogp.sum(1)
    if k:
        # whole-number keys: the value's order in the upper bits, the lower index first among equals
        bits = (x.float() + 0.0).view(torch.int32)
        order = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long()
        key = (order << 32) + (V - 1 - torch.arange(V, device=x.device))
        index = V - 1 - (key.topk(k, 1)[0] & 0xFFFFFFFF)
        out["top"], out["index"] = logp.gather(1, index), index.int()
    if case["grad"]:
        grad = torch.zeros_like(p)
        total = torch.zeros(R, 1, device=x.device)
        if s["targets"] is not None:
            d = torch.where(t >= 0, s["g_lp"], torch.zeros_like(s["g_lp"]))
            grad.scatter_add_(1, t.clamp(min=0), d)
            total += d.sum(1, keepdim=True)
        if k:
            grad.scatter_add_(1, index, s["g_top"])
            total += s["g_top"].sum(1, keepdim=True)
        grad -= p * total
        if case["entropy"]:
            grad -= s["g_ent"][:, None] * (plogp + p * out["entropy"][:, None])
        out["grad"] = (grad / case["tau"]).to(x.dtype)
    return out


def _distill(case, s):
    x, index = s["x"], s["index"].long()
    R, V = x.shape
    tau = case["tau"]
    logp = _plain_log_probs(x, tau)
    p = logp.exp()
    if case["tail"]:
        q = s["teacher"].exp()
        logq = s["teacher"]
    else:
        logq = _plain_log_probs(s["teacher"], tau)
        q = logq.exp()
    each = (torch.where(q > 0, q * (logq - logp.gather(1, index)), torch.zeros_like(q))).sum(1)
    w = s["weight"] if s["weight"] is not None else torch.ones(R, device=x.device)
    grad = p * q.sum(1, keepdim=True)
    if case["tail"] and V > case["K"]:
        # what the teacher leaves for the other tokens: a small difference, taken in 64 bits
        q_rest = (1.0 - s["teacher"].double().exp().sum(1)).clamp(min=0.0).float()
        listed_ = torch.zeros_like(p, dtype=torch.bool).scatter_(1, index, True)
        other = torch.where(listed_, torch.full_like(logp, -math.inf), logp)
        m = other.amax(1)
        log_rest = m + (other - m[:, None]).exp().sum(1).log()
        each = each + torch.where(q_rest > 0, q_rest * (q_rest.log() - log_rest), torch.zeros_like(q_rest))
        grad += p * q_rest[:, None]
        grad -= torch.where(listed_, torch.zeros_like(p), q_rest[:, None] * (other - log_rest[:, None]).exp())
    grad.scatter_add_(1, index, -q)
    grad *= (w / (R * tau))[:, None]
    return {"loss": (w * each).double().sum().div(R).float(), "grad": grad.to(x.dtype)}


def _act(name, z):
    if name == "relu":
        return z.clamp(min=0.0), (z > 0).float()
    if name == "tanh":
        e = z.tanh()
        return e, 1.0 - e * e
    if name == "silu":
        sg = 1.0 / (1.0 + (-z).exp())
        return z * sg, sg * (1.0 + z * (1.0 - sg))
    return z, None


def _linear(case, s):
    x, W = s["x"].float(), s["weight"].float()
    z = x @ W.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    a, slope = _act(s["activation"], z)
    y = a if s["residual"] is None else a + s["residual"].float()
    out = {"y": y.to(s["x"].dtype)}
    if case["grad"]:
        dy = s["dy"].float()
        dz = dy if slope is None else dy * slope
        out["x"] = (dz @ W).to(s["x"].dtype)
        out["weight"] = (dz.t() @ x).to(s["x"].dtype)
        if s["bias"] is not None:
            out["bias"] = dz.sum(0).to(s["x"].dtype)
        if s["residual"] is not None:
            out["residual"] = dy.to(s["x"].dtype)
    return out


# ------------------------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    """The definitions in 64 bits: scores and losses written out, gradients by differentiating them."""
    s = prepare(case, seed)
    if case["op"] == "linear":
        return _exact_linear(case, s)
    step = max(1, (1 << 25) // case["V"])
    parts = [_exact_rows(case, {k: (v[a:a + step].detach() if torch.is_tensor(v) else v) for k, v in s.items()})
             for a in range(0, case["rows"], step)]
    out = {k: None if parts[0][k] is None else torch.cat([p[k] for p in parts]) for k in parts[0]}
    if case["op"] == "distill":
        out["loss"] = out["loss"].sum()
    return out


def _exact_rows(case, s):
    x = s["x"].double().requires_grad_(True)
    with torch.enable_grad():
        lp = torch.log_softmax(x / case["tau"], 1)
        if case["op"] == "scores":
            out, total = {"log_probs": None, "entropy": None, "top": None, "index": None}, 0.0
            if s["targets"] is not None:
                hit = s["targets"] >= 0
                got = lp.gather(1, s["targets"].clamp(min=0).long())
                out["log_probs"] = torch.where(hit, got, 0.0)
                total = total + ((out["log_probs"] * s["g_lp"].double()).sum() if case["grad"] else 0.0)
            if case["entropy"]:
                seen = lp.masked_fill(x == -math.inf, 0.0)
                out["entropy"] = -(seen * seen.exp()).masked_fill(x == -math.inf, 0.0).sum(1)
                total = total + ((out["entropy"] * s["g_ent"].double()).sum() if case["grad"] else 0.0)
            if case["top"]:
                first = torch.sort(x.detach(), dim=1, descending=True, stable=True)[1][:, :case["top"]]
                out["top"] = lp.gather(1, first)
                total = total + ((out["top"] * s["g_top"].double()).sum() if case["grad"] else 0.0)
            if case["grad"]:
                out["grad"], = torch.autograd.grad(total, x)
            return {k: None if v is None else v.detach() for k, v in out.items()}
        a = s["teacher"].double()
        index = s["index"].long()
        if case["tail"]:
            q = a.exp()
        else:
            q = torch.softmax(a / case["tau"], 1)
        D = (torch.special.xlogy(q, q) - q * lp.gather(1, index)).sum(1)
        if case["tail"] and case["K"] < case["V"]:
            left = (1.0 - q.sum(1)).clamp(min=0.0)
            rest = torch.logsumexp(lp.scatter(1, index, -math.inf), 1)
            D = D + torch.special.xlogy(left, left) - left * rest
        if s["weight"] is not None:
            D = D * s["weight"].double()
        D = D / case["rows"]
        grad, = torch.autograd.grad(D.sum(), x)
        return {"loss": D.detach(), "grad": grad}


def _exact_linear(case, s):
    leaf = {n: s[n].detach().double() for n in ("x", "weight", "bias", "residual") if s[n] is not None}
    if case["grad"]:
        for v in leaf.values():
            v.requires_grad_(True)
    with torch.set_grad_enabled(case["grad"]):
        y = torch.matmul(leaf["x"], leaf["weight"].transpose(0, 1))
        if "bias" in leaf:
            y = torch.add(y, leaf["bias"])
        y = {"none": lambda v: v, "relu": torch.relu, "tanh": torch.tanh,
             "silu": torch.nn.functional.silu}[case["act"]](y)
        if "residual" in leaf:
            y = torch.add(y, leaf["residual"])
        out = {"y": y.detach()}
        if case["grad"]:
            out.update(zip(leaf, torch.autograd.grad([y], list(leaf.values()), [s["dy"].double()])))
    return out
