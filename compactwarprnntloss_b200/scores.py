"""`token_scores`: log-probabilities of given tokens, entropy and the best alternatives of rows of logits.

    s = token_scores(logits, targets, top_k=8, entropy=True)     # any [..., V] rows, f32 / f16 / bf16 / f64
    s.log_probs, s.entropy, s.top_log_probs, s.top_indices

One pass over the logits; all log-probabilities and the entropy are differentiable with respect to them (one more pass,
which reads the logits and writes their gradient). Confidence scores of a lattice, the alternatives of a beam search
step, and the entries that `distill_loss` takes from a teacher are calls of this function. The reference project has
no counterpart; its callers go through `log_softmax` (test/test.py:19-20). The CUDA library is mandatory (no CPU or
PyTorch fallback).
"""
from typing import NamedTuple, Optional

import torch

try:
    from . import _C as core
except ImportError as e:  # pragma: no cover - exercised only on a box without the built extension
    raise ImportError("compactwarprnntloss_b200._C is not built; run `python -m compactwarprnntloss_b200.build` "
                      "(the package has no CPU or PyTorch fallback)") from e

__all__ = ["token_scores", "TokenScores"]


class TokenScores(NamedTuple):
    """float32 (float64 for float64 logits); None for what was not asked for."""
    log_probs: Optional[torch.Tensor]      # [..., P] (or [...] for targets without the last axis)
    entropy: Optional[torch.Tensor]        # [...]
    top_log_probs: Optional[torch.Tensor]  # [..., k], largest first
    top_indices: Optional[torch.Tensor]    # [..., k] int32, the lower index first among equal logits


def as_rows(x: torch.Tensor) -> torch.Tensor:
    """[..., V] -> [rows, V] with unit column stride, without a copy where the rows lie evenly spaced in memory."""
    if x.dim() == 2 and x.is_contiguous():
        return x
    rows = x.reshape(-1, x.size(-1))
    if (rows.size(1) > 1 and rows.stride(1) != 1) or (rows.size(0) > 1 and rows.stride(0) < rows.size(1)):
        rows = rows.contiguous()
    return rows


def token_scores(x: torch.Tensor, targets: Optional[torch.Tensor] = None, *, top_k: int = 0, entropy: bool = False,
                 temperature: float = 1.0) -> TokenScores:
    """Scores of the rows of `x` [..., V] (logits; log-probabilities do as well) under softmax(x / temperature).

    targets      int32, shape x.shape[:-1] (one token a row) or x.shape[:-1] + (P,), P <= 32; a negative target has no
                 token (log-probability 0, no gradient), one of V or more gives NaN
    top_k        number of best alternatives, 0 <= top_k <= min(V, 32)
    entropy      whether to compute the rows' entropy

    A row whose logits are all -inf has log-probabilities of -inf, entropy 0 and a zero gradient. Reverse mode, once:
    second and forward-mode derivatives are refused."""
    assert x.dim() >= 1 and x.size(-1) >= 1
    assert targets is not None or top_k > 0 or entropy, "nothing asked for"
    lead = x.shape[:-1]
    rows = as_rows(x)
    wanted = None
    if targets is not None:
        assert targets.dtype == torch.int32
        assert targets.shape == lead or targets.shape[:-1] == lead, "targets must match the rows of x"
        per_row = targets.size(-1) if targets.dim() > len(lead) else 1
        wanted = targets.reshape(rows.size(0), per_row).contiguous()
    lp, ent, top, index = core._token_scores(rows, wanted, top_k, entropy, temperature)
    if len(lead) != 1:
        ent = None if ent is None else ent.reshape(lead)
        top, index = (None if t is None else t.reshape(lead + (top_k,)) for t in (top, index))
    if lp is not None and lp.shape != targets.shape:
        lp = lp.reshape(targets.shape)
    return TokenScores(lp, ent, top, index)
