"""`distill_loss`: distillation of rows of logits from a teacher's top entries, loss and gradient in one pass.

    t    = token_scores(teacher_logits, top_k=16)                       # or any stored list of entries
    loss = distill_loss(student_logits, t.top_log_probs, t.top_indices) # KL over the list and one class for the rest

A transducer is distilled the same way with two entries per lattice node: the blank and the node's label, everything
else being the rest, weighted by the node posteriors that `analyse` returns. The reference project has no counterpart.
The CUDA library is mandatory (no CPU or PyTorch fallback).
"""
from typing import Literal, Optional

import torch

from .scores import as_rows, core

__all__ = ["distill_loss"]


def distill_loss(x: torch.Tensor, teacher: torch.Tensor, indices: torch.Tensor, *,
                 weight: Optional[torch.Tensor] = None, tail: bool = True, temperature: float = 1.0,
                 reduction: Optional[Literal["mean", "sum", "none"]] = "mean", mean_denominator: float = 0,
                 eager_grad: bool = True) -> torch.Tensor:
    """Divergence of softmax(x / temperature) from the teacher, row by row of `x` [..., V] (f32 / f16 / bf16 / f64).

    teacher, indices   x.shape[:-1] + (K,), 1 <= K <= 32: the teacher's values (float32, float64 for float64 logits)
                       and their tokens (int32). A negative index is an unused slot; a token named twice counts twice;
                       an index of V or more makes the row's loss and gradient NaN, and so does a NaN at a used slot
                       (without a tail, where the values are renormalised, a +inf as well).
    tail               True: the values are log-probabilities, taken at `temperature`; every token that is not listed
                       belongs to one more class. D = sum q (ln q - ln p) over the listed tokens and that class.
                       False: the values are logits or log-probabilities, q = softmax(values / temperature) over the
                       list; D = sum q (ln q - ln p), p over the whole row.
    weight             x.shape[:-1], type of `teacher`: the rows' factors. Rows of weight 0 are not read at all.
    reduction          'mean': sum of the weighted rows / mean_denominator (0: the number of rows); 'sum'; 'none' or
                       None: one value a row. No factor temperature^2 is applied.
    eager_grad         True: with 'mean' and 'sum' the gradient is computed inside the forward call, in the same pass;
                       `backward` only scales it (nothing is touched when the upstream gradient is 1). float16
                       gradients are not scaled, which would lose what lies below their range, but computed once more
                       where the upstream gradient is not 1 (a loss scale); x has to be unchanged until then. False: it
                       is computed by `backward`, and not at all if that never comes; with a loss scale on float16 that
                       is the shorter way.

    Neither teacher nor weight is differentiated. A row whose logits are all -inf contributes nothing. Reverse
    mode, once: second and forward-mode derivatives of x are refused."""
    assert reduction in ["mean", "sum", "none"] or reduction is None
    assert x.dim() >= 1 and x.size(-1) >= 1
    lead = x.shape[:-1]
    assert indices.dtype == torch.int32
    assert teacher.shape == indices.shape and teacher.dim() == x.dim() and teacher.shape[:-1] == lead
    assert teacher.dtype == (torch.float64 if x.dtype == torch.float64 else torch.float32)
    K = indices.size(-1)
    assert 1 <= K <= core.MAX_LIST
    rows = as_rows(x)
    n = rows.size(0)
    teacher = teacher.detach().reshape(n, K).contiguous()
    indices = indices.reshape(n, K).contiguous()
    if weight is not None:
        assert weight.shape == lead and weight.dtype == teacher.dtype
        weight = weight.detach().reshape(n).contiguous()
    reduced = reduction in ("mean", "sum")
    scale = 1.0 / float(mean_denominator or max(n, 1)) if reduction == "mean" else 1.0
    out = core._distill(rows, teacher, indices, weight, tail, temperature, scale, reduced, eager_grad)
    return out if reduced or len(lead) == 1 else out.reshape(lead)
