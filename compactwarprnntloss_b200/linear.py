"""`fused_linear`: the joint's linear layers on the tensor cores, bias, activation and residual in the epilogue.

    h      = compact_joint(enc, pred, lx, ly)                    # [n_rows, H]
    logits = fused_linear(h, W, b)                               # [n_rows, V]
    loss   = transducer_loss(logits, lx, y, ly, fused_log_softmax=True)

y = act(x W^T + b) + residual with float sums, float16 or bfloat16 throughout (the tensor cores' types; other types are
refused, `torch.nn.functional.linear` has them). The backward pass keeps nothing but the inputs: it multiplies the
pre-activations out again and differentiates the activation in that product's epilogue. The reference project leaves
the layer to its callers. The CUDA library is mandatory (no CPU or PyTorch fallback).
"""
from typing import Optional

import torch

from .scores import core

__all__ = ["fused_linear", "LINEAR_ACTIVATIONS"]

LINEAR_ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "tanh": 2, "silu": 3}


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 residual: Optional[torch.Tensor] = None, *, activation: Optional[str] = None) -> torch.Tensor:
    """act(x W^T + bias) + residual: x [..., n_in], weight [n_out, n_in], bias [n_out], residual [..., n_out], all of
    one type (float16 or bfloat16) on one device. activation: None, 'relu', 'tanh' or 'silu'. Differentiable in all
    four tensors, in reverse mode, once (second and forward-mode derivatives are refused); rows of x and weight may be
    strided."""
    assert activation in LINEAR_ACTIVATIONS
    assert x.dim() >= 1 and weight.dim() == 2 and x.size(-1) == weight.size(1)
    assert x.dtype in (torch.float16, torch.bfloat16), "fused_linear takes float16 and bfloat16"
    lead = x.shape[:-1]
    rows = x.reshape(-1, x.size(-1))
    if bias is not None:
        assert bias.shape == (weight.size(0),)
        bias = bias.contiguous()
    if residual is not None:
        assert residual.shape == lead + (weight.size(0),)
        residual = residual.reshape(-1, weight.size(0)).contiguous()
    y = core._linear(rows, weight, bias, residual, LINEAR_ACTIVATIONS[activation])
    return y if len(lead) == 1 else y.reshape(lead + (weight.size(0),))
