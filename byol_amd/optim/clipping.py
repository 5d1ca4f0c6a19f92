"""Gradient clipping over a model's parameters, by global norm or by value.

The calls of ``torch.nn.utils``, without its ``foreach``: the gradients of all
parameters that have one are handed to the fused operators of
:mod:`byol_amd.ops.grad_clip`.  Those take fp32, bf16 and fp16 gradients on one
device, no two of which reach into each other's memory.  By value, other
gradients are bounded one by one in torch operations; by norm they are refused,
and so are norms other than 2 and inf.  Under data parallelism call them after
the gradients are synchronised (``FlatDDP.finish_grad_sync``): every replica then
computes the same norm from the same values, without another collective.
"""

import torch

from ..ops import clip_grads_by_norm_, clip_grads_by_value_
from ..ops.grad_clip import check_clip_value

__all__ = ["clip_grad_norm_", "clip_grad_value_"]


def _grads(parameters):
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = (p.grad for p in parameters)
    return [g for g in grads if g is not None]


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scale all gradients together so that their norm is at most
    ``max_norm``; returns the norm before clipping (fp32, on the device).

    ``error_if_nonfinite`` raises where that norm is infinite or NaN.  It
    waits for the device, and the gradients are already scaled then; it is
    refused while a graph is captured."""
    grads = _grads(parameters)
    if error_if_nonfinite and torch.cuda.is_available() \
            and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("clip_grad_norm_: error_if_nonfinite waits for "
                           "the device and cannot be captured into a graph")
    norm = clip_grads_by_norm_(grads, max_norm, norm_type)
    if error_if_nonfinite and not torch.isfinite(norm):
        raise RuntimeError(f"the {norm_type}-norm of the gradients is "
                           f"{norm.item()}: they cannot be clipped")
    return norm


@torch.no_grad()
def clip_grad_value_(parameters, clip_value: float) -> None:
    """Bound every gradient value to ``[-clip_value, clip_value]``."""
    clip_value = check_clip_value(clip_value)
    grads = _grads(parameters)
    try:
        clip_grads_by_value_(grads, clip_value)
    except (TypeError, ValueError):
        # a list that the operator does not take; it has written nothing, and
        # to bound a value twice is to bound it
        for g in grads:
            g.clamp_(-clip_value, clip_value)
