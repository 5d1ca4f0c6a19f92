"""One LAMB step over a list of parameters (You et al., arXiv:1904.00962).

With ``g' = c g`` (``c`` the global-norm clipping factor, or 1)::

    m = b1 m + (1 - b1) g'          v = b2 v + (1 - b2) g'^2
    u = (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps) + wd p
    p = p - lr r u,   r = ||p|| / ||u|| of the tensor (1 if either is 0)

The reference takes an external fused optimizer for this (its
``main.py:324-326``).  On GPU a step is one pass of the kernels in
``csrc/lamb.hip`` over all tensors together and never waits for the host;
clipping costs one more reading of the gradients, which stay as they are.
Elsewhere the same step runs tensor by tensor in torch operations.
"""

from typing import Optional, Sequence, Tuple, Union

import torch

from . import require_extension
from .grad_clip import SharedMemoryError, check_writable, global_grad_norm

__all__ = ["fused_lamb_step"]


def _check(name: str, value: float, ok: bool) -> None:
    if not ok:
        raise ValueError(f"fused_lamb_step: invalid {name}: {value}")


@torch.no_grad()
def fused_lamb_step(params: Sequence[torch.Tensor],
                    grads: Sequence[torch.Tensor],
                    exp_avgs: Sequence[torch.Tensor],
                    exp_avg_sqs: Sequence[torch.Tensor], *, step: int,
                    lr: float, betas: Tuple[float, float] = (0.9, 0.999),
                    eps: float = 1e-6,
                    weight_decay: Union[float, Sequence[float]] = 0.0,
                    max_grad_norm: float = 0.0,
                    grad_norm: Optional[torch.Tensor] = None) -> None:
    """Update parameters and moments in place.

    ``step`` counts from 1 (the step that is taken now).  ``weight_decay`` is
    one number or one for each tensor.  With ``max_grad_norm > 0`` the
    gradients count as scaled by ``min(1, max_grad_norm / (norm + 1e-6))``;
    the norm is ``grad_norm`` (one fp32 value on the device, from
    ``global_grad_norm``) or, without it, that of ``grads``.

    Parameters and moments are dense fp32 tensors of one layout each, no two
    of which share memory; gradients do not share theirs and are fp32,
    bf16 or fp16, all of one type.
    ``step`` and ``lr`` are numbers of the host, so the call refuses to be
    captured into a graph, which would repeat them."""
    b1, b2 = (float(b) for b in betas)
    step, lr, eps = int(step), float(lr), float(eps)
    max_grad_norm = float(max_grad_norm)
    _check("step", step, step >= 1)
    _check("betas", betas, 0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0)
    _check("eps", eps, eps >= 0.0)
    _check("max_grad_norm", max_grad_norm, max_grad_norm >= 0.0)
    params, grads = list(params), list(grads)
    exp_avgs, exp_avg_sqs = list(exp_avgs), list(exp_avg_sqs)
    if isinstance(weight_decay, (int, float)):
        decay = [float(weight_decay)] * len(params)
    else:
        decay = [float(w) for w in weight_decay]
    if not len(params) == len(grads) == len(exp_avgs) == len(exp_avg_sqs) \
            == len(decay):
        raise ValueError("fused_lamb_step: lists of different lengths")
    if not params:
        return
    on_gpu = any(p.is_cuda for p in params)
    if on_gpu and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("fused_lamb_step cannot be captured into a graph: "
                           "its step count and learning rate are host values")
    if max_grad_norm > 0 and grad_norm is None:
        grad_norm = global_grad_norm(grads)
    if max_grad_norm == 0:
        grad_norm = None
    if on_gpu:
        if not require_extension("fused_lamb_step").lamb_step(
                params, grads, exp_avgs, exp_avg_sqs, decay, step, lr, b1, b2,
                eps, max_grad_norm, grad_norm, refuse_shared=False):
            raise SharedMemoryError(
                "fused_lamb_step: a tensor is listed twice, or two share "
                "memory")
        return
    _reference_step(params, grads, exp_avgs, exp_avg_sqs, decay, step, lr,
                    b1, b2, eps, max_grad_norm, grad_norm)


def _reference_step(params, grads, exp_avgs, exp_avg_sqs, decay, step, lr,
                    b1, b2, eps, max_grad_norm, grad_norm) -> None:
    for p, g, m, v in zip(params, grads, exp_avgs, exp_avg_sqs):
        if not p.dtype == m.dtype == v.dtype == torch.float32:
            raise TypeError("fused_lamb_step: parameters and moments must be "
                            "fp32")
        if not p.shape == g.shape == m.shape == v.shape:
            raise ValueError("fused_lamb_step: a gradient or moment has "
                             "another shape than its parameter")
    devices = {t.device for ts in (params, grads, exp_avgs, exp_avg_sqs)
               for t in ts}
    if len(devices) > 1:
        raise ValueError("fused_lamb_step: expected all tensors on one "
                         f"device, got {sorted(map(str, devices))}")
    check_writable([*params, *exp_avgs, *exp_avg_sqs], "fused_lamb_step",
                   read=grads)
    factor = 1.0
    if grad_norm is not None:
        factor = (max_grad_norm / (grad_norm.double() + 1e-6)) \
            .clamp(max=1.0).float()
    for p, g, m, v, wd in zip(params, grads, exp_avgs, exp_avg_sqs, decay):
        g = g.float() * factor
        m.mul_(b1).add_(g, alpha=1 - b1)
        v.mul_(b2).addcmul_(g, g, value=1 - b2)
        u = (m / (1 - b1 ** step)).div_(
            (v / (1 - b2 ** step)).sqrt_().add_(eps)).add_(p, alpha=wd)
        p_norm, u_norm = p.norm(), u.norm()
        ratio = torch.where((p_norm > 0) & (u_norm > 0), p_norm / u_norm,
                            torch.ones_like(p_norm))
        p.sub_(u * (lr * ratio))
