"""Global gradient norm over many tensors, and clipping by it or by value.

``N = sqrt(sum_t ||g_t||^2)`` (or the largest magnitude), then
``g <- min(1, max_norm / (N + 1e-6)) * g``; by value, ``g`` is bounded to
``[-clip_value, clip_value]``.  The reference clips by value before its
optimizer step (its ``main.py:618-624``).

On GPU a list of any length is a few launches of the kernels in
``csrc/gradclip.hip`` and never waits for the host, so the calls can be
captured into a graph; sums are held in 64 bits and joined in a fixed order.
Neighbouring views of one buffer (``FlatParamSpace.flat_grads``) are worked on
as one tensor.  Elsewhere the same values come from elementary torch
operations, the oracle of the tests.  In eager calls the norm's last block
joins the others' sums while they come in, for which places are kept for the
streams used last; in a captured graph a launch of its own joins them.

Gradients are fp32, bf16 or fp16, types may differ within a list; strided
tensors are taken as they are.  Tensors that are written must not overlap:
their ranges of memory, also where views interleave, have to be apart.  NaN and
infinities propagate: an infinite norm scales finite gradients to zero, a NaN
norm makes all of them NaN.  Nothing here is differentiated through.
"""

import bisect
import math
from typing import Sequence

import torch

from . import require_extension

__all__ = ["global_grad_norm", "clip_grads_by_norm_",
           "clip_grads_by_value_"]

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _is_inf(norm_type: float) -> bool:
    norm_type = float(norm_type)
    if norm_type not in (2.0, math.inf):
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    return norm_type == math.inf


def _as_list(grads) -> list:
    return [grads] if isinstance(grads, torch.Tensor) else list(grads)


def _on_gpu(grads: Sequence[torch.Tensor], what: str) -> bool:
    """Whether the HIP kernels take the list (their binding then checks it);
    a list on the CPU is checked here."""
    if getattr(grads[0], "is_cuda", False) \
            or any(getattr(t, "is_cuda", False) for t in grads):
        return True
    for t in grads:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: expected tensors, got {type(t)}")
        if t.dtype not in _DTYPES or t.layout is not torch.strided:
            raise TypeError(f"{what}: expected dense fp32, bf16 or fp16 "
                            f"tensors, got {t.dtype} ({t.layout})")
    return False


class SharedMemoryError(ValueError):
    """Tensors that are written share memory."""


def _reach(t: torch.Tensor):
    """The memory from a tensor's first element to its last."""
    n = 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + n * t.element_size()


def check_writable(grads: Sequence[torch.Tensor], what: str,
                   read: Sequence[torch.Tensor] = ()) -> None:
    """Refuse tensors that are written and share memory, among each other or
    with those that are `read`."""
    ranges = []
    for t in grads:
        if t.numel() == 0:
            continue
        if any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
            raise SharedMemoryError(f"{what}: elements of a tensor share memory "
                                    "(an expanded view); it cannot be written "
                                    "in place")
        ranges.append(_reach(t))
    ranges.sort()
    for a, b in zip(ranges, ranges[1:]):
        if a[1] > b[0]:
            raise SharedMemoryError(f"{what}: a tensor is listed twice, or "
                                    "two share memory")
    for t in read:
        if t.numel() == 0:
            continue
        begin, end = _reach(t)
        at = bisect.bisect_left(ranges, (end, 0))
        if at > 0 and ranges[at - 1][1] > begin:
            raise SharedMemoryError(f"{what}: a tensor that is read shares "
                                    "memory with one that is written")


def _reference_norm(grads, inf: bool) -> torch.Tensor:
    if inf:
        parts = [t.abs().max().double() for t in grads if t.numel()]
        return torch.stack(parts).max() if parts else torch.zeros(()).double()
    parts = [t.double().square().sum() for t in grads]
    return torch.stack(parts).sum().sqrt()


def global_grad_norm(grads: Sequence[torch.Tensor],
                     norm_type: float = 2.0) -> torch.Tensor:
    """The 2-norm (or, with ``math.inf``, the largest magnitude) of all
    elements of all tensors, as one fp32 value on their device.  An empty
    list has norm 0."""
    inf = _is_inf(norm_type)
    grads = _as_list(grads)
    if not grads:
        return torch.zeros(())
    if _on_gpu(grads, "global_grad_norm"):
        return require_extension("global_grad_norm").grad_norm(grads, inf)
    with torch.no_grad():
        return _reference_norm(grads, inf).float()


def clip_grads_by_norm_(grads: Sequence[torch.Tensor], max_norm: float,
                        norm_type: float = 2.0) -> torch.Tensor:
    """Scale all tensors in place by ``min(1, max_norm / (norm + 1e-6))``,
    each value rounded once; returns the norm before clipping.  Tensors stay
    untouched where the factor is 1."""
    inf = _is_inf(norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must be >= 0, got {max_norm}")
    grads = _as_list(grads)
    if not grads:
        return torch.zeros(())
    what = "clip_grads_by_norm_"
    if _on_gpu(grads, what):
        return require_extension(what).grad_clip_norm(grads, max_norm, inf)
    check_writable(grads, what)
    with torch.no_grad():
        norm = _reference_norm(grads, inf)
        factor = (max_norm / (norm + 1e-6)).clamp(max=1.0).float()
        if factor != 1.0:
            for t in grads:
                t.copy_(t.float() * factor)
        return norm.float()


def check_clip_value(clip_value: float) -> float:
    clip_value = float(clip_value)
    if not clip_value >= 0:
        raise ValueError(f"clip_value must be >= 0, got {clip_value}")
    return clip_value


def clip_grads_by_value_(grads: Sequence[torch.Tensor],
                         clip_value: float) -> None:
    """Bound every element to ``[-clip_value, clip_value]`` in place; NaN
    stays."""
    clip_value = check_clip_value(clip_value)
    grads = _as_list(grads)
    if not grads:
        return
    what = "clip_grads_by_value_"
    if _on_gpu(grads, what):
        require_extension(what).grad_clip_value(grads, clip_value)
        return
    check_writable(grads, what)
    with torch.no_grad():
        for t in grads:
            t.copy_(t.float().clamp(-clip_value, clip_value))
