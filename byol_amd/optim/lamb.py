"""LAMB optimizer (the reference takes one from another package, its
``main.py:324-326``): the LAMB update (You et al., arXiv:1904.00962) —
Adam-style moments, then a per-layer trust ratio ``||p|| / ||update||`` scales
the step.

fp32 parameters on a GPU take the fused step (``byol_amd/ops/lamb_step.py``):
all tensors together, without a host wait.  Other parameters are updated one by
one in torch operations.  ``max_grad_norm`` clips the global norm of all
gradients inside the step; the gradients themselves are left as they are.
"""

import torch
from torch.optim.optimizer import Optimizer

__all__ = ["LAMB"]

_GRAD_DTYPES = (torch.float32, torch.bfloat16, torch.float16)

def _norm_of(grads) -> torch.Tensor:
    """The 2-norm of all gradients; those that the operator does not take in
    one list (other types, several devices) are joined in fp64."""
    from ..ops import global_grad_norm
    device = grads[0].device
    if len({g.device for g in grads}) == 1 \
            and {g.dtype for g in grads} <= set(_GRAD_DTYPES):
        return global_grad_norm(grads)
    return torch.stack([g.double().square().sum().to(device)
                        for g in grads]).sum().sqrt()


def _on(norm, device):
    """The norm as the fused step reads it."""
    return None if norm is None else norm.to(device, torch.float32)


class LAMB(Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-6,
                 weight_decay=0.0, max_grad_norm=0.0):
        if not max_grad_norm >= 0:
            raise ValueError(f"invalid max_grad_norm: {max_grad_norm}")
        defaults = dict(lr=lr, betas=betas, eps=eps,
                        weight_decay=weight_decay)
        super().__init__(params, defaults)
        self.defaults["max_grad_norm"] = float(max_grad_norm)

    @property
    def max_grad_norm(self) -> float:
        """Bound on the global gradient norm; 0 means no clipping."""
        return self.defaults.get("max_grad_norm", 0.0)

    def attach_flat_space(self, flat_space):
        """Keep gradients as views of the model's flat buffer: the kernels
        pass over it as one tensor, and
        :class:`~byol_amd.parallel.FlatDDP` reduces it.

        ``zero_grad`` still leaves no gradient behind, and ``step`` skips the
        parameters that no backward pass reaches.  Where FlatDDP reduces the
        buffer a parameter may have its gradient from another rank, so there
        the gradients are cleared in place, and one that no rank reaches
        counts as zeros: its update is the weight decay alone, which the trust
        ratio scales to ``lr * |p|`` whatever the decay is."""
        flat_space.verify()
        self._flat_space = flat_space

    def zero_grad(self, set_to_none: bool = True):
        space = getattr(self, "_flat_space", None)
        if space is None:
            super().zero_grad(set_to_none=set_to_none)
        elif set_to_none and not space.reduced:
            space.drop_grads()
        else:
            space.zero_grads()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups = []
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            if params:
                groups.append((group, params, [p.grad for p in params]))
        if any(params[0].is_cuda for _, params, _ in groups) \
                and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("LAMB.step cannot be captured into a graph: "
                               "its step count and learning rate are host "
                               "values")
        norm = None
        if self.max_grad_norm > 0 and groups:
            norm = _norm_of([g for _, _, gs in groups for g in gs])
        fused = {}
        for group, params, grads in groups:
            states = [self._state_of(p) for p in params]
            lists = (params, grads, [s["exp_avg"] for s in states],
                     [s["exp_avg_sq"] for s in states])
            if self._fit_one_step(lists, states):
                self._add_to_step(fused, group, lists, states)
            else:
                self._step_each(fused, group, params, states, norm)
        if fused:
            from ..ops import fused_lamb_step
            from ..ops.grad_clip import SharedMemoryError
            for (_, _, step, lr, betas, eps), lists in fused.items():
                try:
                    fused_lamb_step(*lists[:4], step=step, lr=lr, betas=betas,
                                    eps=eps, weight_decay=lists[4],
                                    max_grad_norm=self.max_grad_norm,
                                    grad_norm=_on(norm, lists[0][0].device))
                except SharedMemoryError:  # nothing has been written
                    for p, state, group in zip(lists[0], *lists[5:]):
                        self._step_one(p, state, group, norm)
                    continue
                # counted when taken: a refused step leaves the count
                for state in lists[5]:
                    state["step"] = step
        return loss

    def _state_of(self, p):
        state = self.state[p]
        if len(state) == 0:
            state["step"] = 0
            state["exp_avg"] = torch.zeros_like(p)
            state["exp_avg_sq"] = torch.zeros_like(p)
        return state

    @staticmethod
    def _fit_one_step(lists, states) -> bool:
        """Whether a group's tensors can all go into the same fused step.
        The one rule for it, for a single tensor too."""
        if not lists[0][0].is_cuda:
            return False
        from ..ops import require_extension
        return require_extension("LAMB.step").lamb_fits(*lists) \
            and len({s["step"] for s in states}) == 1

    @staticmethod
    def _add_to_step(fused, group, lists, states):
        params, grads = lists[:2]
        key = (params[0].device, grads[0].dtype, states[0]["step"] + 1,
               group["lr"], tuple(group["betas"]), group["eps"])
        all_lists = fused.setdefault(key, tuple([] for _ in range(7)))
        for values, more in zip(all_lists, lists):
            values.extend(more)
        all_lists[4].extend([max(group["weight_decay"], 0.0)] * len(params))
        all_lists[5].extend(states)
        all_lists[6].extend([group] * len(params))

    def _step_each(self, fused, group, params, states, norm):
        for p, state in zip(params, states):
            if p.is_cuda and p.dtype == torch.float32 and (
                    p.is_contiguous() or p.is_contiguous(
                        memory_format=torch.channels_last)):
                for name in ("exp_avg", "exp_avg_sq"):
                    # a checkpoint of another memory format or type
                    if state[name].stride() != p.stride() \
                            or state[name].dtype != p.dtype:
                        state[name] = torch.empty_like(p).copy_(state[name])
            lists = ([p], [p.grad], [state["exp_avg"]], [state["exp_avg_sq"]])
            if self._fit_one_step(lists, [state]):
                self._add_to_step(fused, group, lists, [state])
            else:
                self._step_one(p, state, group, norm)

    def _step_one(self, p, state, group, norm):
        beta1, beta2 = group["betas"]
        grad = p.grad
        if norm is not None:
            # not in a half-precision gradient's own type: fp16 has no factor
            # below 3e-8, and bf16 would round twice
            kind = torch.promote_types(grad.dtype, torch.float32)
            grad = grad.to(kind) * (
                self.max_grad_norm / (norm.double() + 1e-6)) \
                .clamp(max=1.0).to(grad.device, kind)
        exp_avg, exp_avg_sq = state["exp_avg"], state["exp_avg_sq"]
        exp_avg.mul_(beta1).add_(grad, alpha=1 - beta1)
        exp_avg_sq.mul_(beta2).addcmul_(grad, grad, value=1 - beta2)
        state["step"] += 1
        bias1 = 1 - beta1 ** state["step"]
        bias2 = 1 - beta2 ** state["step"]
        update = (exp_avg / bias1) / (
            (exp_avg_sq / bias2).sqrt().add_(group["eps"]))
        if group["weight_decay"] > 0:
            update.add_(p, alpha=group["weight_decay"])
        w_norm = p.norm()
        u_norm = update.norm()
        trust = torch.where(
            (w_norm > 0) & (u_norm > 0),
            w_norm / u_norm, torch.ones_like(w_norm))
        p.add_(update, alpha=-group["lr"] * float(trust))
