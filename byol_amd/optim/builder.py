"""Optimizer + LR-schedule builders, flag-compatible with the reference
(``/root/reference/main.py:279-344``): the same optimizer map
(rmsprop/adam/adadelta/sgd/momentum/lbfgs/lamb), ``lars_*`` prefix wrapping in
LARS with eps=0.0, linear LR scaling ``lr * global_batch/256`` for the
sgd/momentum family, weight-decay param groups via ``add_weight_decay``, and
warmup->cosine scheduling stepped per epoch."""

import functools

import torch.optim as optim

from .. import layers
from .lars import LARS
from .scheduler import LinearWarmup, Scheduler

__all__ = ["build_optimizer", "build_lr_schedule"]


def build_lr_schedule(optimizer, args, last_epoch=-1):
    if args.lr_update_schedule == "fixed":
        sched = optim.lr_scheduler.LambdaLR(
            optimizer, lambda epoch: 1.0, last_epoch=last_epoch)
    elif args.lr_update_schedule == "cosine":
        total_epochs = args.epochs - args.warmup
        sched = optim.lr_scheduler.CosineAnnealingLR(
            optimizer, T_max=total_epochs, last_epoch=last_epoch)
    else:
        raise NotImplementedError(
            f"lr scheduler {args.lr_update_schedule} not implemented")

    if args.warmup > 0:
        warmup = LinearWarmup(optimizer, warmup_steps=args.warmup,
                              last_epoch=last_epoch)
        sched = Scheduler(sched, warmup)
    return sched


def build_optimizer(model, args, last_epoch=-1):
    """Returns (optimizer, scheduler).  When the model exposes a flat
    parameter space (``finalize()``d BYOL) the LARS wrapper gets it attached
    so its step runs as four fused HIP kernel launches on GPU; LAMB gets it
    so its gradients stay in the buffer that FlatDDP reduces.  LAMB clips by
    ``--clip-norm`` inside its own step."""
    optim_map = {
        "rmsprop": optim.RMSprop,
        "adam": optim.Adam,
        "adadelta": optim.Adadelta,
        "sgd": optim.SGD,
        "momentum": functools.partial(optim.SGD, momentum=0.9),
        "lbfgs": optim.LBFGS,
    }

    params_to_optimize = layers.add_weight_decay(model, args.weight_decay)
    full_opt_name = args.optimizer.lower().strip()
    is_lars = "lars" in full_opt_name
    if full_opt_name == "lamb":
        # bf16 autocast replaces the reference's fp16-only Apex FusedLAMB
        # gate; fp32 parameters on GPU take the fused HIP step
        from .lamb import LAMB
        optim_map["lamb"] = functools.partial(
            LAMB, max_grad_norm=getattr(args, "clip_norm", 0.0))

    opt_name = full_opt_name.split("_")[-1] if is_lars else full_opt_name
    if opt_name not in optim_map:
        raise ValueError(f"unknown optimizer {args.optimizer!r}")

    lr = args.lr
    if opt_name in ("momentum", "sgd"):
        # linear scaling on the GLOBAL batch (batch_size here is per-replica,
        # divided during distributed init — /root/reference/main.py:333-335,725)
        lr = args.lr * (args.batch_size * args.num_replicas / 256)

    opt = optim_map[opt_name](params_to_optimize, lr=lr)

    if is_lars or opt_name == "lamb":
        if is_lars:
            opt = LARS(opt, eps=0.0)
        target = model.module if hasattr(model, "module") else model
        flat_space = getattr(target, "_flat_space", None)
        if flat_space is not None:
            # flat zero_grad always; the fused step additionally verifies the
            # inner optimizer is plain SGD+momentum before engaging
            opt.attach_flat_space(flat_space)

    sched = build_lr_schedule(opt, args, last_epoch=last_epoch)
    return opt, sched
