from .clipping import clip_grad_norm_, clip_grad_value_
from .lars import LARS
from .scheduler import LinearWarmup, Scheduler
from .builder import build_optimizer, build_lr_schedule

__all__ = ["LARS", "LinearWarmup", "Scheduler", "build_optimizer",
           "build_lr_schedule", "clip_grad_norm_", "clip_grad_value_"]
