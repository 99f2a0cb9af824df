from .adam import AdamOptimizer
from .adam_offload import AdamOffloadOptimizer
from .clip import clip_grads
from .optim_manager import OptimManager

__all__ = ["AdamOptimizer", "AdamOffloadOptimizer", "OptimManager", "clip_grads"]
