"""MI355X-native replacement for the per-GPU hot path of BMTrain.

Mirrors the reference's public layout for that path only:

    bmtrain_amd.C                   <- bmtrain.C            (compiled launchers)
    bmtrain_amd.optim._function     <- bmtrain.optim._function
    bmtrain_amd.optim.AdamOptimizer / AdamOffloadOptimizer / OptimManager
    bmtrain_amd.loss._function      <- bmtrain.loss._function
    bmtrain_amd.loss.FusedCrossEntropy
"""
import torch as _torch  # noqa: F401  first: the libraries below use the ones that torch brings

from .global_var import config
from . import C
try:
    from . import _tensors  # noqa: F401
except ImportError as e:
    raise ImportError(f"{__path__[0]}/_tensors.so is missing or does not fit this torch: build it with "
                      f"`make -C {__path__[0]}/csrc`") from e
from . import optim
from . import loss

__all__ = ["C", "config", "optim", "loss"]
