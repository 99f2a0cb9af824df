from .cross_entropy import FusedCrossEntropy, OpFusedCrossEntropy, VPFusedCrossEntropy
from .token_logprobs import TokenLogProbs
from .policy import PolicyLoss
from .preference import PreferenceLoss

__all__ = ["FusedCrossEntropy", "OpFusedCrossEntropy", "VPFusedCrossEntropy", "TokenLogProbs", "PolicyLoss",
           "PreferenceLoss"]
