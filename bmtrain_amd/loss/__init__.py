from .cross_entropy import FusedCrossEntropy, OpFusedCrossEntropy, VPFusedCrossEntropy
from .token_logprobs import OpTokenLogProbs, TokenLogProbs
from .policy import OpPolicyLoss, PolicyLoss
from .preference import OpPreferenceLoss, PreferenceLoss

__all__ = ["FusedCrossEntropy", "OpFusedCrossEntropy", "VPFusedCrossEntropy", "OpTokenLogProbs", "TokenLogProbs",
           "OpPolicyLoss", "PolicyLoss", "OpPreferenceLoss", "PreferenceLoss"]
