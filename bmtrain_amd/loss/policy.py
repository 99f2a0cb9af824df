"""Clipped policy loss with KL and entropy terms over padded batches; no counterpart in the reference."""
import math
from typing import Optional

import torch

from .. import _tensors

_REDUCTIONS = {"mean": 0, "sequence": 1, "sum": 2}


class PolicyLoss(torch.nn.Module):
    r"""Clipped policy-gradient loss of answers sampled from an older policy.  Per token, with
    :math:`r = \exp(\text{logprob} - \text{old\_logprob})` and :math:`q = \text{ref\_logprob} - \text{logprob}`:

    .. math::
        \text{policy} &= -\min(r A,\ \operatorname{clip}(r, 1 - \text{clip\_low}, 1 + \text{clip\_high}) A) \\
        \text{kl} &= e^q - 1 - q \\
        \text{loss} &= R(\text{policy}) + \text{kl\_coef}\, R(\text{kl}) - \text{entropy\_coef}\, R(\text{entropy})

    For :math:`A < 0`, ``dual_clip`` = c bounds the policy term by :math:`-c A`.  Returns ``(loss, stats)``: ``stats`` holds
    R(policy), R(kl), R(entropy), R(clipped) and R(old_kl), with clipped = 1 where the policy term has no gradient
    and old_kl = r - 1 - log r, and carries no gradient.

    Args:
        clip_low, clip_high: the clip range around 1 (``clip_high`` defaults to ``clip_low``).
        dual_clip: bound for negative advantages, above 1; None for none.
        kl_coef, entropy_coef: weights of the terms; a term of weight 0 is only measured, one without its input is 0.
        reduction: R is ``'mean'``: the mean over all tokens under the mask, ``'sequence'``: the mean over the sequences
            with at least one such token of their own means, ``'sum'``: the sum.  With nothing under the mask R is 0.

    ``forward`` takes ``logprob`` [sequences, tokens] (fp32, fp16 or bf16), ``old_logprob`` and optionally
    ``ref_logprob`` and ``entropy`` of the same shape and type, ``advantages`` ([sequences], [sequences, 1] or
    [sequences, tokens]) and ``mask`` (non-zero: the token counts; None: all do).  Gradients go to ``logprob`` and
    ``entropy``; the other inputs are constants.  What stands under an unset mask, NaN or infinity included, has no
    influence, and its gradient is 0.  Sums are held in 64 bits; gradients are rounded once to the inputs' type.  A token's
    own terms are fp32: log-probabilities more than 88 apart make its ratio (or e^q) infinite, which a clip or an advantage
    of 0 takes away again.
    """

    def __init__(self, clip_low: float = 0.2, clip_high: Optional[float] = None, dual_clip: Optional[float] = None,
                 kl_coef: float = 0.0, entropy_coef: float = 0.0, reduction: str = "mean") -> None:
        super().__init__()
        clip_high = clip_low if clip_high is None else clip_high
        if not 0 <= clip_low <= 1:
            raise ValueError(f"clip_low must be in [0, 1], not {clip_low}")
        if not (clip_high >= 0 and math.isfinite(clip_high)):
            raise ValueError(f"clip_high must not be negative, nor infinite: {clip_high}")
        if dual_clip is not None and not (dual_clip > 1 and math.isfinite(dual_clip)):
            raise ValueError(f"dual_clip must be above 1, or None: {dual_clip}")
        if reduction not in _REDUCTIONS:
            raise ValueError(f"{reduction} is not a valid value for reduction")
        self.clip_low, self.clip_high, self.dual_clip = float(clip_low), float(clip_high), dual_clip
        self.kl_coef, self.entropy_coef = float(kl_coef), float(entropy_coef)
        self.reduction = reduction

    def forward(self, logprob: torch.Tensor, old_logprob: torch.Tensor, advantages: torch.Tensor,
                mask: Optional[torch.Tensor] = None, ref_logprob: Optional[torch.Tensor] = None,
                entropy: Optional[torch.Tensor] = None):
        return _tensors.policy_loss(logprob, old_logprob, advantages, mask, ref_logprob, entropy, self.clip_low, self.clip_high,
                                    self.dual_clip or 0.0, self.kl_coef, self.entropy_coef, _REDUCTIONS[self.reduction])
