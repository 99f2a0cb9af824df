"""Loss of paired answers on sums of token log-ratios; no counterpart in the reference."""
import math
from typing import Optional

import torch

from .. import _tensors

_KINDS = {"sigmoid": 0, "ipo": 1, "hinge": 2}


class PreferenceLoss(torch.nn.Module):
    r"""Loss of chosen against rejected answers.  With the sums of a row's tokens under the mask
    :math:`s = \sum_t (\text{logprob} - \text{ref\_logprob})` (divided by their number when ``average``) and
    :math:`h = s_\text{chosen} - s_\text{rejected}`:

    * ``'sigmoid'``: :math:`-(1 - \epsilon) \log\sigma(\beta h) - \epsilon \log\sigma(-\beta h)`, :math:`\epsilon` = ``label_smoothing``
    * ``'ipo'``: :math:`(h - 1 / 2\beta)^2`
    * ``'hinge'``: :math:`\max(0, 1 - \beta h)`

    averaged over the pairs that have a token under the mask in either row (0 when none has).  Returns
    ``(loss, chosen_rewards, rejected_rewards)`` with rewards :math:`\beta s` per pair; the rewards carry no gradient.

    ``forward`` takes ``logprob`` [2 * pairs, tokens] (fp32, fp16 or bf16), the chosen answers in the first half of the
    rows and the rejected ones in the same order in the second, ``ref_logprob`` of the same shape and type (None: 0) and
    ``mask`` (non-zero: the token counts; None: all do).  Sums per row given as [2 * pairs] are taken as one token each.
    What stands under an unset mask, NaN or infinity included, has no influence, and its gradient is 0.  Everything
    between the tokens and the results is held in 64 bits.
    """

    def __init__(self, beta: float = 0.1, kind: str = "sigmoid", label_smoothing: float = 0.0, average: bool = False) -> None:
        super().__init__()
        if not (beta > 0 and math.isfinite(beta)):
            raise ValueError(f"beta must be positive and finite, not {beta}")
        if kind not in _KINDS:
            raise ValueError(f"{kind} is not a valid kind of preference loss")
        if not 0 <= label_smoothing <= 1:
            raise ValueError(f"label_smoothing must be in [0, 1], not {label_smoothing}")
        if label_smoothing and kind != "sigmoid":
            raise ValueError("label_smoothing is for the kind 'sigmoid'")
        self.beta, self.kind, self.label_smoothing, self.average = float(beta), kind, float(label_smoothing), average

    def forward(self, logprob: torch.Tensor, ref_logprob: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None):
        return _tensors.preference_loss(logprob, ref_logprob, mask, _KINDS[self.kind], bool(self.average), self.beta,
                                        self.label_smoothing)
