"""Log-probabilities and entropies of given tokens under logits, without a stored softmax.

The reference has only the cross-entropy (bmtrain/loss/cross_entropy.py); preference and policy losses need the
log-probability of every token as a value with a gradient, often under a temperature and together with the entropy.
"""
import math

import torch

from .. import _tensors


class TokenLogProbs(torch.nn.Module):
    r"""Log-probability of every token ``target`` (shape ``[...]``) under ``logits`` (shape ``[..., C]``):

    .. math::
        \log p_n = \frac{x_{n,y_n}}{T} - \log \sum_c \exp\frac{x_{n,c}}{T}, \qquad
        H_n = -\sum_c p_{n,c} \log p_{n,c}

    with a gradient for the logits of both.  fp32, fp16 or bf16 logits; the results are fp32, sums and exponents too,
    and the gradient is rounded to the logits' type once.  Up to three dimensions with any strides between rows
    (``logits[:, :-1]`` is not copied); other layouts are copied first.

    Args:
        ignore_index: target whose token gets the results 0 and a gradient of 0; its logits are not read, whatever they hold.
        temperature: :math:`T`, positive.
        entropy: return ``(logprob, entropy)`` instead of ``logprob``.

    A token whose upstream gradients are 0 gets a gradient of exactly 0 without its logits being read again.  Another
    target outside ``[0, C)`` gives a log-probability of NaN and no one-hot term in the gradient.  Classes of logit
    ``-inf`` have probability 0 and add nothing to the entropy; a row with ``+inf`` or NaN, or with ``-inf`` only, gives NaN.

    Example::

        >>> logprobs = bmtrain_amd.loss.TokenLogProbs(entropy=True)
        >>> logp, entropy = logprobs(logits[:, :-1], tokens[:, 1:])
    """

    def __init__(self, ignore_index: int = -100, temperature: float = 1.0, entropy: bool = False) -> None:
        super().__init__()
        if not (temperature > 0 and math.isfinite(temperature)):
            raise ValueError(f"temperature must be positive and finite, not {temperature}")
        self.ignore_index = ignore_index
        self.temperature = float(temperature)
        self.entropy = entropy

    def forward(self, logits: torch.Tensor, target: torch.Tensor):
        logprob, entropy = _tensors.token_logprobs(logits, target, self.ignore_index, self.temperature, self.entropy)
        return (logprob, entropy) if self.entropy else logprob
