"""Log-probabilities and entropies of given tokens under logits, without a stored softmax.

The reference has only the cross-entropy (bmtrain/loss/cross_entropy.py); preference and policy losses need the
log-probability of every token as a value with a gradient, often under a temperature and together with the entropy.
"""
import math

import torch
from torch.autograd.function import once_differentiable

from . import _function as F


def _forward(logits, target, ignore_index, temperature, entropy, keep):
    """(logprob or (logprob, entropy), what the backward pass needs if `keep`)."""
    with F.on_device_of(logits):
        layout = F.row_layout(logits)
        device = logits.device
        logprob = torch.empty(target.shape, device=device, dtype=torch.float)
        entropies = torch.empty(target.shape, device=device, dtype=torch.float) if entropy else None
        stats = torch.empty((layout[1], 4), device=device, dtype=torch.float) if keep else None
        F.token_logprobs_forward(layout, target, ignore_index, temperature, logprob, entropies, stats)
    return ((logprob, entropies) if entropy else logprob), stats


class OpTokenLogProbs(torch.autograd.Function):
    """fp32 ``log softmax(logits / temperature)[target]`` per token (and the entropy of every token's distribution).
    Keeps the logits and four numbers per token for the backward pass, which reads the logits once more."""

    @staticmethod
    def forward(ctx, logits: torch.Tensor, target: torch.Tensor, ignore_index: int, temperature: float, entropy: bool):
        target = target.contiguous()
        out, stats = _forward(logits, target, ignore_index, temperature, entropy, ctx.needs_input_grad[0])
        ctx.args = (ignore_index, temperature)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, target, stats)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_logprob, grad_entropy=None):
        if grad_logprob is None and grad_entropy is None:
            return None, None, None, None, None
        logits, target, stats = ctx.saved_tensors
        with F.on_device_of(logits):
            grad = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
            F.token_logprobs_backward(F.row_layout(logits), target, *ctx.args, stats,
                                      None if grad_logprob is None else grad_logprob.contiguous(),
                                      None if grad_entropy is None else grad_entropy.contiguous(), grad)
        return grad, None, None, None, None


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
        assert logits.dim() >= 1 and logits.shape[:-1] == target.shape, "target must have the shape of logits without its last dimension"
        if not (logits.requires_grad and torch.is_grad_enabled()):          # scoring: nothing to remember
            return _forward(logits, target.contiguous(), self.ignore_index, self.temperature, self.entropy, False)[0]
        return OpTokenLogProbs.apply(logits, target, self.ignore_index, self.temperature, self.entropy)
