"""Clipped policy loss with KL and entropy terms over padded batches; no counterpart in the reference."""
import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import C
from . import _function as F

_REDUCTIONS = {"mean": 0, "sequence": 1, "sum": 2}


def _tokens_adjacent(t):
    """`t` with its last dimension's elements next to each other (a copy where they are not); None stays None."""
    return t if t is None or t.is_contiguous() or t.size(-1) <= 1 or t.stride(-1) == 1 else t.contiguous()


def constant(t):
    """`t` without its gradient, its tokens next to each other; None stays None."""
    return _tokens_adjacent(t.detach() if t is not None and t.requires_grad else t)


def as_mask(mask):
    """A bool / uint8 mask as it is; anything else as ``mask != 0``."""
    if mask is not None and mask.dtype not in (torch.bool, torch.uint8):
        mask = mask != 0
    return _tokens_adjacent(mask)


class OpPolicyLoss(torch.autograd.Function):
    """Loss and statistics in two launches, both gradients in one."""

    @staticmethod
    def forward(ctx, logprob, entropy, old_logprob, advantages, mask, ref_logprob, clips, kl_coef, entropy_coef, reduction):
        with F.on_device_of(logprob):
            shape, device = logprob.shape, logprob.device
            offsets = F.policy_loss_scratch(*shape, reduction == 1, ctx.needs_input_grad[0])
            loss = torch.empty((), device=device, dtype=torch.float)
            stats = torch.empty(5, device=device, dtype=torch.float)
            scratch = torch.empty(offsets[0], device=device, dtype=torch.float)
            F.policy_loss_forward(logprob, old_logprob, ref_logprob, entropy, advantages, mask, *clips, kl_coef, entropy_coef,
                                  reduction, scratch, offsets, loss, stats)
        ctx.args = (reduction, offsets, entropy_coef, shape, logprob.dtype)
        ctx.mark_non_differentiable(stats)
        ctx.set_materialize_grads(False)                # nothing is to be filled with zeros for the statistics
        ctx.save_for_backward(scratch, mask)
        return loss, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream, _):
        if upstream is None:
            return (None,) * 10
        scratch, mask = ctx.saved_tensors
        reduction, offsets, entropy_coef, shape, dtype = ctx.args
        with F.on_device_of(scratch):
            device = scratch.device
            grad_logprob = torch.empty(shape, device=device, dtype=dtype) if ctx.needs_input_grad[0] else None
            grad_entropy = torch.empty(shape, device=device, dtype=dtype) if ctx.needs_input_grad[1] else None
            F.policy_loss_backward(reduction, scratch, offsets, upstream, mask, entropy_coef, grad_logprob, grad_entropy)
        return grad_logprob, grad_entropy, None, None, None, None, None, None, None, None


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
    influence, and its gradient is 0.  Sums are held in 64 bits; gradients are rounded once to the inputs' type.
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
        assert logprob.dim() == 2, "logprob must be [sequences, tokens]"
        if advantages.dim() == 2 and advantages.size(1) and (advantages.shape != logprob.shape or advantages.stride(1) == 0):
            assert advantages.size(1) == 1 or advantages.shape == logprob.shape, "advantages must be one to a sequence or one to a token"
            advantages = advantages[:, 0]              # one to a sequence: [sequences, 1], or an expanded view
        if advantages.dtype != torch.float32:
            advantages = advantages.float()
        advantages = constant(advantages) if advantages.dim() == 2 else advantages.detach() if advantages.requires_grad else advantages
        return OpPolicyLoss.apply(_tokens_adjacent(logprob), _tokens_adjacent(entropy), constant(old_logprob), advantages,
                                  as_mask(mask), constant(ref_logprob),
                                  (self.clip_low, self.clip_high, self.dual_clip or 0.0), self.kl_coef, self.entropy_coef,
                                  _REDUCTIONS[self.reduction])
