"""Global norm and clipping over a list of gradients without a host read; for programs that step their gradients
without :class:`OptimManager` (whose ``clip_grad_norm`` uses the same scaling kernel), or keep fp32 accumulators
(bmtrain/optim/optim_manager.py:158-200 is the reference's clipping)."""
import math
from typing import Optional, Sequence

import torch

from .. import _tensors


def clip_grads(grads: Sequence[torch.Tensor], max_norm: float, norm_type=2.0, eps: float = 1e-6, scale: float = 1.0,
               out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    r"""Clips ``grads`` to the global norm ``max_norm`` and returns their norm before clipping, a 0-dim fp32 tensor on
    their device:

    .. math::
        n = \Big(\sum_k \sum_i g_{k,i}^2\Big)^{1/2} \text{ or } \max |g_{k,i}|, \qquad
        c = \frac{\text{max\_norm} \cdot \text{scale}}{n + \text{eps}}, \qquad
        \text{out} = c < 1\ ?\ c\, g : g

    Args:
        grads: fp32, fp16 and bf16 tensors on one GPU, in any mixture; each dense (contiguous in some order of its dimensions).
        max_norm: the largest norm of the unscaled gradients.
        norm_type: 2.0, or ``math.inf`` / ``'inf'`` for the largest magnitude.
        scale: the loss scale the gradients carry; the returned norm is divided by it.
        out: tensors of as many elements as the gradients (of their shapes and strides, where those are not contiguous),
            of any of the three types, that receive the clipped gradients - fp32 accumulators into the 16-bit gradients
            of an optimizer, say; ``None`` clips in place.  An output may be its own gradient but share memory with
            nothing else of the call (``RuntimeError``; the gradients themselves are not listed twice either when they
            are clipped in place).  A leaf that requires a gradient is written under ``torch.no_grad()`` only.

    Nothing is read by the host, so the call can be captured into a graph.  Squares are summed in 64 bits in a fixed
    order, the product with the factor is fp32 and rounded to the output's type once.  With an infinite norm the factor
    is 0 (infinities turn into NaN); a NaN norm leaves the gradients as they are.  Gradients of ``None`` are skipped,
    together with their output.
    """
    grads = list(grads)
    outs = grads if out is None else list(out)
    if len(outs) != len(grads):
        raise ValueError(f"{len(grads)} gradients but {len(outs)} outputs")
    if type(None) in set(map(type, grads)):
        outs = [o for g, o in zip(grads, outs) if g is not None]
        grads = [g for g in grads if g is not None]
        outs = grads if out is None else outs
    if type(None) in set(map(type, outs)):
        raise ValueError("a gradient without an output")
    if not (max_norm >= 0 and eps >= 0 and scale > 0 and math.isfinite(scale)):
        raise ValueError(f"max_norm and eps must not be negative and scale must be positive: {max_norm}, {eps}, {scale}")
    use_max = norm_type in ("inf", math.inf)
    if not use_max and norm_type != 2:
        raise ValueError(f"norm_type must be 2 or inf, not {norm_type}")
    if not grads:
        return torch.zeros((), dtype=torch.float32, device="cuda" if torch.cuda.is_available() else "cpu")
    return _tensors.clip_grads(grads, None if out is None else outs, float(max_norm), use_max, float(eps), float(scale))
