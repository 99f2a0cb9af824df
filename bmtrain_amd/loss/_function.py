"""Argument checking and dispatch in front of the overflow-check and cross-entropy
launchers.  Same functions, argument order and exception types as
bmtrain/loss/_function.py (ValueError for a dtype that is not 16-bit,
NotImplementedError when bf16 is unavailable, AssertionError for the rest).
"""
import torch

from .. import C


def _current_stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _on_gpu(t: torch.Tensor) -> bool:
    return t.is_contiguous() and t.is_cuda


def _pick(op: str, dtype: torch.dtype, fp16, bf16):
    if dtype == torch.float16:
        return fp16
    if dtype == torch.bfloat16:
        if not C.is_bf16_supported():
            raise NotImplementedError("bfloat16 is not supported on current GPU")
        return bf16
    raise ValueError(f"{op} not supported for dtype {dtype}")


def has_inf_nan(g_half: torch.Tensor, out: torch.Tensor) -> None:
    """Sets the uint8 flag ``out`` to 1 when ``g_half`` holds an inf or NaN; leaves it
    alone otherwise, so one flag can be accumulated over many tensors
    (bmtrain/loss/_function.py:7-24).  The reference allocates and zeroes a 1024-byte
    scratch tensor per call for its two-kernel reduction; the single-kernel scan here
    needs none, so none is allocated."""
    assert out.dtype == torch.uint8, "out must be a uint8 tensor"
    assert _on_gpu(g_half), "g_fp16 must be contiguous and on cuda"
    assert _on_gpu(out), "out must be contiguous and on cuda"
    launcher = _pick("has_inf_nan", g_half.dtype, C.has_nan_inf_fp16_launcher, C.has_nan_inf_bf16_launcher)
    launcher(g_half.numel(), g_half.data_ptr(), 0, out.data_ptr(), _current_stream())


def cross_entropy_forward(m: int, n: int, input: torch.Tensor, target: torch.Tensor, softmax: torch.Tensor,
                          output: torch.Tensor, ignore_index: int) -> None:
    """softmax[m, n] and per-row loss output[m] from logits input[m, n]
    (bmtrain/loss/_function.py:27-78)."""
    for name, t in (("input", input), ("target", target), ("softmax", softmax), ("output", output)):
        assert _on_gpu(t), f"{name} must be contiguous and on cuda"
    assert target.dtype == torch.int32, "target must be an int tensor"
    assert output.dtype == torch.float32, "output must be a float tensor"
    assert input.numel() == softmax.numel(), "input and softmax must have the same number of elements"
    assert target.numel() == output.numel(), "target and output must have the same number of elements"
    assert softmax.dtype == input.dtype, "input and softmax must have the same dtype"
    assert input.numel() == m * n and target.numel() == m, "m, n must describe input and target"
    launcher = _pick("cross_entropy_forward", input.dtype,
                     C.cross_entropy_forward_fp16_launcher, C.cross_entropy_forward_bf16_launcher)
    launcher(m, n, input.data_ptr(), target.data_ptr(), softmax.data_ptr(), output.data_ptr(), ignore_index,
             _current_stream())


def cross_entropy_backward_inplace(m: int, n: int, grad_output: torch.Tensor, target: torch.Tensor, x: torch.Tensor,
                                   ignore_index: int) -> None:
    """Turns the stored softmax ``x`` into the logits gradient in place
    (bmtrain/loss/_function.py:81-115)."""
    for name, t in (("grad_output", grad_output), ("target", target), ("x", x)):
        assert _on_gpu(t), f"{name} must be contiguous and on cuda"
    assert grad_output.dtype == torch.float32, "grad_output must be a float tensor"
    assert target.dtype == torch.int32, "target must be an int tensor"
    assert target.numel() == grad_output.numel(), "target and grad_output must have the same number of elements"
    assert x.numel() == m * n and target.numel() == m, "m, n must describe x and target"
    launcher = _pick("cross_entropy_backward", x.dtype,
                     C.cross_entropy_backward_inplace_fp16_launcher, C.cross_entropy_backward_inplace_bf16_launcher)
    launcher(m, n, grad_output.data_ptr(), target.data_ptr(), x.data_ptr(), ignore_index, _current_stream())


def fused_sumexp(logits: torch.Tensor, max_logits: torch.Tensor) -> torch.Tensor:
    """Row sums of exp(logits - max_logits[:, None]) as fp32 (bmtrain/loss/_function.py:118-147)."""
    assert _on_gpu(logits), "logits must be contiguous and on cuda"
    assert _on_gpu(max_logits), "max_logits must be contiguous and on cuda"
    assert max_logits.dtype == torch.float32, "max_logits must be float tensor"
    assert max_logits.size(0) == logits.size(0), "max_logits must have same size(0) as logits"
    m, n = logits.size(0), logits.size(1)
    sum_exp_logits = torch.empty(m, dtype=torch.float32, device=logits.device)
    launcher = _pick("fused_sumexp", logits.dtype, C.fused_sumexp_fp16_launcher, C.fused_sumexp_bf16_launcher)
    launcher(m, n, logits.data_ptr(), max_logits.data_ptr(), sum_exp_logits.data_ptr(), _current_stream())
    return sum_exp_logits


def fused_softmax_inplace(logits: torch.Tensor, max_logits: torch.Tensor, sum_exp_logits: torch.Tensor) -> None:
    """logits <- exp(logits - max) / sum, row-wise and in place (bmtrain/loss/_function.py:150-182)."""
    for name, t in (("logits", logits), ("max_logits", max_logits), ("sum_exp_logits", sum_exp_logits)):
        assert _on_gpu(t), f"{name} must be contiguous and on cuda"
    assert max_logits.dtype == torch.float32, "max_logits must be float tensor"
    assert sum_exp_logits.dtype == torch.float32, "sum_exp_logits must be float tensor"
    assert max_logits.size(0) == logits.size(0), "max_logits must have same size(0) as logits"
    assert sum_exp_logits.size(0) == logits.size(0), "sum_exp_logits must have same size(0) as logits"
    m, n = logits.size(0), logits.size(1)
    launcher = _pick("fused_softmax_inplace", logits.dtype,
                     C.fused_softmax_inplace_fp16_launcher, C.fused_softmax_inplace_bf16_launcher)
    launcher(m, n, logits.data_ptr(), max_logits.data_ptr(), sum_exp_logits.data_ptr(), _current_stream())


def loss_reduce_forward(losses: torch.Tensor, target: torch.Tensor, weight, n_classes: int, ignore_index: int,
                        mean: bool, result: torch.Tensor, weight_sum: torch.Tensor) -> None:
    """``result = sum_r w_r * losses[r]`` (divided by ``weight_sum = sum_r w_r`` when ``mean``) with
    ``w_r = 0`` for ignored rows and otherwise ``weight[target[r]]`` (1 without ``weight``): the reduction that
    bmtrain/loss/cross_entropy.py:243-260 writes in torch operations, in one launch."""
    for name, t in (("losses", losses), ("target", target), ("result", result), ("weight_sum", weight_sum)):
        assert _on_gpu(t), f"{name} must be contiguous and on cuda"
    assert losses.dtype == torch.float32 and result.dtype == torch.float32 and weight_sum.dtype == torch.float32
    assert target.dtype == torch.int32, "target must be an int tensor"
    assert target.numel() == losses.numel(), "target and losses must have the same number of elements"
    if weight is not None:
        assert _on_gpu(weight) and weight.dtype == torch.float32 and weight.numel() == n_classes, \
            "weight must be a contiguous float tensor of n_classes elements on cuda"
    C.cross_entropy_reduce_forward_launcher(losses.numel(), losses.data_ptr(), target.data_ptr(),
                                            weight.data_ptr() if weight is not None else 0, n_classes, ignore_index,
                                            int(mean), result.data_ptr(), weight_sum.data_ptr(), _current_stream())


def loss_reduce_backward(target: torch.Tensor, weight, n_classes: int, ignore_index: int, mean: bool,
                         weight_sum: torch.Tensor, upstream: torch.Tensor, grad_rows: torch.Tensor) -> None:
    """``grad_rows[r] = (upstream / weight_sum if mean else upstream) * w_r``: what autograd derives from the
    torch operations of bmtrain/loss/cross_entropy.py:243-260, in one launch."""
    for name, t in (("target", target), ("weight_sum", weight_sum), ("upstream", upstream), ("grad_rows", grad_rows)):
        assert _on_gpu(t), f"{name} must be contiguous and on cuda"
    assert upstream.dtype == torch.float32 and upstream.numel() == 1, "upstream must be one float"
    assert weight_sum.dtype == torch.float32 and grad_rows.dtype == torch.float32
    assert target.dtype == torch.int32 and target.numel() == grad_rows.numel()
    if weight is not None:
        assert _on_gpu(weight) and weight.dtype == torch.float32 and weight.numel() == n_classes
    C.cross_entropy_reduce_backward_launcher(target.numel(), target.data_ptr(),
                                             weight.data_ptr() if weight is not None else 0, n_classes, ignore_index,
                                             int(mean), weight_sum.data_ptr(), upstream.data_ptr(), grad_rows.data_ptr(),
                                             _current_stream())


# ---- token log-probabilities, policy and preference losses: fp32, fp16 and bf16 alike --------------------------------

_TYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _type_code(op: str, dtype: torch.dtype) -> int:
    if dtype not in _TYPE_CODES:
        raise ValueError(f"{op} not supported for dtype {dtype}")
    return _TYPE_CODES[dtype]


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _together(first: torch.Tensor, **others) -> None:
    """All tensors on the GPU of the first one."""
    assert first.is_cuda, "tensors must be on cuda"
    for name, t in others.items():
        assert t is None or t.device == first.device, f"{name} must be on the same device as the first tensor"


def on_device_of(t: torch.Tensor):
    """The context in which launches go to the device of `t` and its current stream."""
    assert t.is_cuda, "tensors must be on cuda"
    return torch.cuda.device(t.device)


def row_layout(logits: torch.Tensor):
    """(logits, rows, n, inner, outer stride, inner stride) of logits [..., n]: at most two strides lead from row to row
    and the classes lie next to each other; a tensor laid out otherwise is copied first."""
    n = logits.size(-1)
    if logits.dim() > 3 or (n > 1 and logits.stride(-1) != 1):
        logits = logits.contiguous()
        rows = logits.numel() // n if n else 0
        return logits, rows, n, max(rows, 1), 0, n
    if logits.dim() == 1:
        return logits, 1, n, 1, 0, n
    if logits.dim() == 2:
        return logits, logits.size(0), n, max(logits.size(0), 1), 0, logits.stride(0)
    return logits, logits.size(0) * logits.size(1), n, max(logits.size(1), 1), logits.stride(0), logits.stride(1)


def token_logprobs_forward(layout, target: torch.Tensor, ignore_index: int, temperature: float, logprob: torch.Tensor,
                           entropy, stats) -> None:
    """``logprob`` (and ``entropy``, or None) of the tokens ``target`` under the logits of ``layout`` (``row_layout``);
    ``stats`` (fp32, 4 per row, or None) keeps what ``token_logprobs_backward`` needs."""
    logits, rows, n, inner, outer_stride, inner_stride = layout
    _together(logits, target=target, logprob=logprob, entropy=entropy, stats=stats)
    code = _type_code("token_logprobs", logits.dtype)
    assert target.dtype in (torch.int32, torch.int64), "target must be an int or long tensor"
    assert target.is_contiguous() and target.numel() == rows, "target must be contiguous, one class to a row of the logits"
    assert n > 0 or rows == 0, "logits must have at least one class"
    for t in (logprob, entropy):
        assert t is None or (t.is_contiguous() and t.dtype == torch.float32 and t.numel() == rows)
    assert stats is None or (stats.is_contiguous() and stats.dtype == torch.float32 and stats.numel() == 4 * rows)
    C.token_logprobs_forward_launcher(rows, n, inner, outer_stride, inner_stride, logits.data_ptr(), code, target.data_ptr(),
                                      8 * target.element_size(), ignore_index, temperature, logprob.data_ptr(), _ptr(entropy),
                                      _ptr(stats), _current_stream())


def token_logprobs_backward(layout, target: torch.Tensor, ignore_index: int, temperature: float, stats: torch.Tensor,
                            grad_logprob, grad_entropy, grad: torch.Tensor) -> None:
    """``grad`` (contiguous, the logits' shape and type) from the gradients of the log-probabilities and entropies
    (contiguous fp32, either may be None)."""
    logits, rows, n, inner, outer_stride, inner_stride = layout
    _together(logits, target=target, stats=stats, grad_logprob=grad_logprob, grad_entropy=grad_entropy, grad=grad)
    for t in (grad_logprob, grad_entropy):
        assert t is None or (t.is_contiguous() and t.dtype == torch.float32 and t.numel() == rows)
    assert stats.is_contiguous() and stats.dtype == torch.float32 and stats.numel() == 4 * rows
    assert grad.is_contiguous() and grad.dtype == logits.dtype and grad.numel() == rows * n
    assert target.is_contiguous() and target.numel() == rows and target.dtype in (torch.int32, torch.int64)
    C.token_logprobs_backward_launcher(rows, n, inner, outer_stride, inner_stride, logits.data_ptr(),
                                       _type_code("token_logprobs", logits.dtype), target.data_ptr(),
                                       8 * target.element_size(), ignore_index, temperature, stats.data_ptr(),
                                       _ptr(grad_logprob), _ptr(grad_entropy), grad.data_ptr(), _current_stream())


def _row(t):
    """Pointer and row stride of a [rows, time] tensor whose tokens lie next to each other; (0, 0) for None."""
    return (0, 0) if t is None else (t.data_ptr(), t.stride(0))


def _check_tokens(shape, dtype, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None:
            assert t.shape == shape, f"{name} must have the shape of logprob"
            assert t.size(1) <= 1 or t.stride(1) == 1, f"{name}'s tokens must lie next to each other"
            if dtype is not None and t.dtype != dtype:
                raise ValueError(f"{name} must have the dtype of logprob, {dtype}")


def policy_loss_forward(logprob, old_logprob, ref_logprob, entropy, advantages, mask, clip_low: float, clip_high: float,
                        dual_clip: float, kl_coef: float, entropy_coef: float, reduction: int, saved, weights, workspace, loss,
                        stats) -> None:
    """Loss and statistics of include/bmt_hip.h ``policy_loss_forward_launcher`` for [rows, time] tensors;
    ``advantages`` is fp32, [rows] or [rows, time]; ``mask`` bool / uint8 or None."""
    _together(logprob, old_logprob=old_logprob, ref_logprob=ref_logprob, entropy=entropy, advantages=advantages, mask=mask,
              saved=saved, weights=weights, workspace=workspace, loss=loss, stats=stats)
    code = _type_code("policy_loss", logprob.dtype)
    assert logprob.dim() == 2, "logprob must be [sequences, tokens]"
    rows, time = logprob.shape
    _check_tokens(logprob.shape, logprob.dtype, logprob=logprob, old_logprob=old_logprob, ref_logprob=ref_logprob, entropy=entropy)
    _check_tokens(logprob.shape, None, mask=mask)
    assert mask is None or mask.dtype in (torch.bool, torch.uint8), "mask must be a bool or uint8 tensor"
    assert advantages.dtype == torch.float32, "advantages must be a float tensor"
    per_token = advantages.dim() == 2
    if per_token:
        _check_tokens(logprob.shape, None, advantages=advantages)
    else:
        assert advantages.shape == (rows,), "advantages must be one to a sequence or one to a token"
    assert saved is None or (saved.is_contiguous() and saved.dtype == torch.float32 and saved.numel() == rows * time)
    assert weights.is_contiguous() and weights.dtype == torch.float32 and weights.numel() >= (1 + rows if reduction == 1 else 1)
    assert workspace.dtype == torch.float64 and workspace.numel() >= C.policy_loss_workspace_doubles(rows, time)
    assert loss.dtype == torch.float32 and stats.dtype == torch.float32 and stats.numel() == 5 and stats.is_contiguous()
    C.policy_loss_forward_launcher(rows, time, code, *_row(logprob), *_row(old_logprob), *_row(ref_logprob), *_row(entropy),
                                   advantages.data_ptr(), advantages.stride(0), int(per_token), *_row(mask), clip_low, clip_high,
                                   dual_clip, kl_coef, entropy_coef, reduction, _ptr(saved), weights.data_ptr(),
                                   workspace.data_ptr(), loss.data_ptr(), stats.data_ptr(), _current_stream())


def policy_loss_backward(reduction: int, saved, weights, upstream, mask, entropy_coef: float, grad_logprob, grad_entropy) -> None:
    """Gradients (contiguous [rows, time], of the log-probabilities' type; either may be None) of ``policy_loss_forward``."""
    first = grad_logprob if grad_logprob is not None else grad_entropy
    if first is None:
        return
    _together(first, saved=saved, weights=weights, upstream=upstream, mask=mask, grad_entropy=grad_entropy)
    rows, time = first.shape
    for t in (grad_logprob, grad_entropy):
        assert t is None or (t.is_contiguous() and t.shape == first.shape and t.dtype == first.dtype)
    assert saved is None or (saved.is_contiguous() and saved.dtype == torch.float32 and saved.numel() == rows * time)
    assert weights.is_contiguous() and weights.dtype == torch.float32 and weights.numel() >= (1 + rows if reduction == 1 else 1)
    assert upstream.dtype == torch.float32 and upstream.numel() == 1, "upstream must be one float"
    _check_tokens(first.shape, None, mask=mask)
    C.policy_loss_backward_launcher(rows, time, _type_code("policy_loss", first.dtype), reduction, _ptr(saved),
                                    weights.data_ptr(), upstream.data_ptr(), *_row(mask), entropy_coef, _ptr(grad_logprob),
                                    _ptr(grad_entropy), _current_stream())


def preference_loss_forward(logprob, ref_logprob, mask, kind: int, average: bool, beta: float, label_smoothing: float, workspace,
                            loss, chosen, rejected, slope) -> None:
    """Loss and rewards of include/bmt_hip.h ``preference_loss_forward_launcher`` for [2 * pairs, time] tensors, the
    chosen answers in front of the rejected ones; ``slope`` (1 + 2 * pairs) is for the backward call."""
    _together(logprob, ref_logprob=ref_logprob, mask=mask, workspace=workspace, loss=loss, chosen=chosen, rejected=rejected,
              slope=slope)
    code = _type_code("preference_loss", logprob.dtype)
    assert logprob.dim() == 2 and logprob.size(0) % 2 == 0, "logprob must be [2 * pairs, tokens]"
    pairs, time = logprob.size(0) // 2, logprob.size(1)
    _check_tokens(logprob.shape, logprob.dtype, logprob=logprob, ref_logprob=ref_logprob)
    _check_tokens(logprob.shape, None, mask=mask)
    assert mask is None or mask.dtype in (torch.bool, torch.uint8), "mask must be a bool or uint8 tensor"
    for t, n in ((loss, 1), (chosen, pairs), (rejected, pairs), (slope, 1 + 2 * pairs)):
        assert t.is_contiguous() and t.dtype == torch.float32 and t.numel() == n
    assert workspace.dtype == torch.float64 and workspace.numel() >= C.preference_loss_workspace_doubles(pairs, time)
    C.preference_loss_forward_launcher(pairs, time, code, *_row(logprob), *_row(ref_logprob), *_row(mask), kind, int(average), beta,
                                       label_smoothing, workspace.data_ptr(), loss.data_ptr(), chosen.data_ptr(),
                                       rejected.data_ptr(), slope.data_ptr(), _current_stream())


def preference_loss_backward(slope, upstream, mask, grad_logprob) -> None:
    """Gradient (contiguous [2 * pairs, time]) of ``preference_loss_forward``."""
    _together(grad_logprob, slope=slope, upstream=upstream, mask=mask)
    rows, time = grad_logprob.shape
    assert grad_logprob.is_contiguous() and rows % 2 == 0
    assert slope.is_contiguous() and slope.dtype == torch.float32 and slope.numel() == 1 + rows
    assert upstream.dtype == torch.float32 and upstream.numel() == 1, "upstream must be one float"
    _check_tokens(grad_logprob.shape, None, mask=mask)
    C.preference_loss_backward_launcher(rows // 2, time, _type_code("preference_loss", grad_logprob.dtype), slope.data_ptr(),
                                        upstream.data_ptr(), *_row(mask), grad_logprob.data_ptr(), _current_stream())
