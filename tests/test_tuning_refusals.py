"""What the tuning operators refuse, without a GPU: argument checks of the modules and of the C entries, all of which are
made on the host before any device call."""
import math

import pytest
import torch

from bmtrain_amd import C, _tensors
from bmtrain_amd.loss import PolicyLoss, PreferenceLoss, TokenLogProbs
from bmtrain_amd.optim import clip_grads


def test_module_arguments():
    for bad in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            TokenLogProbs(temperature=bad)
    for options, text in (({"clip_low": -0.1}, "clip_low"), ({"clip_low": 1.1}, "clip_low"), ({"clip_high": -1.0}, "clip_high"),
                          ({"clip_high": math.nan}, "clip_high"), ({"dual_clip": 1.0}, "dual_clip"), ({"dual_clip": math.inf}, "dual_clip"),
                          ({"reduction": "none"}, "reduction")):
        with pytest.raises(ValueError, match=text):
            PolicyLoss(**options)
    for options, text in (({"beta": 0.0}, "beta"), ({"beta": math.inf}, "beta"), ({"kind": "dpo"}, "kind"),
                          ({"label_smoothing": 1.5}, "label_smoothing"), ({"label_smoothing": 0.1, "kind": "ipo"}, "label_smoothing")):
        with pytest.raises(ValueError, match=text):
            PreferenceLoss(**options)
    assert PolicyLoss(clip_low=0.3).clip_high == 0.3


def test_cpu_tensors_and_shapes():
    x, t = torch.zeros(3, 5), torch.zeros(3, dtype=torch.long)
    with pytest.raises(AssertionError, match="cuda"):
        TokenLogProbs()(x, t)
    with pytest.raises(AssertionError, match="shape"):
        TokenLogProbs()(x, t[:2])
    with pytest.raises(AssertionError, match="cuda"):
        PolicyLoss()(x, x, torch.zeros(3))
    with pytest.raises(AssertionError, match="sequences"):
        PolicyLoss()(x[0], x[0], torch.zeros(5))
    with pytest.raises(AssertionError, match="one to a sequence"):
        PolicyLoss()(x, x, torch.zeros(3, 4))
    for advantages in (torch.zeros(3, 1), torch.zeros(3, 1).expand(3, 0), torch.zeros(3, 0)):      # all of them are taken
        with pytest.raises(AssertionError, match="cuda"):
            PolicyLoss()(x[:, :0], x[:, :0], advantages)
    with pytest.raises(AssertionError, match="cuda"):
        PreferenceLoss()(torch.zeros(4, 5))
    with pytest.raises(AssertionError, match="pairs"):
        PreferenceLoss()(x)
    with pytest.raises(AssertionError, match="cuda"):
        clip_grads([x], 1.0)
    with pytest.raises(ValueError, match="norm_type"):
        clip_grads([x], 1.0, norm_type=1.0)
    with pytest.raises(ValueError, match="must not be negative"):
        clip_grads([x], -1.0)
    with pytest.raises(ValueError, match="scale"):
        clip_grads([x], 1.0, scale=0.0)
    with pytest.raises(ValueError, match="outputs"):
        clip_grads([x], 1.0, out=[])
    with pytest.raises(ValueError, match="float64"):
        clip_grads([x.double()], 1.0)


def test_row_layout():
    x = torch.zeros(4, 7, 10)
    assert _tensors.row_layout(x)[1:] == (28, 10, 7, 70, 10)
    assert _tensors.row_layout(x[:, :-1])[1:] == (24, 10, 6, 70, 10)
    assert _tensors.row_layout(x[:, :, 2:9])[1:] == (28, 7, 7, 70, 10)
    assert _tensors.row_layout(x[1])[1:] == (7, 10, 7, 0, 10)
    assert _tensors.row_layout(x[1, 2])[1:] == (1, 10, 1, 0, 10)
    turned = _tensors.row_layout(x.transpose(1, 2))
    assert turned[0].is_contiguous() and turned[1:] == (40, 7, 40, 0, 7)
    assert _tensors.row_layout(torch.zeros(2, 3, 4, 5))[1:] == (24, 5, 24, 0, 5)
    assert _tensors.row_layout(torch.zeros(0, 5))[1:4] == (0, 5, 1)


def test_dense():
    x = torch.zeros(4, 6, 5)
    for t, dense in ((x, True), (x.permute(2, 0, 1), True), (x[:, :3], False), (x[:, ::2], False), (x[:1].expand(4, 6, 5), False),
                     (x[:1], True), (x[:, :1, :1], False), (x[:0, :3], True), (torch.zeros(()), True)):
        assert _tensors.is_dense(t) is dense


def logprobs(rows=2, n=8, inner=2, x=0x1000, code=0, target=0x2000, bits=64, temperature=1.0, logprob=0x3000, entropy=0, stats=0):
    C.token_logprobs_forward_launcher(rows, n, inner, 0, n, x, code, target, bits, -100, temperature, logprob, entropy, stats, 0)


def test_tensors_that_are_none():
    """What is no plain tensor of numbers is refused, not read."""
    for bad in (torch.zeros(3).to_sparse(), torch.zeros(3, device="meta"), torch.zeros(3, dtype=torch.complex64).conj(), 1.0, "grad"):
        with pytest.raises((RuntimeError, ValueError, TypeError, AssertionError)):
            clip_grads([bad], 1.0)
        with pytest.raises((RuntimeError, ValueError, TypeError, AssertionError)):
            PolicyLoss()(bad, bad, bad)
        with pytest.raises((RuntimeError, ValueError, TypeError, AssertionError)):
            PreferenceLoss()(bad)
        with pytest.raises((RuntimeError, ValueError, TypeError, AssertionError)):
            TokenLogProbs()(bad, torch.zeros(3, dtype=torch.long))
    with pytest.raises(TypeError):
        PolicyLoss()(torch.zeros(2, 3), None, torch.zeros(2))


def test_clip_grads_without_an_output():
    with pytest.raises(ValueError, match="without an output"):
        clip_grads([torch.zeros(3)], 1.0, out=[None])


def test_c_entries_refuse_on_the_host():
    logprobs(rows=0)
    for bad, text in (({"code": 3}, "type code"), ({"x": 0}, "null"), ({"target": 0}, "null"), ({"logprob": 0}, "null"), ({"bits": 16}, "bits"),
                      ({"x": 0x1002}, "aligned"), ({"target": 0x2004}, "aligned"), ({"stats": 0x4008}, "misaligned"),
                      ({"temperature": 0.0}, "temperature"), ({"temperature": math.nan}, "temperature"), ({"temperature": 1e-45}, "temperature"),
                      ({"rows": 1 << 31}, "too many"), ({"n": 1 << 31}, "too many"), ({"rows": 1 << 26, "n": 5000}, "too many"), ({"inner": 0}, "too many")):
        with pytest.raises(RuntimeError, match=text):
            logprobs(**bad)
    with pytest.raises(RuntimeError, match="null"):
        C.token_logprobs_backward_launcher(2, 8, 2, 0, 8, 0x1000, 0, 0x2000, 64, -100, 1.0, 0, 0, 0, 0x5000, 0)
    with pytest.raises(RuntimeError, match="too many"):
        C.token_logprobs_backward_launcher(1 << 30, 1 << 20, 1 << 30, 0, 1 << 20, 0x1000, 0, 0x2000, 64, -100, 1.0, 0x3000, 0, 0, 0x5000, 0)


def policy(rows=2, time=8, code=0, logprob=0x1000, old=0x2000, advantage=0x3000, col=0, low=0.2, high=0.2, dual=0.0, reduction=0,
           weights=0x4000, workspace=0x5000, loss=0x6000, stats=0x7000):
    C.policy_loss_forward_launcher(rows, time, code, logprob, time, old, time, 0, 0, 0, 0, advantage, 1, col, 0, 0, low, high, dual, 0.0, 0.0,
                                   reduction, 0, weights, workspace, loss, stats, 0)


def test_policy_entry():
    for bad, text in (({"rows": -1}, "negative"), ({"reduction": 3}, "reduction"), ({"code": 7}, "type code"), ({"low": 1.5}, "clip"),
                      ({"high": math.nan}, "clip"), ({"dual": 0.5}, "dual_clip"), ({"loss": 0}, "null"), ({"weights": 0}, "null"),
                      ({"logprob": 0}, "null"), ({"logprob": 0x1002}, "misaligned"), ({"workspace": 0x5004}, "misaligned"), ({"col": 2}, "one to a"),
                      ({"time": 1 << 31}, "too many"), ({"rows": 1 << 40}, "too many"),
                      ({"rows": 1 << 24, "time": 1 << 10}, "too many")):
        with pytest.raises(RuntimeError, match=text):
            policy(**bad)
    C.policy_loss_backward_launcher(0, 8, 0, 0, 0, 0, 0, 0, 0, 0.0, 0x1000, 0, 0)
    with pytest.raises(RuntimeError, match="null"):
        C.policy_loss_backward_launcher(2, 8, 0, 0, 0, 0x2000, 0x3000, 0, 0, 0.0, 0x1000, 0, 0)
    assert C.policy_loss_workspace_doubles(0, 5) == 1 and C.policy_loss_workspace_doubles(3, 9000) == 3 * 9 * 6 and C.policy_loss_workspace_doubles(1024, 8192) == 1024 * 6


def preference(pairs=2, time=8, code=0, logprob=0x1000, kind=0, beta=0.1, smoothing=0.0, workspace=0x2000, loss=0x3000, chosen=0x4000,
               rejected=0x5000, slope=0x6000):
    C.preference_loss_forward_launcher(pairs, time, code, logprob, time, 0, 0, 0, 0, kind, 0, beta, smoothing, workspace, loss, chosen, rejected,
                                       slope, 0)


def test_preference_entry():
    for bad, text in (({"pairs": -1}, "negative"), ({"kind": 3}, "kind"), ({"code": -1}, "type code"), ({"beta": 0.0}, "beta"),
                      ({"beta": math.inf}, "beta"), ({"smoothing": -0.1}, "smoothing"), ({"logprob": 0}, "null"), ({"slope": 0}, "null"),
                      ({"chosen": 0x4002}, "misaligned"), ({"time": 1 << 31}, "too many"), ({"pairs": 1 << 31}, "too many"),
                      ({"pairs": 1 << 20, "time": 1 << 14}, "too many")):
        with pytest.raises(RuntimeError, match=text):
            preference(**bad)
    with pytest.raises(RuntimeError, match="null"):
        C.preference_loss_backward_launcher(2, 8, 0, 0x1000, 0, 0, 0, 0x2000, 0)


def test_clip_entries():
    def scale(rows, coef=0x100000):
        table = C.clip_table(*[list(column) for column in zip(*rows)]) if rows else C.clip_table([], [], [], [], [])
        C.grad_scale_multi_launcher(len(rows), table.buffer_info()[0], coef, 0, 0)
    scale([])
    scale([(0, 0, 0, 0, 0)])                                                # entries without elements are skipped
    a, b = 0x10000, 0x20000
    for rows, text in (([(a, a, 10, 0, 0), (a, a, 10, 0, 0)], "shares"), ([(a, b, 10, 0, 0), (b, b, 10, 0, 0)], "shares"),
                       ([(a, a + 4, 10, 0, 0)], "shares"), ([(a, a, 10, 0, 2)], "shares"), ([(a, b, 10, 0, 0), (b + 36, b + 0x800, 4, 0, 0)], "shares"),
                       ([(a, b, 100, 0, 0), (b + 0x1000, b + 8, 2, 0, 0)], "shares"), ([(a, b, 10, 3, 0)], "type code"), ([(0, b, 10, 0, 0)], "null"),
                       ([(a + 2, b, 10, 0, 0)], "aligned"), ([(a, b + 1, 10, 0, 2)], "aligned"), ([(a, b, 1 << 50, 0, 0)], "too large")):
        with pytest.raises(RuntimeError, match=text):
            scale(rows)
    with pytest.raises(RuntimeError, match="null"):
        scale([(a, b, 10, 0, 0)], coef=0)
    table = C.clip_table([a], [0], [10], [0], [0])
    address = table.buffer_info()[0]
    with pytest.raises(RuntimeError, match="scale"):
        C.grad_norm_multi_launcher(1, address, 0, 1.0, 1e-6, 0.0, 0x1000, 0x2000, 0)
    with pytest.raises(RuntimeError, match="null"):
        C.grad_norm_multi_launcher(1, address, 0, 1.0, 1e-6, 1.0, 0, 0x2000, 0)
    assert C.grad_norm_workspace_doubles(1, address) == 2 and C.grad_norm_workspace_doubles(0, 0) == 1


def test_leaves_are_written_under_no_grad_only():
    """As with any in-place operation: the write would be no part of the leaf's graph."""
    for device in ("cpu", "cuda") if torch.cuda.is_available() else ("cpu",):
        leaf = torch.full((8,), 2.0, device=device, requires_grad=True)
        plain = torch.full((8,), 2.0, device=device)
        for call in (lambda: clip_grads([leaf], 0.1), lambda: clip_grads([plain], 0.1, out=[leaf]), lambda: clip_grads([leaf[2:6]], 0.1),
                     lambda: clip_grads([plain, plain.clone()], 0.1, out=[torch.empty_like(plain), leaf])):
            with pytest.raises(RuntimeError, match="leaf"):
                call()
        assert (leaf == 2).all() and (plain == 2).all()
