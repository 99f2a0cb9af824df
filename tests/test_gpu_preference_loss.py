"""PreferenceLoss against the definition in 64 bits.

Tolerances.  Token differences, sums and everything per pair are 64 bits in the kernel, so results differ from the
reference by 64-bit roundings of the sums (2^-50 of the sum of magnitudes is ample) and one rounding to fp32 (2^-24).
A gradient is a product of three fp32 factors (2^-22) and rounded to its type (half a step).
"""
import pytest
import torch

from bmtrain_amd.loss import PreferenceLoss

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(pairs, time, dtype, seed, noise=0.3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    logprob = -torch.randn(2 * pairs, time, generator=gen, device="cuda").abs() * 2
    ref = logprob + noise * torch.randn(2 * pairs, time, generator=gen, device="cuda")
    lengths = torch.randint(0, time + 1, (2 * pairs, 1), generator=gen, device="cuda")
    mask = torch.arange(time, device="cuda").view(1, -1) < lengths
    return logprob.to(dtype), ref.to(dtype), mask


def reference(logprob, ref, mask, beta=0.1, kind="sigmoid", label_smoothing=0.0, average=False):
    x = logprob.double() - (0 if ref is None else ref.double())
    keep = torch.ones_like(x, dtype=torch.bool) if mask is None else mask != 0
    x = torch.where(keep, x, 0.0)
    n = keep.sum(1)
    norm = n.clamp(min=1).double() if average else torch.ones_like(n, dtype=torch.float64)
    s = x.sum(1) / norm
    size = x.abs().sum(1) / norm
    pairs = s.numel() // 2
    h = s[:pairs] - s[pairs:]
    leaf = h.clone().requires_grad_()
    y = beta * leaf
    if kind == "sigmoid":
        one = -(1 - label_smoothing) * torch.nn.functional.logsigmoid(y) - label_smoothing * torch.nn.functional.logsigmoid(-y)
    elif kind == "ipo":
        one = (leaf - 0.5 / beta) ** 2
    else:
        one = (1 - y).clamp(min=0)
    d, = torch.autograd.grad(one.sum(), leaf) if pairs else (leaf,)
    counts = (n[:pairs] + n[pairs:] > 0).double()
    share = counts / counts.sum().clamp(min=1)
    row = torch.cat([d * share, -d * share]) / norm
    h_size = size[:pairs] + size[pairs:]
    loss_tol = (share * (2.0 ** -50 * h_size * (d.abs() + 1) + 2.0 ** -50 * one.detach())).sum()
    return (one.detach() * share).sum(), beta * s[:pairs], beta * s[pairs:], keep * row.unsqueeze(1), loss_tol, beta * size


def check(logprob, ref, mask, upstream=5.0, **options):
    leaf = logprob.detach().requires_grad_()
    loss, chosen, rejected = PreferenceLoss(**options)(leaf, ref, mask)
    want = reference(logprob, ref, mask, **options)
    pairs = chosen.numel()
    assert loss.shape == () and loss.dtype == torch.float32 and not chosen.requires_grad and not rejected.requires_grad
    assert abs(loss.double() - want[0]) <= want[4] + U * want[0].abs() * 1.01
    for got, exact, size in ((chosen, want[1], want[5][:pairs]), (rejected, want[2], want[5][pairs:])):
        assert ((got.double() - exact).abs() <= U * 1.01 * exact.abs() + 2.0 ** -50 * size + 1e-44).all()
    grad, = torch.autograd.grad(loss, leaf, torch.tensor(upstream, device="cuda"))
    assert grad.shape == logprob.shape and grad.dtype == logprob.dtype
    exact = upstream * want[3]
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}[logprob.dtype]
    bound = (1.01 * torch.finfo(logprob.dtype).eps / 2 + 4 * U) * exact.abs() + tiny
    if options.get("kind") == "ipo":        # dloss/dh = 2 (h - 1/(2 beta)) crosses zero: the sums' own roundings remain
        bound = bound + abs(upstream) * 2.0 ** -48 * float(want[5].max() / options.get("beta", 0.1) + 10)
    assert ((grad.double() - exact).abs() <= bound).all(), float((grad.double() - exact).abs().max())
    if mask is not None:
        assert (grad[mask == 0] == 0).all()
    return loss.detach(), chosen, rejected, grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["sigmoid", "ipo", "hinge"])
@pytest.mark.parametrize("pairs,time", [(1, 1), (1, 3), (5, 31), (3, 32), (4, 33), (2, 1023), (3, 1025), (1, 4097), (2, 12290), (3000, 5),
                                        (700, 90)])
def test_sizes(pairs, time, dtype, kind):
    logprob, ref, mask = make(pairs, time, dtype, pairs + time)
    check(logprob, ref, mask, kind=kind)
    check(logprob, ref, mask, kind=kind, average=True, beta=0.5)
    check(logprob, None, None, kind=kind, beta=0.05)


@pytest.mark.parametrize("smoothing", [0.0, 0.1, 0.5, 1.0])
def test_label_smoothing_and_large_margins(smoothing):
    """Margins of a few hundred: the logistic loss is linear there, nothing overflows."""
    logprob, ref, mask = make(16, 2000, torch.float32, 4)
    logprob[:8] -= 2.0
    check(logprob, ref, mask, label_smoothing=smoothing, beta=1.0)


@pytest.mark.parametrize("time", [7, 600, 9001])
def test_empty_rows_pairs_and_batches(time):
    logprob, ref, mask = make(6, time, torch.float32, time)
    mask[0] = False                     # one side without a token
    mask[7] = False
    mask[2] = mask[8] = False           # a whole pair: it does not count
    clean = check(logprob, ref, mask)
    garbage = torch.tensor([float("nan"), float("inf"), float("-inf"), 3.4e38], device="cuda")
    fill = garbage[torch.arange(time, device="cuda") % 4].expand(12, time)
    dirty = check(torch.where(mask, logprob, fill), torch.where(mask, ref, fill.flip(1)), mask)
    for a, b in zip(clean, dirty):
        assert torch.equal(a, b)
    mask[:] = False
    for kind in ("sigmoid", "ipo", "hinge"):
        loss, chosen, rejected, grad = check(logprob, ref, mask, kind=kind)
        assert loss == 0 and (grad == 0).all() and (chosen == 0).all()


def test_sums_per_row_and_layouts():
    logprob, ref, mask = make(5, 64, torch.float32, 8)
    sums, ref_sums = logprob.sum(1), ref.sum(1)
    leaf = sums.clone().requires_grad_()
    loss, chosen, rejected = PreferenceLoss()(leaf, ref_sums)
    want = reference(sums.unsqueeze(1), ref_sums.unsqueeze(1), None)
    assert abs(loss.double() - want[0]) <= 1e-6 * want[0]
    grad, = torch.autograd.grad(loss, leaf)
    assert grad.shape == sums.shape and torch.allclose(grad.double(), want[3][:, 0], rtol=1e-6)
    wide = torch.zeros(10, 80, device="cuda")
    wide[:, 3:67] = logprob
    want = check(logprob, ref, mask)
    for view in (wide[:, 3:67], logprob.t().contiguous().t()):
        for a, b in zip(check(view, ref, mask.to(torch.int32)), want):
            assert torch.equal(a, b)
    for shape in ((0, 4), (6, 0)):
        leaf = torch.zeros(shape, device="cuda", requires_grad=True)
        loss, chosen, rejected = PreferenceLoss()(leaf)
        assert loss == 0 and chosen.shape == (shape[0] // 2,) == rejected.shape
        grad, = torch.autograd.grad(loss, leaf)
        assert grad.shape == shape


class Stop(torch.autograd.Function):
    """Hands no gradient on, not even zeros."""

    @staticmethod
    def forward(ctx, x):
        return x.clone()

    @staticmethod
    def backward(ctx, upstream):
        return None


def test_no_gradient_from_behind():
    leaf = torch.zeros(4, 6, device="cuda", requires_grad=True)
    Stop.apply(PreferenceLoss()(leaf)[0]).backward()
    assert leaf.grad is None or (leaf.grad == 0).all()


def test_gradient_against_differences():
    logprob, ref, mask = make(4, 30, torch.float32, 12)
    for kind in ("sigmoid", "ipo"):
        leaf = logprob.clone().requires_grad_()
        loss, *_ = PreferenceLoss(kind=kind, average=True)(leaf, ref, mask)
        grad, = torch.autograd.grad(loss, leaf)
        way, step = torch.randn(8, 30, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").double(), 1e-4
        up, down = [reference(logprob.double() + s * step * way, ref, mask, kind=kind, average=True)[0] for s in (1, -1)]
        assert abs(float((grad.double() * way).sum() - (up - down) / (2 * step))) <= 1e-5 * float((grad.double() * way).abs().sum())


def test_equal_bits_and_graph():
    logprob, ref, mask = make(24, 5000, torch.bfloat16, 3)
    module = PreferenceLoss(label_smoothing=0.1)
    upstream = torch.tensor(64.0, device="cuda")

    def step(l, f, m):
        leaf = l.detach().requires_grad_()
        loss, chosen, rejected = module(leaf, f, m)
        return (loss.detach(), chosen, rejected, *torch.autograd.grad(loss, leaf, upstream))
    for a, b in zip(step(logprob, ref, mask), step(logprob, ref, mask)):
        assert torch.equal(a, b)
    still = [t.clone() for t in (logprob, ref, mask)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*still)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step(*still)
    for seed in range(4):
        fresh = make(24, 5000, torch.bfloat16, 70 + seed)
        for s, f in zip(still, fresh):
            s.copy_(f)
        want = step(*fresh)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), seed


@pytest.mark.parametrize("dtype", TYPES)
def test_infinite_margins_without_smoothing(dtype):
    """A rejected token of probability 0 gives the margin +inf and the loss 0, with its gradient; so does a chosen one
    under a smoothing of 1.  Everything but the rewards is what a margin far beyond any exponential gives."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    logprob = -torch.rand(8, 30, generator=gen, device="cuda")
    for smoothing, row in ((0.0, 6), (1.0, 2)):
        outs = []
        for value in (-3e4, float("-inf")):
            x = logprob.clone()
            x[row, 11] = value
            leaf = x.to(dtype).requires_grad_()
            loss, chosen, rejected = PreferenceLoss(beta=0.5, label_smoothing=smoothing)(leaf)
            outs.append((loss.detach(), torch.autograd.grad(loss, leaf)[0]))
            assert torch.isfinite(loss) and torch.isfinite(outs[-1][1]).all() and (outs[-1][1][row] == 0).all()
        assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
        assert torch.cat([chosen, rejected])[row] == float("-inf")
    for smoothing, row in ((0.1, 6), (0.0, 2), (1.0, 6)):           # here the loss is infinite
        x = logprob.clone()
        x[row, 11] = float("-inf")
        assert PreferenceLoss(label_smoothing=smoothing)(x.to(dtype))[0] == float("inf")
