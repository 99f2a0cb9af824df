"""Token log-probabilities and entropies (bmtrain_amd.loss.TokenLogProbs) against the definition in 64 bits.

Tolerances.  u = 2^-24 is half a step of fp32 relative to the value; R is the largest |x - max| / T of the row (over
classes with a finite logit).  A z = (x - max) / T carries at most four roundings, its exponential an error of 4 u |z|
(relative), the sum of exponentials at most 64 additions in a row: L is off by (64 + 8 R) u, a log-probability by twice
that, a probability relatively by the same.  The entropy is a mean of |z| <= R with such weights.  A gradient element is
off by its probability's error times what multiplies it, plus half a step of its own type.
"""
import pytest
import torch

from bmtrain_amd import _tensors
from bmtrain_amd.loss import TokenLogProbs

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def reference(logits, target, ignore, temperature, g=None, h=None):
    """(logprob, entropy, gradient or None, tolerance row scale R) in 64 bits."""
    x = logits.double()
    z = x - x.amax(-1, keepdim=True)
    z = z / temperature
    finite = torch.isfinite(z)
    far = torch.where(finite, z, 0.0).abs().amax(-1).clamp(max=1000.0)
    s = z.exp().sum(-1, keepdim=True)
    logs = z - s.log()
    p = logs.exp()
    entropy = -(torch.where(p > 0, p * logs, 0.0)).sum(-1)
    keep = target != ignore
    at = torch.where(keep, target, 0).long().unsqueeze(-1)
    logprob = torch.where(keep, logs.gather(-1, at).squeeze(-1), 0.0)
    grad = None
    if g is not None:
        g = torch.where(keep, g.double(), 0.0).unsqueeze(-1)
        h = torch.where(keep, h.double(), 0.0).unsqueeze(-1) if h is not None else torch.zeros_like(g)
        grad = -p * g - torch.where(p > 0, h * p * (logs + entropy.unsqueeze(-1)), 0.0)
        grad = grad.scatter_add(-1, at, g) / temperature
    return logprob, torch.where(keep, entropy, 0.0), grad, p, far


def check(logits, target, ignore=-100, temperature=1.0, entropy=True, g=None, h=None):
    """Runs the module on a leaf made of `logits` and compares everything."""
    leaf = logits.detach().requires_grad_(g is not None)
    out = TokenLogProbs(ignore, temperature, entropy)(leaf, target)
    out = out if entropy else (out,)
    if g is not None:
        out += torch.autograd.grad(out, [leaf], [g, h][:len(out)])
    compare(out, logits, target, ignore, temperature, entropy, g, h)
    return out


def compare(out, logits, target, ignore=-100, temperature=1.0, entropy=True, g=None, h=None):
    """Log-probabilities, entropies (with `entropy`) and the gradient (with `g`) in `out` against the definition."""
    want, want_entropy, want_grad, p, far = reference(logits, target, ignore, temperature, g, h if entropy else None)
    tol = U * (160 + 24 * far)
    assert out[0].dtype == torch.float32 and out[0].shape == target.shape
    assert ((out[0].double() - want).abs() <= tol + U * want.abs()).all()
    if entropy:
        assert ((out[1].double() - want_entropy).abs() <= tol * (1 + far)).all()
    if g is None:
        return
    grad = out[-1]
    assert grad.dtype == logits.dtype and grad.shape == logits.shape
    top = (g.abs() + (h.abs() * (2 * far + 16) if entropy and h is not None else 0.0)).double().unsqueeze(-1) / temperature
    step = torch.finfo(logits.dtype).eps / 2
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}[logits.dtype]
    bound = 1.01 * step * want_grad.abs() + p * top * (2 * tol.unsqueeze(-1) + 8 * U) + 4 * U * want_grad.abs() + tiny
    off = (grad.double() - want_grad).abs()
    assert (off <= bound).all(), float((off / bound).max())


def make(rows, n, dtype, seed, spread=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    logits = (torch.randn(rows, n, generator=gen, device="cuda") * spread).to(dtype)
    target = torch.randint(0, n, (rows,), generator=gen, device="cuda")
    g = torch.randn(rows, generator=gen, device="cuda")
    h = torch.randn(rows, generator=gen, device="cuda") * 0.1
    return logits, target, g, h


TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2), (5, 7), (1, 9), (67, 63), (9, 512), (4, 513), (33, 4095), (7, 4096), (5, 4097),
                                    (2, 8192), (6, 8199), (11, 32000), (3, 50257), (1, 131071), (2, 1000003)])
def test_sizes(dtype, rows, n):
    logits, target, g, h = make(rows, n, dtype, rows * 131 + n)
    if rows > 3:
        target[::3] = -100
    check(logits, target, g=g, h=h)
    check(logits, target, entropy=False, g=g)
    check(logits, target.int(), temperature=0.7, g=g, h=h)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [97, 5003])
def test_views_are_not_copied_and_give_the_same(dtype, n):
    """[batch, time, n] views: next-token slices, padded classes, rows backwards in memory order, a broadcast row."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    full = (torch.randn(3, 9, n + 6, generator=gen, device="cuda") * 2).to(dtype)
    for view in (full[:, :-1, :n], full[:, 1:, 5:], full.transpose(0, 1)[:, :, 1:n], full[::2, ::3, :n], full[:, :1, :n],
                 full[1, 2, :n].expand(4, 5, n), full[0, :, :n]):
        assert _tensors.row_layout(view)[0].data_ptr() == view.data_ptr()
        target = torch.randint(0, view.size(-1), view.shape[:-1], generator=gen, device="cuda")
        g, h = torch.randn(target.shape, generator=gen, device="cuda"), torch.randn(target.shape, generator=gen, device="cuda")
        check(view, target, g=g, h=h, temperature=1.3)
    four = full.view(3, 3, 3, n + 6)[..., :n]                       # more strides than two: copied
    target = torch.randint(0, n, four.shape[:-1], generator=gen, device="cuda")
    g = torch.randn(target.shape, generator=gen, device="cuda")
    check(four, target, g=g, h=g)
    strided = full.transpose(1, 2)                                  # classes apart from each other: copied
    target = torch.randint(0, 9, strided.shape[:-1], generator=gen, device="cuda")
    g = torch.randn(target.shape, generator=gen, device="cuda")
    check(strided, target, g=g, h=g)
    one = full[0, 0, :n]                                            # a single distribution
    check(one, torch.tensor(3, device="cuda"), g=torch.tensor(0.5, device="cuda"), h=torch.tensor(-1.0, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [300, 6001])
def test_extreme_logits(dtype, n):
    """Classes masked with -inf or the type's lowest value, rows of equal values, the type's largest values, one finite
    class: probabilities 0 add nothing, nothing turns into NaN."""
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    logits, target, g, h = make(8, n, dtype, n)
    target[:] = 5
    logits[0, 50:] = float("-inf")
    logits[1, 50:] = low
    logits[2, :] = low
    logits[3, :] = high
    logits[4, :] = float("-inf")
    logits[4, 5] = 1.0
    logits[5, :] = low
    logits[5, 5] = high
    logits[6, :] = 0.0
    logits[7, 0] = float("-inf")
    for temperature in (1.0, 0.5):
        out = check(logits, target, temperature=temperature, g=g, h=h)
        for t in out:
            assert torch.isfinite(t).all()
        assert out[0][4] == 0 and out[1][4] == 0 and out[0][5] == 0
    target[0] = 100                                                 # a class of probability 0
    logp, entropy = TokenLogProbs(entropy=True)(logits, target)
    assert logp[0] == float("-inf") and torch.isfinite(entropy).all() and torch.isfinite(logp[1:]).all()
    leaf = logits.requires_grad_()
    grad, = torch.autograd.grad(TokenLogProbs()(leaf, target), leaf, g)
    assert torch.isfinite(grad).all() and grad[0, 100] == g[0].to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_stays_in_its_row(dtype):
    n = 4999
    logits, target, g, h = make(6, n, dtype, 1)
    logits[1, 77] = float("nan")
    logits[3, 4000] = float("inf")
    logits[4, :] = float("-inf")
    leaf = logits.requires_grad_()
    logp, entropy = TokenLogProbs(entropy=True)(leaf, target)
    grad, = torch.autograd.grad((logp, entropy), leaf, (g, h))
    bad = torch.tensor([False, True, False, True, True, False], device="cuda")
    assert torch.equal(torch.isnan(logp), bad) and torch.equal(torch.isnan(entropy), bad)
    assert torch.equal(torch.isnan(grad).any(1), bad)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [129, 7001])
def test_ignored_and_unweighted_rows_are_not_read(dtype, n):
    """Rows whose target is ignored hold NaN throughout: results and gradients are 0.  A row without upstream gradient
    gets a gradient of 0 whatever it holds."""
    logits, target, g, h = make(9, n, dtype, n)
    target[2] = target[8] = -1
    logits[2] = logits[8] = float("nan")
    out = check(logits[:2], target[:2], ignore=-1, g=g[:2], h=h[:2])
    leaf = logits.clone().requires_grad_()
    logp, entropy = TokenLogProbs(ignore_index=-1, entropy=True)(leaf, target)
    g[4] = h[4] = 0
    grad, = torch.autograd.grad((logp, entropy), leaf, (g, h))
    assert logp[2] == 0 and entropy[8] == 0 and (grad[2] == 0).all() and (grad[8] == 0).all() and (grad[4] == 0).all()
    assert torch.equal(grad[:2], out[2]) and torch.isfinite(grad).all()
    target[:] = -1                                                  # nothing counts at all
    leaf = logits.clone().requires_grad_()
    logp = TokenLogProbs(ignore_index=-1)(leaf, target)
    grad, = torch.autograd.grad(logp.sum(), leaf)
    assert (logp == 0).all() and (grad == 0).all()


def test_target_outside_the_classes():
    logits, target, g, h = make(4, 33, torch.float32, 3)
    target[1], target[2] = 33, -7
    leaf = logits.requires_grad_()
    logp, entropy = TokenLogProbs(entropy=True)(leaf, target)
    assert torch.equal(torch.isnan(logp), torch.tensor([False, True, True, False], device="cuda"))
    assert torch.isfinite(entropy).all()
    grad, = torch.autograd.grad(logp, leaf, g)
    p = leaf.detach().double().softmax(-1)
    assert torch.allclose(grad[1].double(), -g[1].double() * p[1], rtol=1e-5, atol=1e-7)


def test_partial_gradients_and_modes():
    """Only one of the two outputs used, no gradient wanted, gradients of an expanded leaf, a frozen graph."""
    logits, target, g, h = make(6, 700, torch.float32, 5)
    leaf = logits.clone().requires_grad_()
    module = TokenLogProbs(entropy=True, temperature=0.9)
    logp, entropy = module(leaf, target)
    only_logp, = torch.autograd.grad(logp, leaf, g, retain_graph=True)
    only_entropy, = torch.autograd.grad(entropy, leaf, h, retain_graph=True)
    both, = torch.autograd.grad((logp, entropy), leaf, (g, h))
    assert torch.allclose(only_logp + only_entropy, both, rtol=1e-5, atol=1e-7)
    with torch.no_grad():
        again = module(leaf, target)
    assert torch.equal(again[0], logp) and torch.equal(again[1], entropy) and not again[0].requires_grad
    row = logits[:1].clone().requires_grad_()
    row_target = target[:1].expand(6).contiguous()
    total, = torch.autograd.grad(module(row.expand(6, 700), row_target)[0], row, torch.ones(6, device="cuda"))
    single, = torch.autograd.grad(module(row, target[:1])[0], row, torch.ones(1, device="cuda"))
    assert torch.allclose(total, 6 * single, rtol=1e-5, atol=1e-6)
    with pytest.raises(RuntimeError, match="once_differentiable|differentiate twice|does not require grad"):
        logp, _ = module(leaf, target)
        first, = torch.autograd.grad(logp.sum(), leaf, create_graph=True)
        first.sum().backward()


def test_empty_batches():
    for shape in ((0, 10), (0, 5, 10), (4, 0, 10)):
        leaf = torch.zeros(shape, device="cuda", requires_grad=True)
        logp, entropy = TokenLogProbs(entropy=True)(leaf, torch.zeros(shape[:-1], dtype=torch.long, device="cuda"))
        assert logp.shape == shape[:-1] == entropy.shape
        (logp.sum() + entropy.sum()).backward()
        assert leaf.grad.shape == shape


def test_gradient_against_differences():
    """Directional derivative of the 64-bit definition by central differences: with step s the difference is off by
    s^2 / 6 times a third derivative (below 1e-6 here) and the fp32 gradient by its own 1e-6 relative."""
    logits, target, g, h = make(5, 211, torch.float32, 9)
    leaf = logits.clone().requires_grad_()
    out = TokenLogProbs(entropy=True, temperature=1.7)(leaf, target)
    grad, = torch.autograd.grad(out, leaf, (g, h))
    gen = torch.Generator(device="cuda").manual_seed(4)
    for _ in range(4):
        way = torch.randn(logits.shape, generator=gen, device="cuda").double()
        step = 1e-4

        def value(x):
            logp, entropy, *_ = reference(x, target, -100, 1.7)
            return (logp * g).sum() + (entropy * h).sum()
        want = (value(logits.double() + step * way) - value(logits.double() - step * way)) / (2 * step)
        got = (grad.double() * way).sum()
        assert abs(float(got - want)) <= 1e-5 * float((grad.double().abs() * way.abs()).sum())


def test_offsets_beyond_32_bits():
    """Rows whose first element lies behind 2^31 elements of the tensor, in logits and gradient."""
    n, rows = 131072, 16400                                         # 2.15e9 elements, 4.3 GB
    logits = torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda")
    target = torch.full((rows,), -100, device="cuda")
    last = slice(rows - 3, rows)
    small, small_target, g, h = make(3, n, torch.bfloat16, 17)
    logits[last] = small
    target[last] = small_target
    leaf = logits.requires_grad_()
    logp, entropy = TokenLogProbs(entropy=True)(leaf, target)
    gg, hh = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    gg[last], hh[last] = g, h
    grad, = torch.autograd.grad((logp, entropy), leaf, (gg, hh))
    compare((logp[last], entropy[last], grad[last]), small, small_target, g=g, h=h)
    assert float(grad[:-3].abs().max()) == 0.0


def test_side_stream_and_graph():
    """On a stream of its own, and forward and backward captured and replayed with eager work in between."""
    logits, target, g, h = make(40, 9001, torch.bfloat16, 21)
    module = TokenLogProbs(entropy=True)

    def step(x):
        leaf = x.detach().requires_grad_()
        out = module(leaf, target)
        return (*[o.detach() for o in out], *torch.autograd.grad(out, leaf, (g, h)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = step(logits)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(aside, step(logits)):
        assert torch.equal(a, b)
    still = logits.clone()
    with torch.cuda.stream(side):
        step(still)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step(still)
    for seed in range(4):
        fresh, *_ = make(40, 9001, torch.bfloat16, 100 + seed)
        still.copy_(fresh)
        want = step(fresh)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), seed


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [5, 257, 4999, 33000])
def test_confident_tokens_keep_their_digits(dtype, n):
    """The target far above everything else: log-probabilities of 1e-2 .. 1e-30 and the gradient 1 - p, relative to
    themselves.  The others' sum has at most 64 additions and exponentials of |z| <= R: (64 + 8 R) u relative, and half
    as much again for its logarithm and the products."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    lifts = torch.tensor([6.0, 14.0, 20.0, 34.0, 60.0], device="cuda")
    logits = (torch.randn(5, n, generator=gen, device="cuda") * 0.5).clamp(-2, 2)
    target = torch.randint(0, n, (5,), generator=gen, device="cuda")
    logits[torch.arange(5), target] = lifts + 2
    logits = logits.to(dtype)
    leaf = logits.clone().requires_grad_()
    logp, entropy = TokenLogProbs(entropy=True)(leaf, target)
    grad, = torch.autograd.grad((logp, entropy), leaf, (torch.ones(5, device="cuda"), torch.zeros(5, device="cuda")))
    x = logits.double()
    others = x - x.gather(1, target.unsqueeze(1))
    rest = others.exp().scatter(1, target.unsqueeze(1), 0.0).sum(1)
    want = -torch.log1p(rest)
    tol = U * 1.5 * (64 + 8 * 66) * 2
    assert ((logp.double() - want).abs() <= tol * want.abs()).all()
    weighted = (others * others.exp()).scatter(1, target.unsqueeze(1), 0.0).sum(1)
    want_entropy = torch.log1p(rest) - weighted / (1 + rest)
    assert ((entropy.double() - want_entropy).abs() <= 4 * tol * want_entropy).all()
    at_target = grad.double().gather(1, target.unsqueeze(1)).squeeze(1)
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}[dtype]
    assert ((at_target - rest / (1 + rest)).abs() <= (tol + torch.finfo(dtype).eps / 2 * 1.01) * rest + tiny).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 5, 300, 4999, 33000, 131072])
def test_an_infinite_logit_at_the_target(dtype, n):
    """A row's only +inf, at the target itself: NaN throughout the row, as with the infinity anywhere else."""
    places = sorted({0, n // 3, n // 2, n - 1})
    logits, target, g, h = make(len(places) + 1, n, dtype, n)
    for r, place in enumerate(places):
        target[r] = place
        logits[r, place] = float("inf")
    bad = torch.arange(len(places) + 1, device="cuda") < len(places)
    for entropy in (True, False):
        leaf = logits.clone().requires_grad_()
        out = TokenLogProbs(entropy=entropy)(leaf, target)
        out = out if entropy else (out,)
        grad, = torch.autograd.grad(out, leaf, (g, h)[:len(out)])
        for t in out:
            assert torch.equal(torch.isnan(t), bad)
        assert torch.equal(torch.isnan(grad).all(1), bad) and torch.equal(torch.isnan(grad).any(1), bad)
