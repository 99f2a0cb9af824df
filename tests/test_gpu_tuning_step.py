"""The operators together, as a tuning step uses them: logits -> token log-probabilities and entropies -> policy or
preference loss under a loss scale -> gradients of the weights -> clipped into the 16-bit gradients -> Adam."""
import pytest
import torch

import bmtrain_amd as bmt

pytestmark = pytest.mark.gpu

VOCAB, HIDDEN, BATCH, TIME = 503, 64, 6, 41


def problem(seed, dtype):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    hidden = torch.randn(BATCH, TIME + 1, HIDDEN, generator=gen, device="cuda").to(dtype)
    tokens = torch.randint(0, VOCAB, (BATCH, TIME + 1), generator=gen, device="cuda")
    weight = (torch.randn(VOCAB, HIDDEN, generator=gen, device="cuda") * 0.2).to(dtype)
    lengths = torch.randint(1, TIME + 1, (BATCH, 1), generator=gen, device="cuda")
    mask = torch.arange(TIME, device="cuda").view(1, -1) < lengths
    mask[2] = False
    noise = 0.3 * torch.randn(BATCH, TIME, generator=gen, device="cuda")
    return hidden, tokens, weight, mask, noise, torch.randn(BATCH, generator=gen, device="cuda")


def run_policy(hidden, tokens, weight, mask, noise, advantages, scale):
    """The step through the framework; returns loss and the weights' gradient (still loss-scaled)."""
    leaf = weight.clone().requires_grad_()
    logits = hidden @ leaf.t()
    target = tokens[:, 1:].masked_fill(~mask, -100)
    logp, entropy = bmt.loss.TokenLogProbs(entropy=True)(logits[:, :-1], target)
    old = (logp + noise).detach()
    loss, stats = bmt.loss.PolicyLoss(kl_coef=0.05, entropy_coef=0.01, dual_clip=3.0, reduction="sequence")(
        logp, old, advantages, mask=mask, ref_logprob=(logp - noise).detach(), entropy=entropy)
    manager = bmt.optim.OptimManager(loss_scale=scale)
    manager.backward(loss)
    return loss.detach(), leaf.grad


def plain_policy(hidden, tokens, weight, mask, noise, advantages, scale):
    """The same in 64 bits from the logits the 16-bit product gives."""
    logits = (hidden @ weight.t()).double().requires_grad_()
    logs = logits[:, :-1].log_softmax(-1)
    logp = logs.gather(-1, tokens[:, 1:].unsqueeze(-1)).squeeze(-1)
    entropy = -(logs.exp() * logs).sum(-1)
    shown = torch.where(mask, logp.detach().float(), 0.0)               # what the framework's ignored tokens show
    old, ref = (shown + noise).double(), (shown - noise).double()
    m = mask.double()
    w = m / m.sum(1, keepdim=True).clamp(min=1) / (m.sum(1) > 0).sum()
    r = torch.where(mask, logp - old, 0.0).exp()
    a = advantages.double().unsqueeze(1)
    value = torch.minimum(r * a, r.clamp(0.8, 1.2) * a)
    value = torch.where((a < 0) & (value < 3 * a), 3 * a, value)
    q = torch.where(mask, ref - logp, 0.0)
    loss = (w * (-value + 0.05 * (q.exp() - 1 - q) - 0.01 * entropy)).sum()
    grad, = torch.autograd.grad(loss * scale, logits)
    return loss.detach(), (grad.flatten(0, 1).t() @ hidden.double().flatten(0, 1))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_policy_step(dtype):
    """The logits' gradient is rounded to their type once (relative 2^-11 / 2^-8), products and their sums over the
    tokens add as much again: 4 half steps of the type, relative to the sums of magnitudes (bounded by norms)."""
    data = problem(1, dtype)
    scale = 1024.0
    loss, grad = run_policy(*data, scale)
    want_loss, want = plain_policy(*data, scale)
    assert abs(float(loss) - float(want_loss)) <= 1e-5 * (1 + abs(float(want_loss)))
    assert grad.dtype == dtype and torch.isfinite(grad).all()
    step = max(torch.finfo(dtype).eps, 1e-6)
    assert float((grad.double() - want).norm()) <= 4 * step * float(want.norm())


def test_preference_step_through_clipping_and_adam():
    """Two micro-batches accumulate in fp32, the accumulators are clipped into the 16-bit gradient and stepped: the
    parameters move as they do when the same gradient is clipped by torch operations."""
    dtype = torch.bfloat16
    scale = 64.0
    total = torch.zeros(VOCAB, HIDDEN, device="cuda")
    weight = problem(5, dtype)[2]
    for seed in (5, 6):
        hidden, tokens, _, mask, noise, _ = problem(seed, dtype)
        leaf = weight.clone().requires_grad_()
        logp = bmt.loss.TokenLogProbs()((hidden @ leaf.t())[:, :-1], tokens[:, 1:].masked_fill(~mask, -100))
        loss, chosen, rejected = bmt.loss.PreferenceLoss(beta=0.3)(logp, (logp + noise).detach(), mask)
        (loss * scale).backward()
        assert torch.isfinite(loss) and chosen.shape == (BATCH // 2,)
        total += leaf.grad.float()
    param = torch.nn.Parameter(weight.clone())
    param.grad = torch.empty_like(weight)
    norm = bmt.optim.clip_grads([total], 0.05, scale=scale, out=[param.grad])
    want_norm = float(total.double().norm()) / scale
    assert abs(float(norm) - want_norm) <= 1e-6 * want_norm and want_norm > 0.05
    coef = 0.05 * scale / (want_norm * scale + 1e-6)
    assert torch.allclose(param.grad.double(), total.double() * coef, rtol=2.0 ** -8 * 1.01, atol=1e-30)
    plain = torch.nn.Parameter(weight.clone())
    plain.grad = param.grad.clone()
    for p in (param, plain):
        bmt.optim.AdamOptimizer([p], lr=1e-2).step(scale=scale)
    assert torch.equal(param, plain) and not torch.equal(param, weight)


def test_whole_step_captured():
    """Log-probabilities, loss, both backward passes and the clipping in one graph, replayed on new inputs."""
    dtype = torch.bfloat16
    still = list(problem(1, dtype))
    out = torch.empty(VOCAB, HIDDEN, dtype=dtype, device="cuda")

    def step(hidden, tokens, weight, mask, noise, advantages, out):
        logits = (hidden @ weight.t()).requires_grad_()
        logp, entropy = bmt.loss.TokenLogProbs(entropy=True)(logits, tokens.masked_fill(tokens % 7 == 0, -100))
        loss, stats = bmt.loss.PolicyLoss(entropy_coef=0.1)(logp[:, 1:], (logp[:, 1:] + noise).detach(), advantages, mask, None,
                                                            entropy[:, 1:])
        grad, = torch.autograd.grad(loss, logits)
        whole = grad.flatten(0, 1).t().contiguous() @ hidden.flatten(0, 1)
        return loss.detach(), stats, bmt.optim.clip_grads([whole], 1e-3, out=[out])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*still, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step(*still, out)
    for seed in range(3):
        fresh = problem(30 + seed, dtype)
        for s, f in zip(still, fresh):
            s.copy_(f)
        want_out = torch.empty_like(out)
        want = step(*fresh, want_out)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((*got, out), (*want, want_out)):
            assert torch.equal(a, b), seed


def test_two_streams_at_once():
    """The same modules used by two streams that run at the same time: nothing is shared between the calls."""
    data = [problem(k, torch.bfloat16) for k in (1, 2)]
    want = [run_policy(*d, 256.0) for d in data]
    streams = [torch.cuda.Stream() for _ in data]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(run_policy(*data[k], 256.0))
    torch.cuda.synchronize()
    for k in range(2):
        for loss, grad in got[k]:
            assert torch.equal(loss, want[k][0]) and torch.equal(grad, want[k][1])


def calls():
    """(name, call of one leaf, the leaf, what else is kept for the backward pass)"""
    gen = torch.Generator(device="cuda").manual_seed(5)
    logits = torch.randn(6, 9, 50, generator=gen, device="cuda")
    target = torch.randint(0, 50, (6, 9), generator=gen, device="cuda")
    old, ref = -torch.rand(6, 9, generator=gen, device="cuda"), -torch.rand(6, 9, generator=gen, device="cuda")
    mask = torch.rand(6, 9, generator=gen, device="cuda") < 0.7
    advantages = torch.randn(6, generator=gen, device="cuda")
    logprobs, policy, preference = bmt.loss.TokenLogProbs(entropy=True), bmt.loss.PolicyLoss(kl_coef=0.1), bmt.loss.PreferenceLoss()

    def of_logits(x):
        logprob, entropy = logprobs(x, target)
        return (logprob * old).sum() + (entropy * ref).sum()
    return [("logprobs", of_logits, logits, target), ("policy", lambda x: policy(x, old, advantages, mask, ref)[0], old + 0.1, mask),
            ("preference", lambda x: preference(x, ref, mask)[0], old - 0.1, mask)]


def test_graphs_as_autograd_knows_them():
    """Saved-tensor hooks, recomputation, two backward passes, a second one too many, and changes to what is kept."""
    for name, call, leaf, kept in calls():
        x = leaf.clone().requires_grad_()
        want, = torch.autograd.grad(call(x), x)
        packed = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t.shape) or t.cpu(), lambda t: t.cuda()):
            got, = torch.autograd.grad(call(x), x)
        assert torch.equal(got, want) and len(packed) >= 2, name
        got, = torch.autograd.grad(torch.utils.checkpoint.checkpoint(call, x, use_reentrant=False), x)
        assert torch.equal(got, want), name
        value = call(x)
        first, = torch.autograd.grad(value, x, retain_graph=True)
        second, = torch.autograd.grad(value, x)
        assert torch.equal(first, want) and torch.equal(second, want), name
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(value, x)
        value = call(x)
        kept.add_(0) if kept.dtype != torch.bool else kept.logical_or_(kept)
        with pytest.raises(RuntimeError, match="inplace"):
            torch.autograd.grad(value, x)
        grad, = torch.autograd.grad(call(x), x, torch.ones((), device="cuda", requires_grad=True), create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            grad.sum().backward()
        assert call(x.detach()).grad_fn is None
        with torch.no_grad():
            assert call(x).grad_fn is None
        with torch.inference_mode():
            call(leaf.clone())


def test_transforms_are_refused():
    for name, call, leaf, _ in calls():
        with pytest.raises(RuntimeError):
            torch.func.grad(call)(leaf)
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(torch.stack([leaf, leaf]))
        with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(torch.autograd.forward_ad.make_dual(leaf, leaf))


def test_lazily_negated_views():
    """The imaginary part of a conjugate is a view whose numbers are the memory's, negated."""
    for name, call, leaf, _ in calls():
        z = torch.complex(torch.zeros_like(leaf), -leaf)
        assert z.conj().imag.is_neg() and torch.equal(z.conj().imag, leaf)
        x = leaf.clone().requires_grad_()
        want = call(x)
        grad, = torch.autograd.grad(want, x)
        view = z.conj().imag.requires_grad_()
        got = call(view)
        assert torch.equal(got, want) and torch.equal(torch.autograd.grad(got, view)[0], grad), name
    with pytest.raises(AssertionError, match="negated"):
        bmt.optim.clip_grads([z.conj().imag], 1.0)


def test_two_threads_and_streams():
    """Calls of two threads, each on its own stream, give what one thread gives."""
    import threading
    want = [torch.autograd.grad(call(x), x)[0] for x, call in ((leaf.clone().requires_grad_(), call) for _, call, leaf, _ in calls())]
    torch.cuda.synchronize()
    got = {}

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            mine = calls()
            for _ in range(30):
                xs = [leaf.clone().requires_grad_() for _, _, leaf, _ in mine]
                got[k] = [torch.autograd.grad(call(x), x)[0] for x, (_, call, _, _) in zip(xs, mine)]
        torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for k in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[k], want))


def test_lazily_negated_upstreams():
    """An upstream gradient may be a view whose numbers are the memory's, negated: what complex arithmetic behind a loss
    hands back, and contiguous, so that nothing on the way makes a copy of it."""
    zero = torch.zeros((), device="cuda")
    for name, call, leaf, _ in calls():
        x = leaf.clone().requires_grad_()
        want, = torch.autograd.grad(call(x), x)
        (torch.complex(zero, call(x)).conj() * (1 + 2j)).imag.backward()             # the loss's share of it is -1
        assert torch.equal(x.grad, -want), name
        got, = torch.autograd.grad(call(x), x, torch._neg_view(torch.ones((), device="cuda")))
        assert torch.equal(got, -want), name
    gen = torch.Generator(device="cuda").manual_seed(3)
    for shape in ((4, 7), (1, 1)):
        x = torch.randn(*shape, 700, generator=gen, device="cuda").requires_grad_()
        target = torch.randint(0, 700, shape, generator=gen, device="cuda")
        g, h = [torch.randn(shape, generator=gen, device="cuda") for _ in range(2)]
        out = bmt.loss.TokenLogProbs(entropy=True)(x, target)
        want, = torch.autograd.grad(out, x, (-g, -h), retain_graph=True)
        assert torch._neg_view(g).is_contiguous()
        got, = torch.autograd.grad(out, x, (torch._neg_view(g), torch._neg_view(h)))
        assert torch.equal(got, want)
