"""PolicyLoss against the definition in 64 bits.

Tolerances.  u = 2^-24.  Per token d = new - old is rounded to fp32 (u |d|), e^d has a relative error of 2 u (1 + |d|), the
products two more roundings: a term is off by at most (8 + 4 |d|) u of its size.  Sums are 64 bits and add nothing, so a
reduced value is off by that share of the reduction of the absolute values, plus one rounding to fp32.  A gradient is
off by the same share of its parts' sizes, four roundings of the weights, and half a step of its own type.
"""
import math

import pytest
import torch

from bmtrain_amd.loss import PolicyLoss

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def make(rows, time, dtype, seed, ref=True, entropy=True, per_token=False, spread=0.4):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")
    logprob = -normal(rows, time).abs()
    lengths = torch.randint(0, time + 1, (rows, 1), generator=gen, device="cuda")
    return {
        "logprob": logprob.to(dtype),
        "old": (logprob + spread * normal(rows, time)).to(dtype),
        "advantages": normal(rows, time) if per_token else normal(rows),
        "mask": torch.arange(time, device="cuda").view(1, -1) < lengths,
        "ref": (logprob + spread * normal(rows, time)).to(dtype) if ref else None,
        "entropy": normal(rows, time).abs().to(dtype) if entropy else None,
    }


def reference(data, clip_low=0.2, clip_high=None, dual_clip=None, kl_coef=0.0, entropy_coef=0.0, reduction="mean", upstream=1.0):
    """(loss, stats, grad of logprob, grad of entropy) and the tolerances of each, from the definition."""
    clip_high = clip_low if clip_high is None else clip_high
    new = data["logprob"].double()
    mask = torch.ones_like(new, dtype=torch.bool) if data["mask"] is None else data["mask"] != 0
    zero = torch.zeros((), dtype=torch.float64, device=new.device)
    d = torch.where(mask, new - data["old"].double(), zero)
    a = data["advantages"].double()
    a = torch.where(mask, a if a.dim() == 2 else a.unsqueeze(1), zero)
    counts = mask.sum(1, keepdim=True).double()
    if reduction == "mean":
        w = mask / counts.sum().clamp(min=1)
    elif reduction == "sequence":
        w = mask / counts.clamp(min=1) / (counts > 0).sum().clamp(min=1)
    else:
        w = mask.double()
    r = d.exp()
    free, bound = r * a, r.clamp(1 - clip_low, 1 + clip_high) * a
    value = torch.minimum(free, bound)
    inside = ((a >= 0) | (r >= 1 - clip_low)) & ((a <= 0) | (r <= 1 + clip_high))
    if dual_clip:
        under = (a < 0) & (r > dual_clip)
        value, inside = torch.where(under, dual_clip * a, value), inside & ~under
    slope = torch.where(inside, -a * r, zero)
    size = (free.abs() + bound.abs()) * (8 + 4 * d.abs())
    kl, kl_size = torch.zeros_like(d), torch.zeros_like(d)
    if data["ref"] is not None:
        q = torch.where(mask, data["ref"].double() - new, zero)
        kl = torch.expm1(q) - q
        kl_size = (torch.expm1(q).abs() + q.abs()) * (8 + 4 * q.abs())
        slope = slope - kl_coef * torch.expm1(q)
    e = torch.zeros_like(d) if data["entropy"] is None else torch.where(mask, data["entropy"].double(), zero)
    old_kl = torch.expm1(d) - d

    def total(x):
        return (w * x).sum()
    stats = torch.stack([total(-value), total(kl), total(e), total((~inside).double()), total(old_kl)])
    loss = stats[0] + kl_coef * stats[1] - entropy_coef * stats[2]
    sizes = torch.stack([total(size), total(kl_size), total(e.abs()), zero, total((torch.expm1(d).abs() + d.abs()) * (8 + 4 * d.abs()))])
    stats_tol = 4 * U * sizes + 4 * U * stats.abs() + 1e-300
    loss_tol = stats_tol[0] + kl_coef * stats_tol[1] + entropy_coef * stats_tol[2] + 4 * U * loss.abs()
    grad = upstream * w * slope
    grad_tol = abs(upstream) * w * (U * (size + kl_coef * kl_size)) + 8 * U * grad.abs()
    return loss, stats, grad, -upstream * entropy_coef * w, loss_tol, stats_tol, grad_tol


def half_step(dtype, want):
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}[dtype]
    return 1.01 * torch.finfo(dtype).eps / 2 * want.abs() + tiny


def check(data, upstream=3.0, **options):
    leaf = data["logprob"].detach().requires_grad_()
    leaves = [leaf]
    if data["entropy"] is not None:
        leaves.append(data["entropy"].detach().requires_grad_())
    loss, stats = PolicyLoss(**options)(leaf, data["old"], data["advantages"], mask=data["mask"], ref_logprob=data["ref"],
                                        entropy=leaves[1] if len(leaves) > 1 else None)
    want = reference(data, upstream=upstream, **options)
    assert loss.dtype == torch.float32 and loss.shape == () and stats.shape == (5,) and not stats.requires_grad
    assert abs(loss.double() - want[0]) <= want[4], (loss, want[0], want[4])
    assert ((stats.double() - want[1]).abs() <= want[5]).all(), (stats, want[1], want[5])
    grads = torch.autograd.grad(loss, leaves, torch.tensor(upstream, device="cuda"))
    for got, exact, tol in zip(grads, want[2:4], (want[6], 8 * U * want[3].abs())):
        assert got.dtype == leaf.dtype and got.shape == leaf.shape
        off = (got.double() - exact).abs()
        assert (off <= tol + half_step(leaf.dtype, exact)).all(), float(off.max())
        if data["mask"] is not None:
            assert (got[data["mask"] == 0] == 0).all()
    return (loss.detach(), stats, *grads)


TYPES = [torch.float32, torch.float16, torch.bfloat16]
FULL = dict(clip_low=0.2, clip_high=0.28, dual_clip=1.6, kl_coef=0.04, entropy_coef=0.01)


@pytest.mark.parametrize("reduction", ["mean", "sequence", "sum"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,time", [(1, 1), (1, 2), (7, 3), (300, 1), (33, 31), (9, 32), (5, 33), (3, 1023), (6, 1024), (3, 1025),
                                       (2, 4095), (3, 4096), (3, 4097), (1, 12289), (2, 20003), (70000, 4), (9000, 40)])
def test_sizes(rows, time, dtype, reduction):
    data = make(rows, time, dtype, rows * 7 + time)
    check(data, reduction=reduction, **FULL)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ref,entropy,per_token,masked", [(False, False, False, False), (True, False, True, True),
                                                          (False, True, True, False), (False, False, True, True),
                                                          (True, True, False, False)])
def test_optional_inputs(dtype, ref, entropy, per_token, masked):
    for rows, time in ((13, 200), (4, 5000)):
        data = make(rows, time, dtype, time, ref, entropy, per_token)
        if not masked:
            data["mask"] = None
        for reduction in ("mean", "sequence"):
            check(data, reduction=reduction, clip_low=0.1, kl_coef=0.1 if ref else 0.0, entropy_coef=0.02 if entropy else 0.0)


@pytest.mark.parametrize("reduction", ["mean", "sequence", "sum"])
@pytest.mark.parametrize("time", [5, 700, 9000])
def test_nothing_under_an_unset_mask_leaves_a_trace(reduction, time):
    """NaN, infinities and the largest values in masked places of every input; rows and whole batches without a token."""
    data = make(6, time, torch.float32, time)
    data["mask"][0] = False
    data["mask"][3] = False
    data["mask"][5, 0] = True
    clean = check(data, reduction=reduction, **FULL)
    garbage = [float("nan"), float("inf"), float("-inf"), torch.finfo(torch.float32).max, torch.finfo(torch.float32).min]
    off = ~data["mask"]
    for k, key in enumerate(("logprob", "old", "ref", "entropy")):
        for j, value in enumerate(garbage):
            pick = off & (torch.arange(time, device="cuda") % 5 == (j + k) % 5)
            data[key] = torch.where(pick, value, data[key])
    data["advantages"][0] = float("nan")
    data["advantages"][3] = float("inf")
    dirty = check({**data, "advantages": torch.where(data["mask"].any(1), data["advantages"], 0.0)}, reduction=reduction, **FULL)
    dirtier = check(data, reduction=reduction, **FULL)
    for a, b, c in zip(clean, dirty, dirtier):
        assert torch.equal(a, b) and torch.equal(a, c)
    data["mask"][:] = False
    loss, stats, *grads = check(data, reduction=reduction, **FULL)
    assert loss == 0 and (stats == 0).all() and all((g == 0).all() for g in grads)


def test_borders_of_the_clips_are_decided_on_the_exact_difference():
    """Ratios a few fp32 steps on either side of every border: which side they fall is that of the exact difference."""
    base, rows = -1.25, []
    for border in (math.log(1.2), math.log(0.8), math.log(2.0)):
        near = torch.tensor(base - border, dtype=torch.float32)
        line = [near]
        for way in (float("inf"), float("-inf")):
            x = near
            for _ in range(6):
                x = torch.nextafter(x, torch.tensor(way))
                line.append(x)
        rows.append(torch.stack(line))
    old = torch.cat(rows).unsqueeze(0).repeat(2, 1).cuda()
    data = {"logprob": torch.full_like(old, base), "old": old, "advantages": torch.tensor([1.0, -1.0], device="cuda"), "mask": None,
            "ref": None, "entropy": None}
    loss, stats, grad = check(data, reduction="sum", dual_clip=2.0)
    d = (data["logprob"].double() - old.double())
    inside = torch.stack([d[0] <= math.log(1.2), (d[1] >= math.log(0.8)) & (d[1] <= math.log(2.0))])
    assert torch.equal(grad != 0, inside) and stats[3] == float((~inside).sum())


def test_terms_without_weight_are_only_measured():
    """kl_coef and entropy_coef 0: an infinite KL or entropy shows in the statistics and nowhere else."""
    data = make(4, 300, torch.float32, 9)
    data["mask"][:, 0] = True
    plain = check({**data, "ref": None, "entropy": None}, reduction="sequence")
    data["ref"][1, 0] = 200.0
    data["entropy"][2, 0] = float("inf")
    leaf = data["logprob"].clone().requires_grad_()
    loss, stats = PolicyLoss(reduction="sequence")(leaf, data["old"], data["advantages"], data["mask"], data["ref"], data["entropy"])
    grad, = torch.autograd.grad(loss, leaf, torch.tensor(3.0, device="cuda"))
    assert torch.equal(loss, plain[0]) and torch.equal(grad, plain[2])
    assert stats[1] == float("inf") and stats[2] == float("inf")
    entropy = data["entropy"].clone().requires_grad_()
    loss, _ = PolicyLoss()(data["logprob"], data["old"], data["advantages"], data["mask"], entropy=entropy)
    grad, = torch.autograd.grad(loss, entropy, torch.tensor(float("inf"), device="cuda"))
    assert (grad == 0).all()


class Stop(torch.autograd.Function):
    """Hands no gradient on, not even zeros."""

    @staticmethod
    def forward(ctx, x):
        return x.clone()

    @staticmethod
    def backward(ctx, upstream):
        return None


def test_no_gradient_from_behind():
    data = make(3, 50, torch.float32, 4)
    leaf = data["logprob"].clone().requires_grad_()
    loss, _ = PolicyLoss()(leaf, data["old"], data["advantages"], data["mask"])
    Stop.apply(loss).backward()
    assert leaf.grad is None or (leaf.grad == 0).all()


def test_small_kl_keeps_its_digits():
    """q around 1e-3 .. 1e-6: e^q - 1 - q = q^2 / 2 (1 + q / 3 + ...), where the plain difference has lost everything."""
    new = torch.full((1, 64), -0.5, device="cuda")
    ref = new + torch.logspace(-6, -0.1, 64, device="cuda")
    data = {"logprob": new, "old": new.clone(), "advantages": torch.zeros(1, device="cuda"), "mask": None, "ref": ref, "entropy": None}
    loss, stats = PolicyLoss(kl_coef=1.0, reduction="sum")(new, data["old"], data["advantages"], ref_logprob=ref)
    q = ref.double() - new.double()
    exact = (torch.expm1(q) - q)
    one = torch.stack([PolicyLoss(kl_coef=1.0, reduction="sum")(new[:, k:k + 1], new[:, k:k + 1], data["advantages"],
                                                                ref_logprob=ref[:, k:k + 1])[0] for k in range(64)])
    assert ((one.double() - exact[0]).abs() <= 24 * U * exact[0]).all()
    assert abs(loss.double() - exact.sum()) <= 24 * U * exact.sum()


@pytest.mark.parametrize("time", [37, 3001])
def test_layouts(time):
    """Row strides, sliced tokens, transposed batches, [sequences, 1] and expanded advantages, masks of other types."""
    data = make(8, time + 5, torch.float32, time, per_token=True)
    plain = {k: v[:, 2:-3].contiguous() for k, v in data.items()}
    want = check(plain, reduction="sequence", **FULL)
    views = {k: v[:, 2:-3] for k, v in data.items()}
    for a, b in zip(check(views, reduction="sequence", **FULL), want):
        assert torch.equal(a, b)
    turned = {k: v.t().contiguous().t() for k, v in plain.items()}
    for a, b in zip(check(turned, reduction="sequence", **FULL), want):
        assert torch.equal(a, b)
    for kind in (torch.uint8, torch.int64, torch.float32):
        for a, b in zip(check({**plain, "mask": plain["mask"].to(kind) * 3}, reduction="sequence", **FULL), want):
            assert torch.equal(a, b)
    per_row = {**plain, "advantages": plain["advantages"][:, 0].contiguous()}
    want = check(per_row, reduction="mean", **FULL)
    expanded = per_row["advantages"].unsqueeze(1).expand(8, time)
    for advantages in (expanded, expanded.contiguous()):
        for a, b in zip(check({**per_row, "advantages": advantages}, reduction="mean", **FULL), want):
            assert torch.equal(a, b)
    module = PolicyLoss(**FULL)
    loss, _ = module(plain["logprob"], plain["old"], per_row["advantages"].unsqueeze(1), plain["mask"], plain["ref"], plain["entropy"])
    assert torch.equal(loss, want[0])                                # [sequences, 1]


def test_partial_gradients():
    data = make(5, 600, torch.float32, 2)
    module = PolicyLoss(**FULL)
    entropy = data["entropy"].clone().requires_grad_()
    loss, _ = module(data["logprob"], data["old"], data["advantages"], data["mask"], data["ref"], entropy)
    only, = torch.autograd.grad(loss, entropy)
    full = check(data, upstream=1.0, **FULL)
    assert torch.equal(only, full[3])
    leaf = data["logprob"].clone().requires_grad_()
    old = data["old"].clone().requires_grad_()                       # a constant of the loss, whatever it requires
    loss, _ = module(leaf, old, data["advantages"], data["mask"], data["ref"], data["entropy"])
    loss.backward()
    assert torch.equal(leaf.grad, full[2]) and old.grad is None
    loss, _ = module(data["logprob"], data["old"], data["advantages"], data["mask"], data["ref"], data["entropy"])
    assert torch.equal(loss, full[0]) and not loss.requires_grad
    loss /= 2                                                        # an output of its own, not a view


def test_empty_batches():
    for shape in ((0, 5), (4, 0), (0, 0)):
        leaf = torch.zeros(shape, device="cuda", requires_grad=True)
        for reduction in ("mean", "sequence", "sum"):
            loss, stats = PolicyLoss(reduction=reduction)(leaf, leaf.detach(), torch.zeros(shape[0], device="cuda"))
            assert loss == 0 and (stats == 0).all()
            grad, = torch.autograd.grad(loss, leaf)
            assert grad.shape == shape
            one_each = torch.zeros(shape[0], 1, device="cuda")
            for advantages in (one_each, one_each.expand(shape), torch.zeros(shape, device="cuda")):
                loss, stats = PolicyLoss(reduction=reduction)(leaf, leaf.detach(), advantages)
                assert loss == 0 and (stats == 0).all()


def test_gradient_against_differences():
    """Central differences of the 64-bit definition away from the clips' corners: off by step^2 / 6 times the third
    derivative (below 1e-7 relative), the fp32 gradient by its own 1e-6."""
    data = make(4, 50, torch.float32, 6, spread=0.05)
    leaf = data["logprob"].clone().requires_grad_()
    loss, _ = PolicyLoss(**FULL)(leaf, data["old"], data["advantages"], data["mask"], data["ref"], data["entropy"])
    grad, = torch.autograd.grad(loss, leaf)
    gen = torch.Generator(device="cuda").manual_seed(4)
    for _ in range(3):
        way, step = torch.randn(4, 50, generator=gen, device="cuda").double(), 1e-5
        up, down = [reference({**data, "logprob": data["logprob"].double() + s * step * way}, **FULL)[0] for s in (1, -1)]
        assert abs(float((grad.double() * way).sum() - (up - down) / (2 * step))) <= 1e-5 * float((grad.double() * way).abs().sum())


def test_equal_calls_give_equal_bits_and_graphs_replay():
    data = make(40, 3000, torch.bfloat16, 11)
    module = PolicyLoss(reduction="sequence", **FULL)
    upstream = torch.tensor(128.0, device="cuda")

    def step(d):
        leaves = [d["logprob"].detach().requires_grad_(), d["entropy"].detach().requires_grad_()]
        loss, stats = module(leaves[0], d["old"], d["advantages"], d["mask"], d["ref"], leaves[1])
        return (loss.detach(), stats, *torch.autograd.grad(loss, leaves, upstream))
    for a, b in zip(step(data), step(data)):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    still = {k: v.clone() for k, v in data.items()}
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(still)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step(still)
    for seed in range(4):
        fresh = make(40, 3000, torch.bfloat16, 50 + seed)
        for k in still:
            still[k].copy_(fresh[k])
        want = step(fresh)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), seed


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,time", [(3, 2), (6, 40), (4, 700), (3, 5000)])
def test_a_class_of_probability_zero_without_a_reference(dtype, rows, time):
    """Tokens whose logit the new policy masks (log-probability -inf): their ratio is 0, and without a reference there is
    no KL to speak of.  Everything but old_kl is what a ratio of e^-200, 0 in fp32, gives."""
    for per_token in (False, True):
        data = make(rows, time, dtype, time, ref=False, entropy=False, per_token=per_token)
        data["mask"] = None
        gone = torch.zeros(rows, time, dtype=torch.bool, device="cuda")
        gone[1, time // 2] = gone[2, 0] = gone[0, time - 1] = True
        outs = []
        for value in (data["old"].float() - 200, torch.full((rows, time), float("-inf"), device="cuda")):
            for kl_coef in (0.0, 0.1):
                leaf = torch.where(gone, value.to(dtype), data["logprob"]).requires_grad_()
                loss, stats = PolicyLoss(kl_coef=kl_coef)(leaf, data["old"], data["advantages"])
                outs.append((loss.detach(), stats, torch.autograd.grad(loss, leaf)[0]))
        for loss, stats, grad in outs:
            assert torch.equal(loss, outs[0][0]) and torch.equal(stats[:4], outs[0][1][:4]) and torch.equal(grad, outs[0][2])
            assert torch.isfinite(loss) and torch.isfinite(grad).all() and stats[1] == 0
        assert outs[-1][1][4] == float("inf")
        for bad in (float("nan"), float("inf")):
            stats = PolicyLoss(kl_coef=0.1)(torch.where(gone, bad, data["logprob"]), data["old"], data["advantages"])[1]
            assert stats[1] == 0 and not torch.isfinite(stats[4])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,time", [(3, 2), (6, 40), (4, 700), (3, 5000)])
def test_no_advantage_and_a_ratio_beyond_fp32(dtype, rows, time):
    """A token without advantage adds nothing to the policy term and its gradient, however far its ratio is from 1: e^100
    is infinite in fp32, the product with 0 is not NaN.  Everything but old_kl is what a ratio of e^2 gives."""
    for per_token in (False, True):
        data = make(rows, time, dtype, time, per_token=per_token)
        data["mask"] = None
        far = torch.zeros(rows, time, dtype=torch.bool, device="cuda")
        far[1, time // 2] = far[1, 0] = far[1, time - 1] = True
        data["advantages"] = torch.where(far if per_token else torch.arange(rows, device="cuda") == 1, 0.0, data["advantages"])
        outs = []
        for gap in (2.0, 100.0):
            leaf = data["logprob"].clone().requires_grad_()
            old = torch.where(far, (data["logprob"].float() - gap).to(dtype), data["old"])
            loss, stats = PolicyLoss(kl_coef=0.1, reduction="sequence")(leaf, old, data["advantages"], None, data["ref"])
            outs.append((loss.detach(), stats, torch.autograd.grad(loss, leaf)[0]))
        (loss, stats, grad), (far_loss, far_stats, far_grad) = outs
        assert torch.isfinite(far_loss) and torch.isfinite(far_grad).all() and far_stats[4] == float("inf")
        assert torch.equal(loss, far_loss) and torch.equal(stats[:4], far_stats[:4]) and torch.equal(grad, far_grad)
        old = torch.where(far, float("-inf"), data["old"])          # what the old policy could not have sampled
        gone, gone_stats = PolicyLoss(kl_coef=0.1, reduction="sequence")(leaf, old, data["advantages"], None, data["ref"])
        assert torch.equal(loss, gone) and torch.equal(stats[:4], gone_stats[:4])
        assert torch.equal(grad, torch.autograd.grad(gone, leaf)[0])
        bad = data["logprob"].clone()
        bad[1, 0] = float("nan")                                    # NaN is no ratio
        assert torch.isnan(PolicyLoss()(bad, data["old"], data["advantages"])[0])
