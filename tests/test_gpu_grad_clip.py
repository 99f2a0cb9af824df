"""clip_grads and the scaling under OptimManager.clip_grad_norm against the definition in 64 bits.

Tolerances.  The norm is summed in 64 bits and rounded to fp32 once (2^-24; 2^-40 for the sums' own order).  The factor is
one more fp32 rounding, the product another, the rounding to the output's type half a step of that type.
"""
import math

import pytest
import torch

from bmtrain_amd import _tensors
from bmtrain_amd.optim import OptimManager, clip_grads

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -126}


def grads_of(sizes, dtypes, seed, spread=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, generator=gen, device="cuda") * spread).to(dtypes[k % len(dtypes)]) for k, n in enumerate(sizes)]


def reference(grads, max_norm, norm_type=2.0, eps=1e-6, scale=1.0):
    flat = [g.double() for g in grads]
    if norm_type == 2.0:
        norm = math.sqrt(sum(float((g * g).sum()) for g in flat))
    else:
        norm = max((float(g.abs().max()) for g in flat if g.numel()), default=0.0)
    coef = max_norm * scale / (norm + eps) if norm + eps else math.inf
    return norm / scale, [g * coef if coef < 1 else g for g in flat], coef


def check(grads, max_norm, out=None, **options):
    want_norm, want, coef = reference([g.clone() for g in grads], max_norm, **options)
    before = [g.clone() for g in grads]
    norm = clip_grads(grads, max_norm, out=out, **options)
    assert norm.dtype == torch.float32 and norm.shape == () and norm.is_cuda
    assert abs(float(norm) - want_norm) <= (1.01 * U + 2.0 ** -40) * want_norm + 1e-44
    for g, b, o, w in zip(grads, before, grads if out is None else out, want):
        bound = (1.01 * torch.finfo(o.dtype).eps / 2 + 4 * U) * w.abs() + TINY[o.dtype]
        assert ((o.double() - w).abs() <= bound).all(), float((o.double() - w).abs().max())
        if out is not None:
            assert torch.equal(g, b)                                # the gradients stay as they are
        elif coef >= 1:
            assert torch.equal(g, b)
    return norm


SIZES = [[1], [2, 3], [7, 8, 9, 0, 1], [4097], [16383, 16384, 16385], [32767, 32769, 65537], [100] * 97, [5] * 300, [1 << 20, 3, 1 << 18],
         [0], [3_000_001]]


@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.float16,), (torch.bfloat16,),
                                    (torch.float32, torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_in_place_and_norm_types(sizes, dtypes):
    for norm_type in (2.0, math.inf):
        for max_norm in (0.05, 1e9, 0.0):
            check(grads_of(sizes, dtypes, len(sizes)), max_norm, norm_type=norm_type)
    check(grads_of(sizes, dtypes, 5, spread=1024.0), 0.5, scale=1024.0, eps=1e-3)


@pytest.mark.parametrize("source", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("to", [torch.float32, torch.float16, torch.bfloat16])
def test_into_other_tensors(source, to):
    """Fresh outputs, and outputs back to back in one buffer so that most start off every vector boundary."""
    sizes = [1, 7, 64, 4099, 70001, 0, 12345]
    for max_norm in (0.3, 1e9):
        grads = grads_of(sizes, (source,), 3)
        check(grads, max_norm, out=[torch.empty_like(g, dtype=to) for g in grads])
        for shift in (0, 1, 3):
            buffer = torch.full((sum(sizes) + 8,), -7.0, device="cuda").to(to)
            check(grads, max_norm, out=list(torch.split(buffer[shift:shift + sum(sizes)], sizes)))
            assert (buffer[:shift] == -7).all() and (buffer[shift + sum(sizes):] == -7).all()


def test_views_off_every_boundary():
    for dtype in (torch.float32, torch.bfloat16):
        for first in range(9):
            buffer = grads_of([50000], (dtype,), first)[0]
            before = buffer.clone()
            check([buffer[first:first + 33000 + first], buffer[40001:40001 + first]], 0.1)
            assert torch.equal(buffer[:first], before[:first]) and torch.equal(buffer[33000 + 2 * first:40001], before[33000 + 2 * first:40001])


def test_dense_layouts():
    base = grads_of([60 * 70 * 5], (torch.float32,), 1)[0].view(60, 70, 5)
    for view in (base.permute(2, 0, 1), base.transpose(0, 1), base[:, :, :]):
        check([view], 0.1)
        check([view], 0.1, out=[torch.empty_like(view, dtype=torch.bfloat16)])
    with pytest.raises(AssertionError, match="gaps"):
        clip_grads([base[:, ::2]], 1.0)
    with pytest.raises(AssertionError, match="gaps"):
        clip_grads([base[:1].expand(4, 70, 5)], 1.0)
    with pytest.raises(AssertionError, match="strides"):
        clip_grads([base.transpose(0, 1)], 1.0, out=[torch.empty(70, 60, 5, device="cuda")])
    with pytest.raises(AssertionError, match="strides"):
        clip_grads([base], 1.0, out=[torch.empty(70, 60, 5, device="cuda").transpose(0, 1)])
    flat = torch.empty(60 * 70 * 5, device="cuda", dtype=torch.bfloat16)               # contiguous: any shape will do
    clip_grads([base], 0.1, out=[flat])
    want = torch.empty_like(base, dtype=torch.bfloat16)
    clip_grads([base], 0.1, out=[want])
    assert torch.equal(flat, want.flatten())


def test_squares_outside_fp32():
    for scale in (1e-25, 1e25):
        check(grads_of([5000, 77], (torch.float32, torch.bfloat16), 2, spread=scale), scale / 3, eps=0.0)


def test_non_finite_gradients():
    for dtype in (torch.float32, torch.bfloat16):
        grads = grads_of([1000, 2000], (dtype,), 4)
        keep = [g.clone() for g in grads]
        grads[1][77] = float("nan")
        for norm_type in (2.0, math.inf):
            norm = clip_grads(grads, 0.1, norm_type=norm_type)
            assert math.isnan(float(norm)) and torch.equal(grads[0], keep[0])          # a NaN norm clips nothing
        grads[1][77] = float("-inf")
        for norm_type in (2.0, math.inf):
            out = [torch.empty_like(g) for g in grads]
            assert float(clip_grads(grads, 0.1, norm_type=norm_type, out=out)) == math.inf
            assert (out[0] == 0).all() and torch.isnan(out[1][77]) and (out[1][:77] == 0).all()


def test_equal_calls_give_equal_bits_and_graphs_replay():
    grads = grads_of([100_003, 5, 70_000, 1 << 20], (torch.float32, torch.float32, torch.bfloat16), 9)
    outs = [torch.empty_like(g, dtype=torch.bfloat16) for g in grads]

    def step(gs, os):
        return clip_grads(gs, 0.7, out=os)
    first = float(step(grads, outs))
    bits = [o.clone() for o in outs]
    assert float(step(grads, outs)) == first and all(torch.equal(a, b) for a, b in zip(outs, bits))
    still = [g.clone() for g in grads]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(still, outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        norm = step(still, outs)
    for seed in range(4):
        fresh = grads_of([g.numel() for g in grads], (torch.float32, torch.float32, torch.bfloat16), 20 + seed, spread=0.001 if seed == 2 else 1.0)
        for s, f in zip(still, fresh):
            s.copy_(f)
        fresh_outs = [torch.empty_like(o) for o in outs]
        want = step(fresh, fresh_outs)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(outs, fresh_outs)), seed


def test_refusals():
    g = grads_of([100, 50], (torch.float32,), 1)
    with pytest.raises(RuntimeError, match="shares memory"):
        clip_grads([g[0], g[0]], 1.0)
    with pytest.raises(RuntimeError, match="shares memory"):
        clip_grads([g[0][:60], g[0][50:]], 1.0)
    with pytest.raises(RuntimeError, match="shares memory"):
        clip_grads([g[0][:50]], 1.0, out=[g[0][1:51]])
    with pytest.raises(RuntimeError, match="shares memory"):
        clip_grads(g, 1.0, out=[g[0].clone(), g[0][:50]])
    with pytest.raises(RuntimeError, match="shares memory"):
        clip_grads([g[0]], 1.0, out=[g[0].view(torch.bfloat16)[:100]])
    check([g[0], g[0]], 1.0, out=[torch.empty_like(g[0]), torch.empty_like(g[0])])     # read twice, written once each
    with pytest.raises(ValueError, match="float64"):
        clip_grads([g[0].double()], 1.0)
    with pytest.raises(AssertionError, match="numbers of elements"):
        clip_grads([g[0]], 1.0, out=[g[1]])
    assert float(clip_grads([], 1.0)) == 0.0
    assert float(clip_grads([None, g[1]], 1e9, out=[None, torch.empty_like(g[1])])) > 0
    assert float(clip_grads([g[0][:0]], 1.0)) == 0.0


def test_a_table_of_gigabytes():
    """More than 2^31 elements in one tensor: offsets pass 32 bits in both passes."""
    n = (1 << 31) + 12345
    big = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    big[-3:] = 3.0
    big[5] = 4.0
    norm = clip_grads([big, torch.full((9,), 2.0, device="cuda")], 1.0)
    want = math.sqrt(27 + 16 + 36)
    assert abs(float(norm) - want) <= 2 * U * want
    coef = torch.tensor(1.0 / (want + 1e-6)).double()
    for value, k in ((3.0, -1), (3.0, -3), (4.0, 5)):
        assert abs(float(big[k]) - value * float(coef)) <= 2.0 ** -8 * value * float(coef) * 1.01
    assert float(big.sum(dtype=torch.float32)) == float(big[-3:].float().sum() + big[5].float())


@pytest.mark.parametrize("dtypes", [(torch.float16,), (torch.bfloat16,), (torch.float32,), (torch.float32, torch.bfloat16)])
def test_manager_scales_with_the_same_bits(dtypes):
    """OptimManager.clip_grad_norm leaves what `p.grad.mul_(clip_coef)` with a 0-dim fp32 factor leaves, for separate and
    back-to-back gradients, strided ones and a parameter listed twice."""
    for max_norm in (0.01, 1e6):
        params = []
        for k, n in enumerate([7, 4096, 100_001, 64]):
            p = torch.nn.Parameter(torch.zeros(n, device="cuda", dtype=dtypes[k % len(dtypes)]))
            p.grad = grads_of([n], (p.dtype,), k)[0]
            params.append(p)
        wide = grads_of([64 * 10], (dtypes[0],), 77)[0].view(64, 10)
        strided = torch.nn.Parameter(torch.zeros(64, 5, device="cuda", dtype=dtypes[0]))
        strided.grad = wide[:, ::2] if dtypes[0] == torch.float32 else wide[:, :5].contiguous()
        params.append(strided)
        params.append(torch.nn.Parameter(torch.zeros(3, device="cuda", dtype=dtypes[0])))       # without a gradient
        manager = OptimManager(loss_scale=8.0)
        before = [None if p.grad is None else p.grad.clone() for p in params]
        norm = manager.clip_grad_norm([{"params": params}], max_norm)
        total = norm * 8.0
        coef = float(max_norm * 8.0) / (total + 1e-6)
        for p, b in zip(params, before):
            if b is not None:
                want = b.clone().mul_(coef) if coef < 1 else b
                assert torch.equal(p.grad, want)
        twice = torch.nn.Parameter(torch.zeros(1000, device="cuda", dtype=dtypes[0]))
        twice.grad = grads_of([1000], (dtypes[0],), 3)[0]
        b = twice.grad.clone()
        norm = manager.clip_grad_norm([{"params": [twice, twice]}], max_norm)
        coef = float(max_norm * 8.0) / (norm * 8.0 + 1e-6)
        assert torch.equal(twice.grad, b.mul_(coef).mul_(coef) if coef < 1 else b)


def test_tensors_of_every_kind_in_one_list():
    """Views, parameters, leaves, scalars, empty tensors and transposed columns next to each other."""
    base = torch.randn(7, 11, device="cuda")
    grads = [base.clone(), base[2:5], torch.empty(0, 3, device="cuda"), torch.nn.Parameter(torch.ones(5, device="cuda")), torch.ones((), device="cuda"),
             torch.ones(6, device="cuda", requires_grad=True), base.clone()[1:2, :].t(), base.bfloat16()[:, :], torch.ones(9, device="cuda").half()]
    outs = [torch.empty_like(g, dtype=torch.bfloat16) for g in grads]
    with torch.no_grad():
        check(grads, 0.3, out=outs)
        check(grads, 0.3)
    for bad in (base[:, 1:], base.cpu(), base.int(), base.to(torch.complex64)):
        with pytest.raises((AssertionError, ValueError)):
            clip_grads([base, bad], 0.3)
    check([base.clone(), base.bfloat16()], 0.3, out=[torch.empty_like(base), torch.empty_like(base).half()])


def test_autograd_notices_the_write():
    x = torch.full((100,), 2.0, device="cuda", requires_grad=True)
    saved = x.detach().clone()
    y = (saved * x).sum()                                           # keeps `saved` for its backward pass
    clip_grads([saved], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_inference_tensors():
    with torch.inference_mode():
        g = grads_of([1000], (torch.float32,), 3)
        check(g, 0.1)
    check([g[0]], 0.05, out=[torch.empty_like(g[0])])
    clip_grads(g, 0.01)


def test_a_larger_grid_than_one_batch_of_every_type():
    """More tensors than a launch takes, types mixed, outputs of mixed types."""
    sizes = [(k * 37) % 999 + 1 for k in range(500)]
    kinds = (torch.float32, torch.bfloat16, torch.float16, torch.float32, torch.bfloat16)
    grads = grads_of(sizes, kinds, 13)
    check(grads, 0.2, out=[torch.empty_like(g, dtype=kinds[k % 3]) for k, g in enumerate(grads)])
    check(grads, 0.2)


def test_rounded_factor():
    """scale_grads: the factor is rounded to each gradient's type first."""
    coef = torch.tensor(0.123456, device="cuda")
    grads = grads_of([1001, 999, 1003], (torch.float32, torch.bfloat16, torch.float16), 6)
    want = [(g.float() * coef.to(g.dtype).float()).to(g.dtype) for g in grads]
    _tensors.scale_grads(grads, coef)
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_manager_scales_negated_and_empty_gradients_without_a_host_read():
    """A contiguous lazily negated gradient is scaled as its numbers are, an empty one has nothing to scale, and neither
    makes the host wait for the factor."""
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for max_norm in (0.01, 1e6):
            before = grads_of([1000, 1, 77], (dtype,), 8)
            params = [torch.nn.Parameter(torch.zeros(g.numel(), device="cuda", dtype=dtype)) for g in before]
            for p, g in zip(params[:2], before):
                p.grad = torch._neg_view(-g)
                assert p.grad.is_neg() and torch.equal(p.grad, g)
            params[2].grad = before[2].clone()
            empty = torch.nn.Parameter(torch.zeros(0, 3, device="cuda", dtype=dtype))
            empty.grad = torch.zeros_like(empty)
            manager = OptimManager(loss_scale=8.0)
            torch.cuda.set_sync_debug_mode("error")
            try:
                norm = manager.clip_grad_norm([{"params": [*params, empty]}], max_norm)
            finally:
                torch.cuda.set_sync_debug_mode("default")
            coef = float(max_norm * 8.0) / (norm * 8.0 + 1e-6)
            for p, g in zip(params, before):
                assert torch.equal(p.grad, g.mul_(coef) if coef < 1 else g)


def test_what_autograd_allows_to_write():
    """Leaves under no_grad, leaves that are only read, and gradients that carry a graph of their own."""
    leaf = torch.full((100,), 2.0, device="cuda", requires_grad=True)
    out = torch.empty(100, device="cuda")
    check([leaf.detach()], 0.1, out=[out])
    clip_grads([leaf], 0.1, out=[out])                              # read only
    want = out.clone()
    grad, = torch.autograd.grad((leaf ** 3).sum(), leaf, create_graph=True)
    assert grad.requires_grad
    clip_grads([grad], 0.1)
    with torch.no_grad():
        clip_grads([leaf], 0.1)
        assert torch.equal(leaf, want)
        clip_grads([leaf[:50]], 0.01)
