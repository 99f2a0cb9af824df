"""The operators between a model's logits and its optimizer that preference and policy tuning add, as measured cases.

Four operators, each in its plain form (elementary torch operations) and as the framework's call:

  logprobs    log-probability (and entropy) of given tokens under logits, and the logits' gradient
  policy      clipped policy loss with KL and entropy terms over a padded batch, and its gradients
  preference  loss of paired log-ratio sums (chosen against rejected), and its gradient
  clip        global norm over a list of gradients and the clipped gradients

listed() names the measured cases, draw() makes more of the same ranges, prepare() makes a case's inputs, run() is one
pass, exact() gives the same outputs in 64 bits from the definitions, work() the bytes and operations of a pass.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}


# ---- the cases --------------------------------------------------------------------------------------------------
def listed():
    return [
        # scoring the last few tokens of a batch of answers: one forward call, latency counts
        {"name": "logprobs_few", "op": "logprobs", "batch": 4, "time": 4, "vocab": 32000, "dtype": "fp16", "ignored": 0.0,
         "entropy": True, "temperature": 1.0, "shifted": False, "train": False, "spread": 2.0},
        # a training step on 8 x 2,048 tokens of a 32,000-token vocabulary, a tenth of them padding
        {"name": "logprobs_fp16", "op": "logprobs", "batch": 8, "time": 2048, "vocab": 32000, "dtype": "fp16", "ignored": 0.1,
         "entropy": False, "temperature": 1.0, "shifted": False, "train": True, "spread": 2.0},
        # the same on 8,192 tokens of a 128,256-token vocabulary with an entropy bonus; prompts are not trained on
        {"name": "logprobs_bf16_entropy", "op": "logprobs", "batch": 4, "time": 2048, "vocab": 128256, "dtype": "bf16",
         "ignored": 0.3, "entropy": True, "temperature": 1.0, "shifted": False, "train": True, "spread": 3.0},
        # fp32 logits of an unpadded vocabulary, next-token view logits[:, :-1], sampling temperature 0.7
        {"name": "logprobs_odd_view", "op": "logprobs", "batch": 3, "time": 683, "vocab": 50257, "dtype": "fp32", "ignored": 0.05,
         "entropy": True, "temperature": 0.7, "shifted": True, "train": True, "spread": 2.0},
        # one micro-batch of short answers
        {"name": "policy_small", "op": "policy", "rows": 8, "time": 512, "dtype": "fp32", "ref": True, "entropy": False,
         "token_advantages": False, "dual": 0.0, "reduction": "mean"},
        # a padded batch of long answers, every sequence with the same weight, reference model and entropy bonus
        {"name": "policy_long", "op": "policy", "rows": 1024, "time": 8192, "dtype": "fp32", "ref": True, "entropy": True,
         "token_advantages": False, "dual": 0.0, "reduction": "sequence"},
        # odd lengths, 16-bit log-probabilities, advantages per token, second clip for negative advantages
        {"name": "policy_odd_bf16", "op": "policy", "rows": 37, "time": 4099, "dtype": "bf16", "ref": False, "entropy": False,
         "token_advantages": True, "dual": 3.0, "reduction": "mean"},
        # four pairs of short answers
        {"name": "preference_small", "op": "preference", "pairs": 4, "time": 511, "dtype": "fp32", "kind": "sigmoid",
         "average": False, "smoothing": 0.0},
        # a large batch of long answers, length-normalised
        {"name": "preference_long", "op": "preference", "pairs": 512, "time": 8192, "dtype": "fp32", "kind": "ipo",
         "average": True, "smoothing": 0.0},
        # fp32 accumulators of a small model's four blocks into 16-bit gradients
        {"name": "clip_small", "op": "clip", "blocks": 4, "hidden": 256, "ffn": 688, "dtype": "fp32", "out": "bf16", "norm": 2.0},
        # the gradients of one block of 202,383,360 parameters, 16-bit
        {"name": "clip_block_bf16", "op": "clip", "blocks": 1, "hidden": 4096, "ffn": 11008, "dtype": "bf16", "out": "bf16",
         "norm": 2.0},
        # fp32 accumulators of five such blocks into the 16-bit gradients the optimizer takes
        {"name": "clip_large_fp32", "op": "clip", "blocks": 5, "hidden": 4096, "ffn": 11008, "dtype": "fp32", "out": "bf16",
         "norm": 2.0},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "policy", "preference", "clip", "clip"])
    if op == "logprobs":
        dtype = rng.choice(["fp32", "fp16", "bf16"])
        vocab = _log_uniform(rng, 300, 160000)
        tokens = max(1, min(_log_uniform(rng, 1, 20000), 2_000_000_000 // (vocab * _BYTES[dtype])))
        batch = rng.randint(1, max(1, min(9, tokens)))
        return {"op": op, "batch": batch, "time": max(1, tokens // batch), "vocab": vocab, "dtype": dtype,
                "ignored": rng.choice([0.0, 0.1, 0.5]), "entropy": rng.random() < 0.5,
                "temperature": rng.choice([1.0, 1.0, 0.6, 1.3]), "shifted": rng.random() < 0.3, "train": rng.random() < 0.8,
                "spread": rng.choice([1.0, 2.0, 3.0])}
    if op == "policy":
        time = _log_uniform(rng, 1, 32768)
        return {"op": op, "rows": max(1, min(_log_uniform(rng, 1, 4096), 8_000_000 // time)), "time": time,
                "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"]), "ref": rng.random() < 0.6, "entropy": rng.random() < 0.4,
                "token_advantages": rng.random() < 0.4, "dual": rng.choice([0.0, 3.0]),
                "reduction": rng.choice(["mean", "sequence", "sum"])}
    if op == "preference":
        time = _log_uniform(rng, 1, 32768)
        return {"op": op, "pairs": max(1, min(_log_uniform(rng, 1, 2048), 4_000_000 // time)), "time": time,
                "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"]), "kind": rng.choice(["sigmoid", "ipo", "hinge"]),
                "average": rng.random() < 0.4, "smoothing": rng.choice([0.0, 0.1])}
    hidden = _log_uniform(rng, 33, 4096)
    ffn = hidden * 43 // 16 + rng.randint(0, 1)
    one = 4 * hidden * hidden + 3 * hidden * ffn + 2 * hidden
    blocks = max(1, min(rng.randint(1, 32), 1_000_000_000 // one))
    dtype, out = rng.choice([("fp32", "bf16"), ("fp32", "fp32"), ("fp32", "fp16"), ("bf16", "bf16"), ("fp16", "fp16")])
    return {"op": op, "blocks": blocks, "hidden": hidden, "ffn": ffn, "dtype": dtype, "out": out,
            "norm": rng.choice([2.0, 2.0, math.inf])}


def _tensor_sizes(case):
    h, f = case["hidden"], case["ffn"]
    return ([h * h] * 4 + [h * f] * 3 + [h] * 2) * case["blocks"]


def work(case):
    if case["op"] == "logprobs":
        rows = case["batch"] * case["time"]
        one = case["vocab"] * _BYTES[case["dtype"]]
        read = rows * (1 - case["ignored"]) * one
        nbytes = read + rows * 12 + (rows * (one + 8) if case["train"] else 0)
        return {"bytes": nbytes, "flops": rows * (1 - case["ignored"]) * case["vocab"] * (12 if case["train"] else 5)}
    if case["op"] == "policy":
        n = case["rows"] * case["time"]
        e = _BYTES[case["dtype"]]
        per = e * (3 + (1 if case["ref"] else 0) + (2 if case["entropy"] else 0)) + 1 + (4 if case["token_advantages"] else 0)
        return {"bytes": n * per + case["rows"] * (0 if case["token_advantages"] else 4), "flops": n * 30}
    if case["op"] == "preference":
        n = 2 * case["pairs"] * case["time"]
        return {"bytes": n * (3 * _BYTES[case["dtype"]] + 1), "flops": n * 4}
    n = sum(_tensor_sizes(case))
    return {"bytes": n * (_BYTES[case["dtype"]] + _BYTES[case["out"]]), "flops": n * 3}


# ---- inputs -----------------------------------------------------------------------------------------------------
def _response_mask(rows, time, gen):
    """Padded answers: every row keeps a first part of random length, one row in 32 nothing."""
    lengths = (torch.rand(rows, 1, generator=gen, device="cuda") * time).ceil().clamp(1, time)
    lengths = torch.where(torch.rand(rows, 1, generator=gen, device="cuda") < 1 / 32, 0, lengths)
    return torch.arange(time, device="cuda").view(1, -1) < lengths


def _token_logprobs(rows, time, gen):
    """Log-probabilities as a trained model gives them: most near zero, a long tail."""
    return -torch.empty(rows, time, device="cuda").exponential_(1.2, generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 11)
    dtype = _TYPES[case["dtype"]]
    state = dict(case)
    if case["op"] == "logprobs":
        b, t, v = case["batch"], case["time"], case["vocab"]
        full = torch.empty(b, t + (1 if case["shifted"] else 0), v, dtype=dtype, device="cuda")
        target = torch.randint(0, v, (b, t), generator=gen, device="cuda")
        lift = torch.rand(b, t, 1, generator=gen, device="cuda") * 12
        for i in range(b):                                      # one sequence at a time keeps the fp32 copy small
            full[i].copy_(torch.randn(full.shape[1:], generator=gen, device="cuda").mul_(case["spread"]))
        full[:, :t].scatter_add_(2, target.unsqueeze(2), lift.to(dtype))
        skipped = torch.rand(b, t, generator=gen, device="cuda") < case["ignored"]
        state.update(logits=(full[:, :-1] if case["shifted"] else full).detach(), target=target.masked_fill(skipped, -100))
        if case["train"]:
            state["logits"].requires_grad_()
            scale = 1024.0 / (b * t)
            state["grad_logprob"] = torch.randn(b, t, generator=gen, device="cuda") * scale
            state["grad_entropy"] = torch.full((b, t), -0.01 * scale, device="cuda")
        return state
    if case["op"] == "policy":
        rows, time = case["rows"], case["time"]
        logprob = _token_logprobs(rows, time, gen).to(dtype)
        noise = torch.randn(rows, time, generator=gen, device="cuda")
        state["old"] = (logprob.float() + 0.2 * noise).to(dtype)
        state["mask"] = _response_mask(rows, time, gen)
        advantages = (rows, time) if case["token_advantages"] else (rows,)
        state["advantages"] = torch.randn(advantages, generator=gen, device="cuda")
        state["ref"] = (logprob.float() + 0.3 * torch.randn(rows, time, generator=gen, device="cuda")).to(dtype) if case["ref"] else None
        state["entropy_in"] = None
        if case["entropy"]:
            state["entropy_in"] = (torch.rand(rows, time, generator=gen, device="cuda") * 3).to(dtype).requires_grad_()
        state["logprob"] = logprob.requires_grad_()
        state["scale"] = torch.full((), 1024.0, device="cuda")   # the loss scale arrives as the upstream gradient
        return state
    if case["op"] == "preference":
        rows, time = 2 * case["pairs"], case["time"]
        state["logprob"] = _token_logprobs(rows, time, gen).to(dtype)
        state["ref"] = (state["logprob"].float() + 0.1 * torch.randn(rows, time, generator=gen, device="cuda")).to(dtype)
        state["mask"] = _response_mask(rows, time, gen)
        state["logprob"].requires_grad_()
        state["scale"] = torch.full((), 1024.0, device="cuda")
        return state
    sizes = _tensor_sizes(case)
    state["grads"] = [(torch.randn(n, generator=gen, device="cuda") * 1e-2).to(dtype) for n in sizes]
    state["flat"] = torch.empty(sum(sizes), dtype=_TYPES[case["out"]], device="cuda")    # the optimizer's gradient buffer
    state["outs"] = list(torch.split(state["flat"], sizes))
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------
def run(state):
    op = state["op"]
    if op == "logprobs":
        return _run_logprobs(state)
    if op == "policy":
        return _run_policy(state)
    if op == "preference":
        return _run_preference(state)
    return _run_clip(state)


def _module(s):
    """The loss module of a case, made at its first pass and kept, as a training program does."""
    if "module" not in s:
        from bmtrain_amd import loss
        if s["op"] == "logprobs":
            s["module"] = loss.TokenLogProbs(ignore_index=-100, temperature=s["temperature"], entropy=s["entropy"])
        elif s["op"] == "policy":
            s["module"] = loss.PolicyLoss(clip_low=0.2, clip_high=0.28, dual_clip=s["dual"] or None, kl_coef=0.04,
                                          entropy_coef=0.01, reduction=s["reduction"])
        else:
            smoothing = s["smoothing"] if s["kind"] == "sigmoid" else 0.0        # the other kinds have none
            s["module"] = loss.PreferenceLoss(beta=0.1, kind=s["kind"], label_smoothing=smoothing, average=s["average"])
    return s["module"]


def _run_logprobs(s):
    if own:
        out = _module(s)(s["logits"], s["target"])
        out = out if s["entropy"] else (out,)
        if not s["train"]:
            return out
        upstream = (s["grad_logprob"], s["grad_entropy"])[:len(out)]
        return tuple(o.detach() for o in out) + torch.autograd.grad(out, [s["logits"]], upstream)
    with torch.no_grad():
        keep = s["target"] != -100
        at = torch.where(keep, s["target"], 0).unsqueeze(-1)
        z = s["logits"].float()
        z = z - z.amax(-1, keepdim=True)
        if s["temperature"] != 1.0:
            z = z / s["temperature"]
        logz = z.exp().sum(-1, keepdim=True).log()
        z = z - logz                                             # the log-probability of every token
        logprob = torch.where(keep, z.gather(-1, at).squeeze(-1), 0.0)
        if not s["entropy"] and not s["train"]:
            return (logprob,)
        p = z.exp()
        out = (logprob,)
        g = torch.where(keep, s["grad_logprob"], 0.0).unsqueeze(-1) if s["train"] else None
        if s["entropy"]:
            entropy = -(p * z).sum(-1, keepdim=True)
            out += (torch.where(keep, entropy.squeeze(-1), 0.0),)
            if not s["train"]:
                return out
            h = torch.where(keep, s["grad_entropy"], 0.0).unsqueeze(-1)
            z = (z + entropy) * h                                # dH/dx_j = -p_j (log p_j + H)
            z = -p * (z + g)
        else:
            z = -p * g
        z.scatter_add_(-1, at, g)
        if s["temperature"] != 1.0:
            z = z / s["temperature"]
        return out + (z.to(s["logits"].dtype),)


def _masked(x, mask):
    return torch.where(mask, x, 0.0)


def _run_policy(s):
    if own:
        leaves = [s["logprob"]] + ([s["entropy_in"]] if s["entropy_in"] is not None else [])
        loss, stats = _module(s)(s["logprob"], s["old"], s["advantages"], mask=s["mask"], ref_logprob=s["ref"],
                                 entropy=s["entropy_in"])
        return (loss.detach(), stats) + torch.autograd.grad(loss, leaves, s["scale"])
    with torch.no_grad():
        mask = s["mask"]
        counts = mask.sum(1, keepdim=True)
        if s["reduction"] == "mean":
            weight = torch.ones_like(counts) / counts.sum().clamp(min=1)
        elif s["reduction"] == "sequence":
            weight = torch.where(counts > 0, 1.0 / counts.clamp(min=1), 0.0) / (counts > 0).sum().clamp(min=1)
        else:
            weight = torch.ones_like(counts)
        weight = weight.double()
        a = s["advantages"].double()
        a = a if a.dim() == 2 else a.unsqueeze(1)
        delta = _masked(s["logprob"].double() - s["old"].double(), mask)     # 64 bits: which side of a clip it falls
        ratio = delta.exp()
        surrogate = torch.minimum(ratio * a, ratio.clamp(0.8, 1.28) * a)
        clipped = torch.where(a > 0, ratio > 1.28, (ratio < 0.8) & (a < 0))
        if s["dual"]:
            far = (a < 0) & (ratio > s["dual"])
            surrogate = torch.where(far, s["dual"] * a, surrogate)
            clipped = clipped | far
        grad = torch.where(clipped, 0.0, -a * ratio)
        policy = -surrogate
        old_kl = ratio - 1 - delta
        kl = torch.zeros_like(delta)
        if s["ref"] is not None:
            back = _masked(s["ref"].double() - s["logprob"].double(), mask)
            kl = back.exp() - 1 - back
            grad = grad + 0.04 * (1 - back.exp())
        entropy = _masked(s["entropy_in"].double(), mask) if s["entropy_in"] is not None else torch.zeros_like(delta)
        stats = torch.stack([(_masked(x, mask) * weight).sum() for x in (policy, kl, entropy, clipped.double(), old_kl)])
        loss = stats[0] + 0.04 * stats[1] - 0.01 * stats[2]
        grads = (_masked(grad, mask) * weight * s["scale"]).to(s["logprob"].dtype),
        if s["entropy_in"] is not None:
            grads += (_masked((-0.01 * s["scale"]) * weight, mask).to(s["entropy_in"].dtype),)
        return (loss.float(), stats.float()) + grads


def _run_preference(s):
    if own:
        loss, chosen, rejected = _module(s)(s["logprob"], ref_logprob=s["ref"], mask=s["mask"])
        return (loss.detach(), chosen, rejected) + torch.autograd.grad(loss, [s["logprob"]], s["scale"])
    with torch.no_grad():
        beta, eps, mask = 0.1, s["smoothing"], s["mask"]
        counts = mask.sum(1)
        sums = _masked(s["logprob"].double() - s["ref"].double(), mask).sum(1)
        norm = counts.clamp(min=1).double() if s["average"] else torch.ones_like(sums)
        sums = sums / norm
        chosen, rejected = sums.chunk(2)
        h = chosen - rejected
        used = (counts.view(2, -1).sum(0) > 0).double()
        if s["kind"] == "sigmoid":
            soft = torch.log1p(torch.exp(-(beta * h).abs()))                # -log sigmoid(x) = max(-x, 0) + log(1 + e^-|x|)
            loss = (1 - eps) * ((-beta * h).clamp(min=0) + soft) + eps * ((beta * h).clamp(min=0) + soft)
            slope = beta * (eps - 1 / (1 + torch.exp(beta * h))) if eps else -beta / (1 + torch.exp(beta * h))
        elif s["kind"] == "ipo":
            loss, slope = (h - 0.5 / beta) ** 2, 2 * (h - 0.5 / beta)
        else:
            loss, slope = (1 - beta * h).clamp(min=0), torch.where(beta * h < 1, -beta, 0.0)
        share = used / used.sum().clamp(min=1)
        each = torch.cat([slope * share, -slope * share]) / norm * s["scale"]
        grad = torch.where(mask, each.unsqueeze(1), 0.0).to(s["logprob"].dtype)
        return (loss * share).sum().float(), (beta * chosen).float(), (beta * rejected).float(), grad


def _run_clip(s):
    if own:
        from bmtrain_amd.optim import clip_grads
        norm = clip_grads(s["grads"], max_norm=1.0, norm_type=s["norm"], out=s["outs"])
        return norm, s["flat"]
    with torch.no_grad():
        flat = torch.cat(s["grads"]).float()
        norm = flat.abs().max() if s["norm"] == math.inf else flat.square().sum(dtype=torch.float64).sqrt()
        coef = (1.0 / (norm + 1e-6)).clamp(max=1.0)
        s["flat"].copy_(flat * coef.float())
        return norm.float(), s["flat"]


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"logprobs": _exact_logprobs, "policy": _exact_policy, "preference": _exact_preference,
                "clip": _exact_clip}[case["op"]](s)


def _exact_logprobs(s):
    v = s["vocab"]
    target = s["target"]
    logprob = torch.zeros(target.shape, dtype=torch.float64, device="cuda")
    entropy = torch.zeros_like(logprob)
    grad = torch.zeros(target.shape + (v,), dtype=torch.float64, device="cuda") if s["train"] else None
    step = max(1, 50_000_000 // v)
    for i in range(target.shape[0]):
        for j in range(0, target.shape[1], step):
            t = target[i, j:j + step]
            all_logs = torch.log_softmax(s["logits"][i, j:j + step].double() / s["temperature"], dim=-1)
            prob = torch.exp(all_logs)
            h = -(prob * all_logs).sum(-1)
            valid = (t >= 0).double()
            hot = torch.zeros_like(prob)
            hot[torch.arange(t.numel(), device="cuda"), t.clamp(min=0)] = 1.0
            logprob[i, j:j + step] = valid * (all_logs * hot).sum(-1)
            entropy[i, j:j + step] = valid * h
            if s["train"]:
                d = (hot - prob) * (valid * s["grad_logprob"][i, j:j + step].double()).unsqueeze(-1)
                if s["entropy"]:
                    d -= prob * (all_logs + h.unsqueeze(-1)) * (valid * s["grad_entropy"][i, j:j + step].double()).unsqueeze(-1)
                grad[i, j:j + step] = d / s["temperature"]
    out = (logprob, entropy) if s["entropy"] else (logprob,)
    return out + ((grad,) if s["train"] else ())


def _exact_policy(s):
    rows, time = s["rows"], s["time"]
    zero = torch.zeros(rows, time, dtype=torch.float64, device="cuda")
    m = s["mask"].double()
    new, old = [torch.where(s["mask"], s[k].double(), zero) for k in ("logprob", "old")]
    adv = s["advantages"].double().reshape(rows, -1).expand(rows, time)
    per_row = m.sum(1)
    w = {"sum": lambda: m,
         "mean": lambda: m / max(1.0, float(per_row.sum())),
         "sequence": lambda: m / per_row.clamp(min=1)[:, None] / max(1, int((per_row > 0).sum()))}[s["reduction"]]()
    r = torch.exp(new - old)
    low, high = r >= 0.8, r <= 1.28
    plain, cut = r * adv, torch.clamp(r, 0.8, 1.28) * adv
    value = torch.where(plain <= cut, plain, cut)
    active = (adv == 0) | (torch.where(adv > 0, high, low))
    if s["dual"]:
        floor = s["dual"] * adv
        under = (adv < 0) & (value < floor)
        value, active = torch.where(under, floor, value), active & ~under
    grad = -adv * r * active.double()
    kl, ent = zero, zero
    if s["ref"] is not None:
        q = torch.where(s["mask"], s["ref"].double(), zero) - new
        kl = torch.expm1(q) - q
        grad = grad - 0.04 * torch.expm1(q)
    if s["entropy_in"] is not None:
        ent = s["entropy_in"].double()
    stats = torch.stack([(w * -value).sum(), (w * kl).sum(), (w * ent).sum(), (w * (~active).double()).sum(),
                         (w * (torch.expm1(new - old) - (new - old))).sum()])
    out = (stats[0] + 0.04 * stats[1] - 0.01 * stats[2], stats, grad * w * 1024.0)
    return out + ((-0.01 * 1024.0 * w,) if s["entropy_in"] is not None else ())


def _exact_preference(s):
    p = s["pairs"]
    m = s["mask"].double()
    n = m.sum(1)
    score = ((s["logprob"].double() - s["ref"].double()) * m).sum(1)
    if s["average"]:
        score = score / torch.where(n > 0, n, torch.ones_like(n))
    margin = score[:p] - score[p:]
    x, eps = 0.1 * margin, s["smoothing"]
    if s["kind"] == "sigmoid":
        one = -(1 - eps) * torch.nn.functional.logsigmoid(x) - eps * torch.nn.functional.logsigmoid(-x)
        d = 0.1 * (torch.sigmoid(x) - (1 - eps))
    elif s["kind"] == "ipo":
        one, d = torch.square(margin - 5.0), 2 * margin - 10.0
    else:
        one, d = torch.relu(1 - x), -0.1 * (x < 1).double()
    counted = ((n[:p] + n[p:]) > 0).double()
    total = max(1.0, float(counted.sum()))
    row = torch.cat([d * counted, -d * counted]) / total * 1024.0
    if s["average"]:
        row = row / torch.where(n > 0, n, torch.ones_like(n))
    return (one * counted).sum() / total, 0.1 * score[:p], 0.1 * score[p:], m * row[:, None]


def _exact_clip(s):
    if s["norm"] == math.inf:
        norm = max(float(g.abs().max()) for g in s["grads"])
    else:
        norm = math.sqrt(math.fsum(float((g.double() ** 2).sum()) for g in s["grads"]))
    factor = min(1.0, 1.0 / (norm + 1e-6))
    return torch.tensor(norm, dtype=torch.float64), torch.cat([g.double() * factor for g in s["grads"]])
