"""The losses over a language model's logits that come after pre-training, as measured cases.

Four operators over logits ``[rows, vocab]``: the log-probabilities of given tokens, the clipped policy
loss with a KL term and an entropy bonus, the preference loss of paired sequences, and distillation from
a teacher's top logits -- each with its gradient.  ``own`` false runs them as elementary torch operations
in 32 bits, ``own`` true through the framework's entry points.
"""

import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_IGNORE = -100
_CLIP_LOW, _CLIP_HIGH = 0.2, 0.28


def _case(name, op, rows, vocab, dtype, **more):
    """One case: sizes and types, plus the defaults of what only some operators look at."""
    c = {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "grad": dtype, "stride": vocab, "masked": 0, "low": 0,
         "tau": 1.0, "grad_scale": 1.0}
    if op == "logprobs":
        c.update(entropy=False)
    elif op == "policy":
        c.update(kl=0.0, entropy=0.0, seqs=max(1, min(8, rows)))
    elif op == "preference":
        c.update(pairs=1, kind="sigmoid", average=False, beta=0.1)
    else:
        c.update(top=16, ragged=False)
    c.update(more)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # scoring the one token that a decode step has just produced (vocabulary 32000, the GPT configuration)
        _case("logprobs 1x32000 bf16", "logprobs", 1, 32000, "bf16", grad=""),
        # reference log-probabilities and entropies of a batch, f32 logits in a buffer padded to a multiple of 64 columns
        _case("logprobs 4096x50257 f32", "logprobs", 4096, 50257, "f32", grad="", stride=50304, entropy=True),
        # a custom loss through autograd: log-probabilities and entropies forward and backward, sampling temperature 0.7
        _case("logprobs grad 2048x32000 bf16", "logprobs", 2048, 32000, "bf16", entropy=True, tau=0.7, masked=300),
        # the byte-level model's training batch (64 x 256 tokens, vocabulary 256)
        _case("policy 16384x256 f32", "policy", 16384, 256, "f32", seqs=64, masked=4096, kl=0.05),
        # one step of policy training on 8 sequences of 1024 tokens, a quarter of them prompt
        _case("policy 8192x32000 bf16", "policy", 8192, 32000, "bf16", seqs=8, masked=2048, kl=0.04),
        # the largest: f32 logits as the tied head writes them, 16-bit gradients as its products take them, entropy bonus
        _case("policy 16384x32000 f32", "policy", 16384, 32000, "f32", grad="bf16", seqs=16, kl=0.04, entropy=0.01),
        # a few short pairs: both passes fit the L2
        _case("preference 517x32000 bf16", "preference", 517, 32000, "bf16", pairs=4, masked=131),
        # a full batch of pairs, a third of it prompts
        _case("preference 16384x32000 bf16", "preference", 16384, 32000, "bf16", pairs=32, masked=5461),
        # odd sizes: length-averaged ratios, squared loss, f16 with a loss scale
        _case("preference 2999x50257 f16", "preference", 2999, 50257, "f16", pairs=8, masked=701, kind="squared", average=True,
              grad_scale=1024.0),
        # a handful of positions, f32 throughout
        _case("distill 64x32000 f32", "distill", 64, 32000, "f32", top=16),
        # a distillation step on 8 x 1024 tokens at temperature 2, lists of uneven length
        _case("distill 8192x32000 bf16", "distill", 8192, 32000, "bf16", top=64, tau=2.0, ragged=True, masked=512),
        # a long vocabulary, long lists, padded columns that hold the type's lowest value
        _case("distill 1000x131072 bf16", "distill", 1000, 131072, "bf16", top=128, low=72),
    ]


def draw(rng):
    op = rng.choice(["logprobs", "policy", "preference", "distill"])
    vocab = int(round(math.exp(rng.uniform(math.log(256), math.log(131072)))))
    if rng.random() < 0.5:
        vocab = max(256, vocab // 64 * 64)
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    grad = "" if op == "logprobs" and rng.random() < 0.5 else dtype
    if op != "logprobs" and dtype == "f32" and rng.random() < 0.5:
        grad = "bf16"
    # no more elements than move two thirds of the largest listed case's bytes
    most = min(16384, int(16384 * 32000 * 4 / (_BYTES[dtype] + _BYTES.get(grad, 0)) / vocab))
    least = 2 if op == "preference" else 1
    rows = max(least, int(round(math.exp(rng.uniform(math.log(least), math.log(max(least + 1, most)))))))
    stride = -(-vocab // 64) * 64 if rng.random() < 0.25 else vocab
    masked = int(rows * rng.choice([0, 0, 0.1, 0.3, 0.6]))
    more = {"grad": grad, "stride": stride, "masked": masked, "low": rng.choice([0, 0, vocab // 50]),
            "tau": rng.choice([1.0, 1.0, 0.7, 2.0]), "grad_scale": 1024.0 if dtype == "f16" else 1.0}
    if op == "logprobs":
        more.update(entropy=rng.random() < 0.5, grad_scale=1.0)
    elif op == "policy":
        more.update(kl=rng.choice([0.0, 0.04, 0.2]), entropy=rng.choice([0.0, 0.0, 0.01]), seqs=max(1, min(rows, rng.choice([1, 8, 64]))))
    elif op == "preference":
        more.update(pairs=max(1, min(rows // 2, int(round(math.exp(rng.uniform(0, math.log(64))))))), kind=rng.choice(["sigmoid", "sigmoid", "squared"]),
                    average=rng.random() < 0.5, beta=rng.choice([0.05, 0.1, 0.5]))
    else:
        more.update(top=min(vocab, int(round(math.exp(rng.uniform(0, math.log(256)))))), ragged=rng.random() < 0.5)
    return _case(None, op, rows, vocab, dtype, **more)


# ---------------------------------------------------------------- inputs


def _masked_rows(starts, ends, masked, rows):
    """The ``masked`` rows that come earliest in their sequences (the prompts), as truth values."""
    place = torch.empty(rows, dtype=torch.float64)
    for a, b in zip(starts, ends):
        place[a:b] = torch.arange(b - a, dtype=torch.float64) / max(1, b - a)
    hide = torch.zeros(rows, dtype=torch.bool)
    hide[torch.sort(place, stable=True).indices[:masked]] = True
    return hide


def _chunks(rows, vocab):
    step = max(1, (1 << 26) // vocab)
    return [(a, min(rows, a + step)) for a in range(0, rows, step)]


def prepare(case, seed):
    rows, vocab, op = case["rows"], case["vocab"], case["op"]
    dtype, dev = _DTYPES[case["dtype"]], "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)

    # logits of a trained model: a broad background, and the token that was written well ahead of it
    buf = torch.empty(rows, case["stride"], dtype=dtype, device=dev)
    targets = torch.randint(0, vocab - case["low"], (rows,), generator=g, device=dev)
    height = math.log(vocab) + 1.0 + 2.0 * torch.randn(rows, generator=g, device=dev)
    logp = torch.empty(rows, device=dev)
    for a, b in _chunks(rows, vocab):
        x = 2.5 * torch.randn(b - a, case["stride"], generator=g, device=dev)
        x[torch.arange(b - a, device=dev), targets[a:b]] = height[a:b]
        if case["low"]:  # the padded end of the vocabulary
            x[:, vocab - case["low"] : vocab] = torch.finfo(dtype).min
        buf[a:b] = x.to(dtype)
        z = buf[a:b, :vocab].float() / case["tau"]
        logp[a:b] = z.gather(1, targets[a:b, None])[:, 0] - torch.logsumexp(z, 1)
    logits = buf[:, :vocab]

    if op == "preference":
        cuts = torch.randperm(rows - 1, generator=host)[: 2 * case["pairs"] - 1].sort().values + 1
        offsets = torch.cat([torch.zeros(1, dtype=torch.long), cuts, torch.tensor([rows])])
    else:
        n = case.get("seqs", 1)
        offsets = torch.arange(n + 1) * rows // n
    hide = _masked_rows(offsets[:-1].tolist(), offsets[1:].tolist(), case["masked"], rows).to(dev)
    state = {"case": case, "logits": logits, "targets": targets}
    live = (~hide).float()
    if op in ("logprobs", "preference"):
        targets[hide] = _IGNORE
    if op == "logprobs":
        state["dlogp"] = torch.randn(rows, generator=g, device=dev)
        state["dentropy"] = 0.1 * torch.randn(rows, generator=g, device=dev)
        if case["grad"]:
            logits.requires_grad_(True)
    elif op == "policy":
        # the policy has moved a little since the tokens were sampled; no ratio sits on a clipping bound
        moved = 0.15 * torch.randn(rows, generator=g, device=dev)
        for edge in (math.log(1 - _CLIP_LOW), math.log(1 + _CLIP_HIGH)):
            moved = torch.where((moved - edge).abs() < 1e-3, torch.full_like(moved, edge + 2e-3), moved)
        state["old"] = logp - moved
        state["ref"] = logp + 0.05 + 0.3 * torch.randn(rows, generator=g, device=dev) if case["kl"] else None
        state["advantages"] = 0.25 + torch.randn(rows, generator=g, device=dev)
        state["weights"] = live / live.sum().clamp_min(1.0)
    elif op == "preference":
        state["ref"] = logp + 0.2 * torch.randn(rows, generator=g, device=dev)
        state["offsets"] = offsets.to(dev)
    else:
        # the teacher's best tokens: near the student's own best, with other values
        values = torch.empty(rows, case["top"], device=dev)
        indices = torch.empty(rows, case["top"], dtype=torch.long, device=dev)
        for a, b in _chunks(rows, vocab):
            x = logits[a:b].float()
            v = (x + 1.5 * torch.randn(x.shape, generator=g, device=dev)).topk(case["top"])
            values[a:b], indices[a:b] = v.values, v.indices
        if case["ragged"]:
            count = torch.randint(1, case["top"] + 1, (rows, 1), generator=g, device=dev)
            indices[torch.arange(case["top"], device=dev)[None, :] >= count] = -1
        state["values"], state["indices"] = values, indices.int()
        state["weights"] = live / live.sum().clamp_min(1.0)
    return state


# ---------------------------------------------------------------- the framework's operators


def _run_own(s):
    root = os.path.join(os.getcwd(), "ferrite-tpu_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from ferrite.kernels.distillation import distillation_loss_and_grad
    from ferrite.kernels.logprobs import token_logprobs
    from ferrite.kernels.policy_loss import policy_loss_and_grad
    from ferrite.kernels.preference_loss import preference_loss_and_grad

    c = s["case"]
    if c["op"] == "logprobs":
        got = token_logprobs(s["logits"], s["targets"], temperature=c["tau"], entropy=c["entropy"])
        got = got if c["entropy"] else (got,)
        if not c["grad"]:
            return got
        (grad,) = torch.autograd.grad(got, [s["logits"]], [s["dlogp"], s["dentropy"]][: len(got)])
        return (*(t.detach() for t in got), grad)
    gd = _DTYPES[c["grad"]]
    if c["op"] == "policy":
        out, grad = policy_loss_and_grad(
            s["logits"], s["targets"], s["old"], s["advantages"], s["weights"], ref_logprobs=s["ref"], clip_low=_CLIP_LOW,
            clip_high=_CLIP_HIGH, kl_coef=c["kl"], entropy_coef=c["entropy"], temperature=c["tau"], grad_scale=c["grad_scale"], grad_dtype=gd)
        return out.loss, out.logprobs, out.entropy, out.kl, out.clipped, grad
    if c["op"] == "preference":
        out, grad = preference_loss_and_grad(
            s["logits"], s["targets"], s["ref"], s["offsets"], beta=c["beta"], kind=c["kind"], label_smoothing=0.05, average=c["average"],
            temperature=c["tau"], grad_scale=c["grad_scale"], grad_dtype=gd)
        return out.loss, out.margins, out.logprobs, grad
    out, grad = distillation_loss_and_grad(
        s["logits"], s["values"], s["indices"], s["weights"], temperature=c["tau"], grad_scale=c["grad_scale"], grad_dtype=gd)
    return out.loss, out.per_token, grad


# ---------------------------------------------------------------- the plain forms


def _softmax(s):
    """z = x / tau, its maximum and sum of exponentials taken per row, as log p and p in 32 bits."""
    z = s["logits"].detach().float() / s["case"]["tau"]
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    return z - torch.log(total), e / total


def _entropy(logp, p):
    return -torch.where(p > 0, p * logp, 0.0).sum(1)


def _one_hot(grad, targets, value):
    """Adds ``value`` at each row's target."""
    grad[torch.arange(grad.shape[0], device=grad.device), targets] += value
    return grad


def _plain_logprobs(s):
    c = s["case"]
    live = s["targets"] != _IGNORE
    t = torch.where(live, s["targets"], 0)
    logp, p = _softmax(s)
    out = [torch.where(live, logp.gather(1, t[:, None])[:, 0], 0.0)]
    if c["entropy"]:
        h = _entropy(logp, p)
        out.append(torch.where(live, h, 0.0))
    if c["grad"]:
        a = torch.where(live, s["dlogp"], 0.0) / c["tau"]
        grad = _one_hot(p * -a[:, None], t, a)
        if c["entropy"]:
            b = torch.where(live, s["dentropy"], 0.0) / c["tau"]
            grad -= b[:, None] * torch.where(p > 0, p * (logp + h[:, None]), 0.0)
        out.append(grad.to(_DTYPES[c["grad"]]))
    return tuple(out)


def _plain_policy(s):
    c = s["case"]
    w, live = s["weights"], s["weights"] != 0
    logp_all, p = _softmax(s)
    logp = logp_all.gather(1, s["targets"][:, None])[:, 0]
    h = _entropy(logp_all, p)
    ratio = torch.exp(logp - s["old"])
    plain, bounded = ratio * s["advantages"], ratio.clamp(1 - _CLIP_LOW, 1 + _CLIP_HIGH) * s["advantages"]
    clipped = bounded < plain
    per = -torch.minimum(plain, bounded)
    a = torch.where(clipped, 0.0, -plain)
    kl = torch.zeros_like(logp)
    if s["ref"] is not None:
        d = s["ref"] - logp
        kl = torch.exp(d) - d - 1
        per = per + c["kl"] * kl
        a = a + c["kl"] * (1 - torch.exp(d))
    per = per - c["entropy"] * h
    loss = torch.where(live, w * per, 0.0).sum()
    a = torch.where(live, w * a, 0.0) * (c["grad_scale"] / c["tau"])
    grad = _one_hot(p * -a[:, None], s["targets"], a)
    if c["entropy"]:
        b = torch.where(live, w, 0.0) * (c["entropy"] * c["grad_scale"] / c["tau"])
        grad += b[:, None] * torch.where(p > 0, p * (logp_all + h[:, None]), 0.0)
    kept = [torch.where(live, v, 0.0) for v in (logp, h, kl)]
    return (loss, *kept, clipped & live, grad.to(_DTYPES[c["grad"]]))


def _plain_preference(s):
    c = s["case"]
    live = s["targets"] != _IGNORE
    t = torch.where(live, s["targets"], 0)
    logp_all, p = _softmax(s)
    logp = torch.where(live, logp_all.gather(1, t[:, None])[:, 0], 0.0)
    # which sequence a row belongs to, as a table of truth values [2 pairs, rows]
    at = torch.arange(c["rows"], device=logp.device)[None, :]
    inside = (at >= s["offsets"][:-1, None]) & (at < s["offsets"][1:, None]) & live[None, :]
    total = torch.where(inside, (logp - s["ref"])[None, :], 0.0).sum(1)
    count = inside.sum(1).clamp_min(1).float() if c["average"] else torch.ones_like(total)
    total = total / count
    h = total[0::2] - total[1::2]
    beta, e = c["beta"], 0.05
    if c["kind"] == "sigmoid":
        per = (1 - e) * torch.log1p(torch.exp(-(beta * h).abs())) + (1 - e) * torch.relu(-beta * h)
        per = per + e * torch.log1p(torch.exp(-(beta * h).abs())) + e * torch.relu(beta * h)
        dh = beta * (torch.sigmoid(beta * h) - (1 - e))
    else:
        per = (h - 0.5 / beta) ** 2
        dh = 2 * (h - 0.5 / beta)
    dh = dh / c["pairs"]
    ds = torch.stack([dh, -dh], 1).reshape(-1) / count
    a = torch.where(inside, ds[:, None], 0.0).sum(0) * (c["grad_scale"] / c["tau"])
    grad = _one_hot(p * -a[:, None], t, a)
    return per.sum() / c["pairs"], beta * h, logp, grad.to(_DTYPES[c["grad"]])


def _plain_distill(s):
    c, tau = s["case"], s["case"]["tau"]
    live = s["weights"] != 0
    listed_ = s["indices"] >= 0
    v = torch.where(listed_, s["values"].float() / tau, -math.inf)
    v = v - v.amax(1, keepdim=True)
    e = torch.exp(v)
    total = e.sum(1, keepdim=True)
    q, logq = e / total, v - torch.log(total)
    logp, p = _softmax(s)
    idx = torch.where(listed_, s["indices"], 0).long()
    kl = torch.where(q > 0, q * (logq - logp.gather(1, idx)), 0.0).sum(1)
    per = torch.where(live, tau * tau * kl, 0.0)
    w = torch.where(live, s["weights"], 0.0)
    grad = p.scatter_add_(1, idx, -q) * (w * (tau * c["grad_scale"]))[:, None]
    return (w * per).sum(), per, grad.to(_DTYPES[c["grad"]])


_PLAIN = {"logprobs": _plain_logprobs, "policy": _plain_policy, "preference": _plain_preference, "distill": _plain_distill}


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------- from the definitions, in 64 bits


def exact(case, seed):
    """The losses as their definitions say, in 64 bits over slices of rows, the gradients by automatic differentiation."""
    s = prepare(case, seed)
    op, tau, rows = case["op"], case["tau"], case["rows"]
    f64 = lambda name: None if s.get(name) is None else s[name].double()  # noqa: E731
    x, targets = s["logits"].detach(), s["targets"]
    live = targets != _IGNORE if op in ("logprobs", "preference") else s["weights"] != 0
    t = targets.clamp_min(0)
    grad = torch.zeros(rows, case["vocab"], dtype=torch.float64, device=x.device) if case["grad"] else None
    old, ref, adv, w = f64("old"), f64("ref"), f64("advantages"), f64("weights")

    def log_softmax(a, b, track):
        z = x[a:b].double().requires_grad_(track)
        return z, torch.log_softmax(z / tau, 1)

    def entropy_of(lp):
        lp = lp.clamp_min(-1e5)  # p is 0 there, and stays so
        return -(lp.exp() * lp).sum(1)

    if op in ("logprobs", "policy"):
        cols = [[], [], [], []]
        total = torch.zeros((), dtype=torch.float64, device=x.device)
        for a, b in _chunks(rows, case["vocab"]):
            z, lp = log_softmax(a, b, bool(case["grad"]))
            on = live[a:b]
            logp, h = lp.gather(1, t[a:b, None])[:, 0], entropy_of(lp)
            if op == "logprobs":
                part = (logp * s["dlogp"][a:b])[on].sum()
                if case["entropy"]:
                    part = part + (h * s["dentropy"][a:b])[on].sum()
                kl, cut = torch.zeros_like(logp), on
            else:
                ratio = (logp - old[a:b]).exp()
                free, held = ratio * adv[a:b], torch.clamp(ratio, 1 - _CLIP_LOW, 1 + _CLIP_HIGH) * adv[a:b]
                cut = (held < free) & on
                d = ref[a:b] - logp if ref is not None else torch.zeros_like(logp)
                kl = torch.expm1(d) - d
                part = (w[a:b] * (-torch.minimum(free, held) + case["kl"] * kl - case["entropy"] * h))[on].sum()
            if case["grad"]:
                grad[a:b] = torch.autograd.grad(part * case["grad_scale"], z)[0]
            total = total + part.detach()
            for c, v in zip(cols, (logp, h, kl, cut)):
                c.append(torch.where(on, v.detach(), torch.zeros_like(v)))
        logp, h, kl, cut = (torch.cat(c) for c in cols)
        if op == "policy":
            return total, logp, h, kl, cut, grad
        return (logp, *([h] if case["entropy"] else []), *([grad] if case["grad"] else []))

    if op == "preference":
        logp = torch.cat([torch.where(live[a:b], log_softmax(a, b, False)[1].gather(1, t[a:b, None])[:, 0], 0.0)
                          for a, b in _chunks(rows, case["vocab"])]).requires_grad_(True)
        ends = s["offsets"].tolist()
        ratios = torch.where(live, logp - ref, 0.0)
        sums = torch.stack([ratios[a:b].sum() for a, b in zip(ends[:-1], ends[1:])])
        if case["average"]:
            sums = sums / torch.stack([live[a:b].sum().clamp_min(1) for a, b in zip(ends[:-1], ends[1:])])
        h, beta = sums[0::2] - sums[1::2], case["beta"]
        if case["kind"] == "sigmoid":
            per = -0.95 * torch.nn.functional.logsigmoid(beta * h) - 0.05 * torch.nn.functional.logsigmoid(-beta * h)
        else:
            per = (h - 0.5 / beta).square()
        loss = per.mean()
        (a_row,) = torch.autograd.grad(loss * case["grad_scale"], logp)
        for a, b in _chunks(rows, case["vocab"]):
            z, lp = log_softmax(a, b, True)
            grad[a:b] = torch.autograd.grad((lp.gather(1, t[a:b, None])[:, 0] * a_row[a:b])[live[a:b]].sum(), z)[0]
        return loss.detach(), (beta * h).detach(), logp.detach(), grad

    total, per = torch.zeros((), dtype=torch.float64, device=x.device), []
    for a, b in _chunks(rows, case["vocab"]):
        z, lp = log_softmax(a, b, True)
        listed_ = s["indices"][a:b] >= 0
        logq = torch.log_softmax(torch.where(listed_, s["values"][a:b].double() / tau, -math.inf), 1)
        picked = lp.gather(1, s["indices"][a:b].clamp_min(0).long())
        kl = torch.where(listed_, logq.exp() * (torch.where(listed_, logq, 0.0) - torch.where(listed_, picked, 0.0)), 0.0).sum(1)
        part = (w[a:b] * tau**2 * kl).sum()
        grad[a:b] = torch.autograd.grad(part * case["grad_scale"], z)[0]
        total = total + part.detach()
        per.append(torch.where(live[a:b], tau**2 * kl.detach(), 0.0))
    return total, torch.cat(per), grad


def work(case):
    """Every live row's logits read once, every row's gradient written once, and what else comes in and goes out by row."""
    rows, vocab = case["rows"], case["vocab"]
    read = (rows - case["masked"]) * vocab
    size = read * _BYTES[case["dtype"]]
    flops = read * (4 + (2 if case.get("entropy") else 0))
    if case["grad"]:
        size += rows * vocab * _BYTES[case["grad"]]
        flops += read * (3 + (2 if case.get("entropy") else 0))
    size += {"logprobs": 16, "policy": 40, "preference": 16, "distill": 8 + 8 * case.get("top", 0)}[case["op"]] * rows
    return {"bytes": size, "flops": flops}
