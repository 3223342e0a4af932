"""The post-training losses against their formulas in 64 bits, on the GPU, where a short test cannot reach:
every entry of gradients that take the whole GPU, rows that start anywhere, unlikely targets, wide margins.

Tolerances.  u = 2^-24 and ``tol(V) = (96 + V / 64) u`` bound the relative error of a row's sum, of a probability,
and the absolute one of a log-probability's 2^y terms (an exponential off by 2^-22, the rounding of y by at most 64 u for
|y| <= 128, V / 64 + 32 additions).  A coefficient a = dL/dlogp is off by its own formula's share of the
log-probability's error; a stored gradient by half a step of its type besides.
"""

import numpy as np
import pytest
import torch

from ferrite import _native as nat
from ferrite.kernels.distillation import distillation_loss, distillation_loss_and_grad, distillation_loss_reference
from ferrite.kernels.logprobs import token_logprobs
from ferrite.kernels.policy_loss import policy_loss, policy_loss_and_grad
from ferrite.kernels.preference_loss import preference_loss_and_grad

U = 2.0**-24
IGN = -100
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def tol(vocab):
    return (96 + vocab / 64) * U


def stored(g, dtype):
    """What storing g as ``dtype`` may change it by: half a step, and half of the smallest f16."""
    step = {torch.float32: U, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}[dtype]
    return step * g.abs() + (2.0**-25 if dtype == torch.float16 else 1e-38)


def softmax64(x, tau=1.0):
    """(log p, p, H) of rows of logits, in 64 bits."""
    lp = torch.log_softmax(x.double() / tau, 1)
    p = lp.exp()
    return lp, p, -torch.where(p > 0, p * lp, 0.0).sum(1)


def check_policy_grad(grad, x, t, old, adv, w, ref, beta, c, lo=0.2, hi=0.2, tau=1.0):
    """Every entry of the policy loss's gradient, slice by slice: w (a ([i = t] - p) + c p (log p + H)) / tau."""
    vocab = x.shape[1]
    for a in range(0, len(t), 500):
        s = slice(a, a + 500)
        lp, p, h = softmax64(x[s], tau)
        logp = lp.gather(1, t[s, None])[:, 0]
        ratio = (logp - old[s].double()).exp()
        free, held = ratio * adv[s], ratio.clamp(1 - lo, 1 + hi) * adv[s]
        d = ref[s].double() - logp
        co = w[s].double() * (torch.where(held < free, 0.0, -free) - beta * torch.expm1(d))
        one = torch.zeros_like(p)
        one[torch.arange(len(logp), device=x.device), t[s]] = 1.0
        own = c * w[s].double()
        want = (co[:, None] * (one - p) + own[:, None] * p * (lp.clamp_min(-1e5) + h[:, None])) / tau
        # the coefficient's error: that of logp, in exp(logp - old) and exp(ref - logp), and their roundings
        e = tol(vocab) * (1 + logp.abs()) + 4 * U * (1 + old[s].abs() + ref[s].abs())
        amp = co.abs() * tol(vocab) + w[s].double() * (free.abs() + beta * d.exp()) * e
        bound = (amp[:, None] * (p + one) + 2 * tol(vocab) * (co.abs() + own)[:, None] * p * (1 + lp.abs().clamp_max(1e5) + h[:, None])) / tau
        bad = (grad[s].double() - want).abs() > 2 * bound + 1.01 * stored(want, grad.dtype)
        assert not bad.any(), f"{int(bad.sum())} entries off, the first in row {a + int(bad.any(1).nonzero()[0])}"


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,dtype", [(4000, 8203, "bf16"), (3500, 12345, "f16"), (3000, 16001, "bf16"), (3000, 8192, "f16"), (3000, 16384, "bf16")])
@pytest.mark.parametrize("c", [0.0, 0.01])
def test_rows_whose_gradient_runs_behind(rows, vocab, dtype, c):
    """16-bit rows of 16 to 33 KB, several to a CTA, on and off 16-byte boundaries, some masked: every entry of the
    policy gradient, the same bits in every call, and those of a few rows alone."""
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    x = (3 * torch.randn(rows, vocab, device="cuda", generator=g)).to(TORCH[dtype])
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    # rows that differ in everything that reaches their coefficients
    logp = torch.cat([torch.log_softmax(x[a : a + 500].float(), 1).gather(1, t[a : a + 500, None])[:, 0] for a in range(0, rows, 500)])
    old, ref = logp + 0.1 * torch.randn(rows, device="cuda", generator=g), logp + 0.3 * torch.randn(rows, device="cuda", generator=g)
    adv = torch.randn(rows, device="cuda", generator=g)
    w = torch.rand(rows, device="cuda", generator=g) * (torch.rand(rows, device="cuda", generator=g) > 0.1)

    def call(a, b):
        out, grad = policy_loss_and_grad(x[a:b], t[a:b], old[a:b], adv[a:b], w[a:b], ref_logprobs=ref[a:b], kl_coef=0.05, entropy_coef=c)
        return out.logprobs, out.entropy, out.kl, out.clipped, grad

    first = call(0, rows)
    edge = (torch.where(adv > 0, first[0] - old - np.log(1.2), first[0] - old - np.log(0.8))).abs() < 1e-4  # either side of a clipping bound
    keep = ~edge
    check_policy_grad(first[4][keep], x[keep], t[keep], old[keep], adv[keep], w[keep], ref[keep], 0.05, c)
    for _ in range(20):
        assert all(torch.equal(p, q) for p, q in zip(call(0, rows), first))
    for a in range(0, rows, rows // 7):
        b = min(rows, a + 50)
        assert all(torch.equal(p, q[a:b]) for p, q in zip(call(a, b), first))
    nat.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("smooth", [0.0, 0.01, 0.1])
def test_preference_gradient_of_wide_margins(smooth):
    """Pairs of one row each, margins from -20 to 20: d loss / d h = beta (e sigma(x) - (1 - e) sigma(-x)), x = beta h, to a
    few roundings of it -- also where the pair is all but settled.  Relative bounds: x is off by its roundings and those
    of two log-probabilities, which exp turns into a relative error; ten more roundings in the sigmoids."""
    vocab, beta = 16, 0.1
    margins = torch.cat([torch.linspace(-20, 20, 81), torch.tensor([30.0, 60.0, -60.0, 85.0])]).double()
    pairs = len(margins)
    x = torch.zeros(2 * pairs, vocab, device="cuda")
    t = torch.zeros(2 * pairs, dtype=torch.long, device="cuda")
    ref = torch.zeros(2 * pairs)
    ref[1::2] = (margins / beta).float()  # h = -ref_chosen + ref_rejected
    got = (ref[1::2].double() * float(np.float32(beta))).cuda()
    out, grad = preference_loss_and_grad(x, t, ref.cuda(), torch.arange(2 * pairs + 1, device="cuda"), beta=beta, label_smoothing=smooth)
    e = float(np.float32(smooth))
    dh = float(np.float32(beta)) / pairs * (e * torch.sigmoid(got) - (1 - e) * torch.sigmoid(-got))
    bound = (4 * tol(vocab) * beta + 4 * U * got.abs() + 16 * U)  # of each of the two terms
    size = float(np.float32(beta)) / pairs * (e * torch.sigmoid(got) + (1 - e) * torch.sigmoid(-got))
    for sign, rows in ((1.0, grad[0::2]), (-1.0, grad[1::2])):
        for col, share in ((0, 15 / 16), (5, -1 / 16)):
            err = (rows[:, col].double() - sign * share * dh).abs()
            assert (err <= size * abs(share) * (bound + 2 * tol(vocab))).all(), (margins[int((err / size).argmax())], (err / size).max())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,dtype", [(40, 1003, "f16"), (40, 1000, "bf16"), (40, 1004, "f32"), (40, 7000, "f16"), (700, 8200, "f16"), (700, 12000, "bf16"), (40, 32008, "f16"), (40, 32000, "bf16"), (40, 50304, "f32"), (10, 131080, "f16")])
@pytest.mark.parametrize("hide", ["nothing", "inf", "lowest"])
@pytest.mark.parametrize("tau", [1.0, 0.7, 3000.0])
def test_logprobs_have_the_same_bits_from_every_operator(rows, vocab, dtype, hide, tau):
    """Log-probabilities alone, with entropies, and those of the policy loss, with and without a gradient and a bonus:
    one row, one result -- masked columns and rows that end inside a vector among them."""
    ld = -(-vocab // 8) * 8
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = (3 * torch.randn(rows, ld, device="cuda", generator=g)).to(TORCH[dtype])[:, :vocab]
    t = torch.randint(0, vocab // 2, (rows,), device="cuda", generator=g)
    if hide != "nothing":
        low = -float("inf") if hide == "inf" else torch.finfo(TORCH[dtype]).min
        x[:, vocab - vocab // 50 :] = low
        x[::2, vocab // 2 :][torch.rand(len(x[::2]), vocab - vocab // 2, device="cuda", generator=g) < 0.1] = low
    alone = token_logprobs(x, t, temperature=tau)
    assert torch.isfinite(alone).all()
    both, _ = token_logprobs(x, t, temperature=tau, entropy=True)
    assert torch.equal(alone, both)
    f = torch.randn(rows, device="cuda", generator=g)
    assert torch.equal(policy_loss(x, t, alone, f, temperature=tau).logprobs, alone)
    for c in (0.0, 0.01):
        out, _ = policy_loss_and_grad(x, t, alone, f, entropy_coef=c, temperature=tau)
        assert torch.equal(out.logprobs, alone)
    off = torch.tensor([0, rows // 2, rows], device="cuda")
    assert torch.equal(preference_loss_and_grad(x, t, alone, off, temperature=tau)[0].logprobs, alone)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1003, 8203, 50257])
@pytest.mark.parametrize("tau", [1.0, 2.0, 300.0, 3000.0, 1e5])
@pytest.mark.parametrize("level", [0.0, -20000.0, -65000.0, 60000.0])
def test_f16_rows_that_end_inside_a_vector(vocab, tau, level):
    """What stands for the elements past a row's end counts for nothing, whatever the temperature and the logits' level."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = (level + 3 * max(1.0, tau / 30) * torch.randn(6, vocab, device="cuda", generator=g)).clamp(-65504, 65504).half()
    t = torch.randint(0, vocab, (6,), device="cuda", generator=g)
    lp, h = token_logprobs(x, t, temperature=tau, entropy=True)
    want, p, wh = softmax64(x, tau)
    want = want.gather(1, t[:, None])[:, 0]
    # at a level of 65000 k m is rounded to 2^-8 / tau: one number for a row, so it does not show in log p or H
    assert ((lp - want).abs() <= tol(vocab) * (1 + want.abs())).all()
    assert ((h - wh).abs() <= 2 * tol(vocab) * (2 + wh + np.log(vocab))).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("gap", [1.0, 4.0, 8.0, 12.0, 20.0, 30.0, 45.0])
def test_entropy_of_peaked_rows_with_unlikely_targets(gap, dtype):
    """One token ``gap`` above all others, the target among those.  With the base b bits below the row's maximum, b
    at most 10 or 0, log2 s and u / s are near b and off by a few of its roundings; the exponentials' error (2^-22 of what is not
    the top token's share) and a row of 64 sums do not count beside H."""
    g = torch.Generator(device="cuda").manual_seed(int(gap))
    rows, vocab = 512, 64
    x = (0.3 * torch.randn(rows, vocab, device="cuda", generator=g)).to(TORCH[dtype])
    t = torch.randint(0, vocab - 1, (rows,), device="cuda", generator=g)
    x[:, vocab - 1] = gap
    want = softmax64(x)[2]
    lp, h = token_logprobs(x, t, entropy=True)
    out, _ = policy_loss_and_grad(x, t, lp, lp)
    bits = min(10.0, gap / np.log(2)) + 1
    err = (h.double() - want).abs()
    assert (err <= 6 * U * (1 + bits) + 2.0**-18 * want).all(), f"{(err / U).max().item():.1f} u"
    assert (h >= 0).all() and torch.equal(out.entropy, h)


@pytest.mark.gpu
@pytest.mark.parametrize("below", [0.0, 5.0, 10.0, 20.0])
def test_entropy_of_long_rows_with_unlikely_targets(below):
    """32000 normal logits, the target ``below`` their mean: the same roundings as with a likely target.  H is near 11,
    half a step there is 8 u; the sums' errors average out over a row's 128 partial sums to a few u of u / s, about
    8: 32 u for the worst of 256 rows, 10 u in the mean."""
    g = torch.Generator(device="cuda").manual_seed(int(below))
    x = 2.0 * torch.randn(256, 32000, device="cuda", generator=g)
    t = torch.randint(0, 32000, (256,), device="cuda", generator=g)
    x[torch.arange(256), t] = -below
    _, h = token_logprobs(x, t, entropy=True)
    err = (h.double() - softmax64(x)[2]).abs() / U
    assert err.max().item() <= 32 and err.mean().item() <= 10, (err.max().item(), err.mean().item())


def _spread(name, rows, vocab, g):
    """Logits of different shapes, and targets."""
    x = torch.randn(rows, vocab, device="cuda", generator=g)
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    r, n = torch.arange(rows, device="cuda"), torch.randn(rows, device="cuda", generator=g)
    if name.startswith("deviation"):
        return float(name.split()[1]) * x, t
    x = 2.5 * x
    if name == "target ahead":
        x[r, t] = np.log(vocab) + 1 + 2 * n
    elif name == "another ahead":
        x[r, (t + 1) % vocab] = np.log(vocab) + 3 + n
    elif name == "target far below":
        x[r, t] = -60 + 4 * n
    elif name == "likeliest":
        t = x.argmax(1)
    return x, t


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["deviation 0.5", "deviation 1", "deviation 2.5", "deviation 8", "target ahead", "another ahead", "target far below", "likeliest"])
@pytest.mark.parametrize("vocab,tau", [(256, 1.0), (32000, 1.0), (32000, 0.7), (32000, 2.0)])
def test_mean_error_of_logprobs(name, vocab, tau):
    """What goes one way adds up over sequences: on average over 16384 rows a log-probability is off by no more than the
    mean error of the hardware's exponential, 5.1e-8, whatever the logits -- and four standard errors of that mean, of
    roundings that have no sign."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    err = []
    for _ in range(8):
        x, t = _spread(name, 2048, vocab, g)
        lp = token_logprobs(x, t, temperature=tau)
        err.append(lp.double() - softmax64(x, tau)[0].gather(1, t[:, None])[:, 0])
    err = torch.cat(err)
    assert abs(err.mean().item()) <= 5.1e-8 + 4 * err.std().item() / len(err) ** 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("tau", [1.0, 2.0])
def test_distillation_near_the_teacher(tau):
    """Where the student has almost learned the lists, the KL is a sum of small differences: no less exact than plain f32
    operations, which take the differences before the sum."""
    g = torch.Generator(device="cuda").manual_seed(5)
    rows, vocab, top = 4096, 512, 256
    x = 3 * torch.randn(rows, vocab, device="cuda", generator=g)
    v, idx = x.topk(top)
    v = v + 0.02 * torch.randn(rows, top, device="cuda", generator=g)
    lq, lp = torch.log_softmax(v.double() / tau, 1), torch.log_softmax(x.double() / tau, 1).gather(1, idx)
    want = tau**2 * (lq.exp() * (lq - lp)).sum(1)
    plain = distillation_loss_reference(x, v, idx, temperature=tau).per_token.double() - want
    own = distillation_loss(x, v, idx, temperature=tau).per_token.double() - want
    assert own.pow(2).mean().sqrt() <= plain.pow(2).mean().sqrt(), (own.pow(2).mean().sqrt().item(), plain.pow(2).mean().sqrt().item())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,dtype", [(6000, 5003, "f16"), (4000, 12345, "bf16"), (2500, 32003, "bf16"), (2000, 12001, "f32"), (1200, 32001, "f32"), (700, 70001, "f16"), (400, 90001, "f32")])
def test_every_entry_where_the_gpu_is_full(rows, vocab, dtype):
    """Several rows to a CTA in every kernel and layout, off 16-byte boundaries, some masked: every entry of the gradients of
    log-probabilities with entropies, of pairs and of distillation, and the same bits again.  An entry is off by tol of each
    of its parts (and its coefficient's own error), and the store."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = (3 * torch.randn(rows, vocab, device="cuda", generator=g)).to(TORCH[dtype])
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    t[torch.rand(rows, device="cuda", generator=g) < 0.15] = IGN
    live = t != IGN
    a, b = torch.randn(2, rows, device="cuda", generator=g)
    ref = torch.randn(rows, device="cuda", generator=g) - 10
    pairs = 4
    off = torch.linspace(0, rows - 3, 2 * pairs + 1, device="cuda").long()
    top = 40
    v, idx = torch.randn(rows, top, device="cuda", generator=g), torch.randint(0, vocab, (rows, top), device="cuda", generator=g)
    w = torch.rand(rows, device="cuda", generator=g) * (torch.rand(rows, device="cuda", generator=g) > 0.15)

    def logprobs():
        leaf = x.detach().requires_grad_(True)
        return torch.autograd.grad(token_logprobs(leaf, t, entropy=True), leaf, (a, b))[0]

    grads = [logprobs(), preference_loss_and_grad(x, t, ref, off, kind="squared", average=True)[1], distillation_loss_and_grad(x, v, idx, w, temperature=2.0)[1]]
    again = [logprobs(), preference_loss_and_grad(x, t, ref, off, kind="squared", average=True)[1], distillation_loss_and_grad(x, v, idx, w, temperature=2.0)[1]]
    assert all(torch.equal(p, q) for p, q in zip(grads, again))
    # the pairs' coefficients: h is a difference of means of logp - ref, dL / dh = 2 (h - 5)
    step = [(r, min(rows, r + 400)) for r in range(0, rows, 400)]
    logp = torch.cat([softmax64(x[r:q])[0].gather(1, t[r:q].clamp_min(0)[:, None])[:, 0] for r, q in step])
    at = torch.arange(rows, device="cuda")
    inside = (at >= off[:-1, None]) & (at < off[1:, None]) & live
    count = inside.sum(1).clamp_min(1)
    d = torch.where(inside, logp - ref.double(), 0.0).sum(1) / count
    dh = 2 * (d[0::2] - d[1::2] - 5) / pairs
    slope = torch.stack([dh, -dh], 1).reshape(-1) / count
    co = (inside * slope[:, None]).sum(0)
    # logp's error in the mean, and the roundings of h and of the coefficient
    shaky = (inside * (2 / pairs / count * 2 * (tol(vocab) * 40 + 8 * U * 40))[:, None]).sum(0) + 8 * U * co.abs()
    for r, q in step:
        s = slice(r, q)
        lp, p, h = softmax64(x[s])
        one = torch.zeros_like(p)
        one[torch.arange(q - r, device="cuda"), t[s].clamp_min(0)] = 1.0
        on = live[s, None]
        ent = p * (lp.clamp_min(-1e5) + h[:, None])
        at_, bt, ct = a[s, None].double(), b[s, None].double(), co[s, None]
        want = torch.where(on, at_ * (one - p) - bt * ent, 0.0)
        bound = 2 * tol(vocab) * (at_.abs() * (p + one) + bt.abs() * p * (lp.abs() + 3 * h[:, None] + 2)) + 4 * U * at_.abs() * one
        wanted = [(want, bound), (torch.where(on, ct * (one - p), 0.0), (2 * tol(vocab) * ct.abs() + shaky[s, None]) * (p + one))]
        lq = torch.log_softmax(v[s].double() / 2, 1)
        p2 = softmax64(x[s], 2.0)[1]
        q2 = torch.zeros_like(p2).scatter_add_(1, idx[s], lq.exp())
        wt = 2 * w[s, None].double()
        wanted.append((wt * (p2 - q2), 2 * wt * (p2 + q2) * (tol(vocab) + tol(64 * top))))
        for n, ((want, bound), got) in enumerate(zip(wanted, grads)):
            bad = (got[s].double() - want).abs() > bound + 1.01 * stored(want, got.dtype)
            assert not bad.any(), f"gradient {n}: {int(bad.sum())} entries off, the first in row {r + int(bad.any(1).nonzero()[0])}"
    nat.device_status()
