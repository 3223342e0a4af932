"""The losses over given tokens -- log-probabilities, policy, preference, distillation -- and their gradients.

CPU: the oracle's gradients against central differences of its own losses (64 bits), and every
refusal of the entry points before a device is touched.
GPU (``-m gpu``): the kernels against the oracle on the same (16-bit) inputs.

Tolerances, with u = 2^-24 the rounding unit of f32 and V the vocabulary: a term 2^y is off by 2^-22
(the hardware's bound) and by the rounding of y, at most 64 u for |y| <= 128; a row's sum passes through at
most V / 64 + 32 additions; so a sum, a probability and a log-probability's error (absolute) are within
``tol(V) = (96 + V / 64) u`` -- 2e-6 + V * 9e-10 relative.  Where a formula scales such an error, its test
scales it.  A gradient is rounded once to its type, by at most half the step there: 2^-8 of its value for
bf16 (8 significant bits), 2^-11 (and half a subnormal step, 2^-25) for f16.
"""

import numpy as np
import pytest
import torch

from helpers import BF16, to_numpy, to_torch
from oracle import posttrain as op

from ferrite import _native as nat
from ferrite.kernels.distillation import distillation_loss, distillation_loss_and_grad, distillation_loss_reference
from ferrite.kernels.logprobs import token_logprobs, token_logprobs_reference
from ferrite.kernels.policy_loss import policy_loss, policy_loss_and_grad, policy_loss_reference
from ferrite.kernels.preference_loss import preference_loss, preference_loss_and_grad, preference_loss_reference

U = 2.0**-24
IGN = -100
NP = {"f32": np.float32, "bf16": BF16, "f16": np.float16}
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def tol(vocab):
    return (96 + vocab / 64) * U


def rounding(g, out):
    """What storing g as ``out`` may change it by."""
    return {"f32": U * np.abs(g), "bf16": 2.0**-8 * np.abs(g), "f16": 2.0**-11 * np.abs(g) + 2.0**-25}[out]


def logits_of(rng, rows, vocab, dtype="f32", std=3.0):
    return (std * rng.standard_normal((rows, vocab))).astype(np.float32).astype(NP[dtype])


def check_grad(got, want, a, b, p, h, t, out, vocab, tau=1.0, scale=1.0):
    """|got - want| within the error of its two parts, a ([i = t] - p) and b p (log p + H), and the store."""
    one = np.zeros_like(p)
    rows = np.arange(len(t))
    one[rows, np.clip(t, 0, vocab - 1)] = 1.0
    lp = np.abs(np.where(p > 0, np.log(np.maximum(p, 1e-300)), 0.0))
    size = np.abs(a)[:, None] * (p + one) + np.abs(b)[:, None] * p * (lp + h[:, None] + 2)
    bound = (2 * tol(vocab) * size / tau + U * np.abs(a)[:, None] * one) * scale + rounding(want, out) * 1.01 + 1e-30
    bad = np.abs(to_numpy(got).astype(np.float64) - want) > bound
    assert not bad.any(), f"{bad.sum()} entries off, the first at {np.argwhere(bad)[0]}"


def close(got, want, bound):
    err = np.abs(to_numpy(got).astype(np.float64) - want)
    assert (err <= bound).all(), f"worst {err.max():.3g} at {int(np.argmax(err))}"


# --------------------------------------------------------------------------- CPU: the oracle


def _differences(f, x, at, eps=1e-6):
    out = []
    for r, c in at:
        up, dn = x.copy(), x.copy()
        up[r, c] += eps
        dn[r, c] -= eps
        out.append((f(up) - f(dn)) / (2 * eps))
    return np.array(out)


PLACES = [(0, 0), (0, 3), (1, 5), (2, 2), (3, 1), (4, 6), (5, 0), (5, 6)]


def _small(rng, rows=6, vocab=7):
    x = 1.5 * rng.standard_normal((rows, vocab))
    t = rng.integers(0, vocab, rows)
    return x, t


def test_oracle_gradients_match_differences(rng):
    x, t = _small(rng)
    a, b = rng.standard_normal(6), rng.standard_normal(6)

    def scores(v):
        lp, h = op.token_logprobs(v, t, 0.7)
        return (a * lp + b * h).sum()

    at = tuple(np.array(PLACES).T)
    np.testing.assert_allclose(op.logits_grad(x, t, a, b, 0.7)[at], _differences(scores, x, PLACES), rtol=1e-6, atol=1e-8)

    old = op.token_logprobs(x, t)[0] + np.array([0.0, 0.5, -0.5, 0.05, -0.1, 0.3])
    kw = dict(old=old, adv=np.array([1.0, -1.0, 2.0, -0.3, 0.0, 1.5]), w=np.array([0.2, 0.1, 0.0, 0.4, 0.3, 0.2]), ref=old + 0.2, beta=0.3, c=0.05, tau=1.3)
    g = op.policy(x, t, **kw)["grad"]
    np.testing.assert_allclose(g[at], _differences(lambda v: op.policy(v, t, **kw)["loss"], x, PLACES), rtol=1e-6, atol=1e-8)
    assert not g[2].any()

    off = np.array([0, 2, 3, 3, 6])
    for kind in ("sigmoid", "squared", "hinge"):
        for average in (False, True):
            kw = dict(ref=old, offsets=off, beta=0.4, kind=kind, e=0.1 if kind == "sigmoid" else 0.0, average=average)
            np.testing.assert_allclose(op.preference(x, t, **kw)["grad"][at], _differences(lambda v: op.preference(v, t, **kw)["loss"], x, PLACES), rtol=1e-6, atol=1e-8)

    idx = np.array([[0, 3, 6], [1, 1, 5], [2, -1, 4], [6, 5, 4], [-1, -1, -1], [3, 2, 0]])
    v = rng.standard_normal((6, 3))
    v[5, 1] = -np.inf
    kw = dict(values=v, indices=idx, w=np.array([1.0, 0.5, 0.2, 0.0, 1.0, 0.7]), tau=2.0)
    g = op.distill(x, **kw)["grad"]
    np.testing.assert_allclose(g[at], _differences(lambda u: op.distill(u, **kw)["loss"], x, PLACES), rtol=1e-6, atol=1e-8)
    assert not g[3].any() and not g[4].any()


def test_plain_forms_match_the_oracle(rng):
    x, t = _small(rng, 6, 7)
    t[1] = IGN
    xt, tt = torch.from_numpy(x), torch.from_numpy(t)
    lp, h = op.token_logprobs(x, t, 0.7)
    glp, gh = token_logprobs_reference(xt, tt, 0.7)
    np.testing.assert_allclose(glp, lp, rtol=1e-5, atol=1e-6)
    np.testing.assert_allclose(gh, h, rtol=1e-5, atol=1e-6)
    old, adv, w, ref = rng.standard_normal(6) - 2, rng.standard_normal(6), rng.random(6), rng.standard_normal(6) - 2
    want = op.policy(x, t, old, adv, w, ref, beta=0.1, c=0.01)
    xg = xt.clone().requires_grad_(True)
    got = policy_loss_reference(xg, tt, *(torch.from_numpy(v) for v in (old, adv, w)), ref_logprobs=torch.from_numpy(ref), kl_coef=0.1, entropy_coef=0.01)
    got.loss.backward()
    assert float(got.loss.detach()) == pytest.approx(want["loss"], rel=1e-5)
    np.testing.assert_allclose(xg.grad, want["grad"], rtol=1e-4, atol=1e-6)
    off = np.array([0, 2, 3, 5, 6])
    want = op.preference(x, t, ref, off, e=0.1)
    got = preference_loss_reference(xt, tt, torch.from_numpy(ref), torch.from_numpy(off), label_smoothing=0.1)
    assert float(got.loss) == pytest.approx(want["loss"], rel=1e-5)
    idx = np.array([[0, 3], [1, 1], [-1, -1], [6, 5], [2, -1], [3, 2]])
    v = rng.standard_normal((6, 2))
    want = op.distill(x, v, idx, w, 2.0)
    got = distillation_loss_reference(xt, torch.from_numpy(v), torch.from_numpy(idx), torch.from_numpy(w), temperature=2.0)
    assert float(got.loss) == pytest.approx(want["loss"], rel=1e-5)
    np.testing.assert_allclose(got.per_token, want["per_token"], rtol=1e-4, atol=1e-6)


def test_rounding_bound_is_that_of_the_types(rng):
    """The bound for storing a value covers numpy's own rounding of it, and is reached to within a few percent."""
    g = rng.standard_normal(200000)
    for out in ("f32", "bf16", "f16"):
        first = 0.0 if out == "f32" else U * np.abs(g)  # numpy rounds to f32 on the way to a 16-bit type
        share = np.abs(g.astype(np.float32).astype(NP[out]).astype(np.float64) - g) / (rounding(g, out) + first)
        assert 0.9 < share.max() <= 1.0


# --------------------------------------------------------------------------- CPU: refusals


def test_cpu_tensors_are_refused():
    x, t, f = torch.zeros(4, 8), torch.zeros(4, dtype=torch.long), torch.zeros(4)
    off = torch.tensor([0, 2, 4])
    for call in (
        lambda: token_logprobs(x, t),
        lambda: policy_loss(x, t, f, f),
        lambda: policy_loss_and_grad(x, t, f, f),
        lambda: preference_loss(x, t, f, off),
        lambda: preference_loss_and_grad(x, t, f, off),
        lambda: distillation_loss(x, torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32)),
        lambda: distillation_loss_and_grad(x, torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32)),
    ):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_python_refusals():
    x, t, f = torch.zeros(4, 8), torch.zeros(4, dtype=torch.long), torch.zeros(4)
    off, v, i = torch.tensor([0, 2, 4]), torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32)
    bad = [
        (ValueError, lambda: token_logprobs(x[0], t)),  # not 2-D
        (ValueError, lambda: token_logprobs(x, t[:3])),
        (ValueError, lambda: token_logprobs(torch.zeros(8, 4).t(), t)),  # column stride
        (ValueError, lambda: token_logprobs(torch.zeros(1, 8).expand(4, 8), t)),  # rows overlap
        (TypeError, lambda: token_logprobs(x, f)),  # float targets
        (TypeError, lambda: token_logprobs(x.double(), t)),
        (ValueError, lambda: token_logprobs(x, t, temperature=0.0)),
        (ValueError, lambda: token_logprobs(x, t, temperature=float("nan"))),
        (ValueError, lambda: policy_loss(x, t, f[:3], f)),
        (ValueError, lambda: policy_loss(x, t, f, f, f[:2])),
        (TypeError, lambda: policy_loss(x, t, t, f)),
        (ValueError, lambda: policy_loss(x, t, f, f, clip_low=-0.1)),
        (TypeError, lambda: policy_loss_and_grad(x.bfloat16(), t, f, f, grad_dtype=torch.float32)),
        (TypeError, lambda: policy_loss_and_grad(x, t, f, f, grad_dtype=torch.float64)),
        (ValueError, lambda: preference_loss(x, t, f, torch.tensor([0, 4]))),  # not pairs
        (ValueError, lambda: preference_loss(x, t, f, torch.tensor([0, 1, 2, 4]))),
        (TypeError, lambda: preference_loss(x, t, f, f[:3])),
        (ValueError, lambda: preference_loss(x, t, f, off, kind="ranking")),
        (ValueError, lambda: preference_loss(x, t, f, off, beta=0.0)),
        (ValueError, lambda: preference_loss(x, t, f, off, label_smoothing=0.5)),
        (ValueError, lambda: distillation_loss(x, v[:3], i[:3])),
        (ValueError, lambda: distillation_loss(x, v, i[:, :1])),
        (ValueError, lambda: distillation_loss(x, torch.zeros(4, 0), torch.zeros(4, 0, dtype=torch.int32))),
        (ValueError, lambda: distillation_loss(x, torch.zeros(4, 1025), torch.zeros(4, 1025, dtype=torch.int32))),
        (TypeError, lambda: distillation_loss(x, v, v)),
        (TypeError, lambda: distillation_loss(x, v.double(), i)),
    ]
    for n, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f"case {n} was accepted")


def test_capi_refusals_without_a_gpu(monkeypatch):
    lib = nat.lib()

    def fwd(logits=16, targets=16, logp=16, stats=16, rows=2, vocab=8, ld=8, temp=1.0, dtype=nat.BF16, tdt=1):
        return lib.ferrite_logprobs_fwd(None, logits, targets, logp, None, stats, rows, vocab, ld, IGN, temp, dtype, tdt)

    assert fwd(rows=-1) == nat.BAD_SHAPE and fwd(vocab=0) == nat.BAD_SHAPE and fwd(ld=7) == nat.BAD_SHAPE
    assert fwd(temp=0.0) == nat.BAD_SHAPE and fwd(temp=float("inf")) == nat.BAD_SHAPE and "temperature" in nat.last_error()
    assert fwd(temp=1e-39) == nat.BAD_SHAPE
    assert fwd(dtype=7) == nat.UNSUPPORTED_DTYPE and fwd(tdt=2) == nat.UNSUPPORTED_DTYPE
    assert fwd(logits=None) == nat.BAD_SHAPE and "null" in nat.last_error()
    assert fwd(logits=17) == nat.BAD_ALIGNMENT and fwd(stats=12) == nat.BAD_ALIGNMENT
    assert fwd(rows=0) == nat.OK

    def bwd(dtype=nat.BF16, out=nat.BF16, ld_out=8, ent=None, dent=None, rows=2):
        return lib.ferrite_logprobs_bwd(None, 16, 16, 16, ent, 16, dent, None, 1.0, 16, rows, 8, 8, ld_out, IGN, 1.0, dtype, 1, out)

    assert bwd(out=nat.F32) == nat.UNSUPPORTED_DTYPE and bwd(out=-1) == nat.UNSUPPORTED_DTYPE
    assert bwd(ld_out=7) == nat.BAD_SHAPE and bwd(dent=16) == nat.BAD_SHAPE
    assert bwd(rows=0) == nat.OK

    def pol(ws=8, lo=0.2, loss=16, grad=16, out=nat.BF16):
        return lib.ferrite_policy_loss(None, 16, 16, 16, None, None, None, lo, 0.2, 0.0, 0.0, 1.0, None, 1.0, loss, 16, 16, 16, 16, grad, 16, ws, 2, 8, 8, 8, IGN, nat.BF16, 1, out)

    assert pol(ws=7) == nat.WORKSPACE_TOO_SMALL and pol(lo=-0.1) == nat.BAD_SHAPE and pol(loss=None) == nat.BAD_SHAPE
    assert pol() == nat.BAD_SHAPE and "null" in nat.last_error()  # advantages missing
    assert pol(out=nat.F16) == nat.UNSUPPORTED_DTYPE

    def prf(beta=0.1, e=0.0, kind=0, ws=4, pairs=1, off=16):
        return lib.ferrite_preference_pairs(None, 16, 16, None, off, beta, e, kind, 0, 16, 16, 16, 16, ws, 2, pairs, IGN, 1)

    assert prf(beta=0.0) == nat.BAD_SHAPE and prf(e=0.5) == nat.BAD_SHAPE and prf(kind=3) == nat.BAD_SHAPE
    assert prf(ws=3) == nat.WORKSPACE_TOO_SMALL and prf(pairs=0) == nat.BAD_SHAPE and prf(off=None) == nat.BAD_SHAPE

    def dst(top=2, ldl=2, vdt=nat.F32, idt=0, ws=8, vals=16):
        return lib.ferrite_distill_loss(None, 16, vals, 16, None, 1.0, None, 1.0, 16, 16, 16, 16, ws, 2, 8, top, 8, 8, ldl, nat.F32, vdt, idt, nat.F32)

    assert dst(top=0) == nat.BAD_SHAPE and dst(top=1025, ldl=1025) == nat.BAD_SHAPE and dst(ldl=1) == nat.BAD_SHAPE
    assert dst(vdt=5) == nat.UNSUPPORTED_DTYPE and dst(idt=2) == nat.UNSUPPORTED_DTYPE
    assert dst(ws=7) == nat.WORKSPACE_TOO_SMALL and dst(vals=None) == nat.BAD_SHAPE
    for name, call in (("logprobs_fwd", fwd), ("logprobs_bwd", bwd), ("policy_loss", pol), ("preference_pairs", prf), ("distill_loss", dst)):
        monkeypatch.setenv("FERRITE_FAULT_INJECT", name)
        assert call() == nat.INJECTED_FAULT


# --------------------------------------------------------------------------- GPU: parity

SHAPES = [(1, 1, "f32"), (3, 2, "bf16"), (5, 7, "f16"), (4, 255, "f32"), (9, 256, "bf16"), (2, 257, "bf16"), (33, 1001, "f16"), (6, 4096, "f32"),
          (5, 32000, "bf16"), (3, 32001, "f32"), (2, 50257, "f16"), (2, 131072, "bf16"), (1, 131075, "f32"), (1, 300000, "f32"), (1, 500001, "bf16")]


def on_gpu(x, stride=None, shift=0):
    """x on the device as a view of rows ``stride`` apart that starts ``shift`` elements into a buffer of NaN."""
    rows, vocab = x.shape
    if not stride and not shift:
        return to_torch(x)
    stride = stride or vocab
    buf = torch.full((rows * stride + shift,), float("nan"), dtype=TORCH[next(k for k, v in NP.items() if np.dtype(v) == x.dtype)], device="cuda")
    view = buf[shift:].view(rows, stride)[:, :vocab]
    view.copy_(to_torch(x))
    return view


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,dtype", SHAPES)
@pytest.mark.parametrize("tau", [1.0, 0.7])
def test_logprobs_forward_and_backward(rows, vocab, dtype, tau):
    rng = np.random.default_rng(rows * vocab)
    x, t = logits_of(rng, rows, vocab, dtype), rng.integers(0, vocab, rows)
    xt = to_torch(x).requires_grad_(True)
    lp, h = token_logprobs(xt, torch.from_numpy(t).cuda(), temperature=tau, entropy=True)
    want, wh = op.token_logprobs(x, t, tau)
    close(lp, want, tol(vocab) * (1 + np.abs(want)))
    close(h, wh, 2 * tol(vocab) * (2 + wh + np.log(vocab)))
    a, b = rng.standard_normal(rows), rng.standard_normal(rows)
    (g,) = torch.autograd.grad([lp, h], [xt], [torch.from_numpy(v).float().cuda() for v in (a, b)])
    a, b = a.astype(np.float32).astype(np.float64), b.astype(np.float32).astype(np.float64)
    assert g.dtype == xt.dtype
    p = np.exp(op.log_softmax(x, tau))
    check_grad(g, op.logits_grad(x, t, a, b, tau), a, b, p, wh + 2 * np.log(vocab), t, dtype, vocab, tau)
    alone = token_logprobs(xt, torch.from_numpy(t.astype(np.int32)).cuda(), temperature=tau)
    assert torch.equal(alone, lp)


def _policy_inputs(rng, x, t, tau):
    rows = len(t)
    lp, _ = op.token_logprobs(x, t, tau)
    old = (lp - 0.3 * rng.standard_normal(rows)).astype(np.float32)
    ref = (lp + 0.5 * rng.standard_normal(rows)).astype(np.float32)
    adv, w = rng.standard_normal(rows).astype(np.float32), rng.random(rows).astype(np.float32)
    return old, adv, w, ref


def _check_policy(out, grad, want, x, t, w, adv, old, vocab, tau, outdt, scale=1.0, beta=0.0, c=0.0):
    e = tol(vocab) * (1 + np.abs(want["logp"]))
    close(out.logprobs, want["logp"], e)
    close(out.entropy, want["entropy"], 2 * tol(vocab) * (2 + want["entropy"] + np.log(vocab)))
    kexp = np.abs(want["kl"]) + 2
    close(out.kl, want["kl"], e * kexp * 2 + 8 * U * kexp)
    assert np.array_equal(to_numpy(out.clipped), want["clipped"])
    ratio = np.exp(want["logp"] - old)
    slack = np.abs(w) * (np.abs(adv) * ratio + beta * kexp) * (2 * e + 8 * U) + np.abs(w) * c * 2 * tol(vocab) * (2 + want["entropy"] + np.log(vocab))
    close(out.loss, want["loss"], slack.sum() + 1e-12)
    if grad is not None:
        p = np.nan_to_num(np.exp(op.log_softmax(x, tau)))
        amp = np.abs(want["a"]) + np.abs(w) * (np.abs(adv) * ratio + beta * kexp) * 2  # the coefficient's own error scales with its parts
        check_grad(grad, want["grad"] * scale, amp, want["b"], p, want["entropy"] + 2 * np.log(vocab), t, outdt, vocab, tau, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,dtype", SHAPES)
@pytest.mark.parametrize("beta,c,tau", [(0.0, 0.0, 1.0), (0.2, 0.02, 0.7)])
def test_policy_loss(rows, vocab, dtype, beta, c, tau):
    rng = np.random.default_rng(rows * vocab + 1)
    x, t = logits_of(rng, rows, vocab, dtype), rng.integers(0, vocab, rows)
    old, adv, w, ref = _policy_inputs(rng, x, t, tau)
    want = op.policy(x, t, old.astype(float), adv.astype(float), w.astype(float), ref.astype(float) if beta else None, 0.2, 0.3, beta, c, tau)
    dev = [torch.from_numpy(v).cuda() for v in (old, adv, w)]
    kw = dict(ref_logprobs=torch.from_numpy(ref).cuda() if beta else None, clip_low=0.2, clip_high=0.3, kl_coef=beta, entropy_coef=c, temperature=tau)
    xt, tt = to_torch(x), torch.from_numpy(t).cuda()
    for outdt in {"f32": ("f32", "bf16", "f16")}.get(dtype, (dtype,)):
        out, grad = policy_loss_and_grad(xt, tt, *dev, grad_dtype=TORCH[outdt], grad_scale=64.0, **kw)
        _check_policy(out, grad, want, x, t, w, adv, old, vocab, tau, outdt, 64.0, beta, c)
    xg = xt.clone().requires_grad_(True)
    auto = policy_loss(xg, tt, *dev, **kw)
    assert torch.equal(auto.loss, out.loss) and torch.equal(auto.logprobs, out.logprobs) and not auto.kl.requires_grad
    (64.0 * auto.loss).backward()
    same = grad if dtype != "f32" else policy_loss_and_grad(xt, tt, *dev, grad_scale=64.0, **kw)[1]
    assert torch.equal(xg.grad, same)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,dtype", SHAPES)
@pytest.mark.parametrize("kind,average", [("sigmoid", False), ("squared", True), ("hinge", False)])
def test_preference_loss(rows, vocab, dtype, kind, average):
    rng = np.random.default_rng(rows * vocab + 2)
    x, t = logits_of(rng, rows, vocab, dtype), rng.integers(0, vocab, rows)
    t[rng.random(rows) < 0.2] = IGN
    ref = (op.token_logprobs(x, t)[0] + 0.3 * rng.standard_normal(rows)).astype(np.float32)
    pairs = max(1, rows // 4)
    off = np.sort(rng.integers(0, rows + 1, 2 * pairs + 1))  # empty sequences, rows outside all of them
    e = 0.1 if kind == "sigmoid" else 0.0
    want = op.preference(x, t, ref.astype(float), off, 0.3, kind, e, average)
    xt, tt, rt, ot = to_torch(x), torch.from_numpy(t).cuda(), torch.from_numpy(ref).cuda(), torch.from_numpy(off).cuda()
    kw = dict(beta=0.3, kind=kind, label_smoothing=e, average=average)
    lp_err = tol(vocab) * (1 + np.abs(want["logp"])) + U * np.abs(ref)
    h_err = lp_err.sum()
    for outdt in {"f32": ("f32", "bf16")}.get(dtype, (dtype,)):
        out, grad = preference_loss_and_grad(xt, tt, rt, ot, grad_dtype=TORCH[outdt], grad_scale=16.0, **kw)
        close(out.logprobs, want["logp"], lp_err)
        close(out.margins, want["margins"], 0.3 * h_err + 4 * U * np.abs(want["margins"]))
        slope = 2 * (np.abs(want["margins"]) / 0.3 + 2) if kind == "squared" else 0.3
        close(out.loss, want["loss"], np.max(slope) * h_err + 8 * U * (1 + abs(want["loss"])))
        p = np.exp(op.log_softmax(x))
        curve = 2.0 if kind == "squared" else 0.09
        amp = np.abs(want["a"]) + (want["a"] != 0) * (curve * h_err + 8 * U) / tol(vocab)
        check_grad(grad, want["grad"] * 16.0, amp, 0 * amp, p, 0 * amp, t, outdt, vocab, 1.0, 16.0)
    xg = xt.clone().requires_grad_(True)
    auto = preference_loss(xg, tt, rt, ot.int(), **kw)
    assert torch.equal(auto.loss, out.loss)
    (16.0 * auto.loss).backward()
    assert torch.equal(xg.grad, preference_loss_and_grad(xt, tt, rt, ot, grad_scale=16.0, **kw)[1])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,dtype", SHAPES)
@pytest.mark.parametrize("top,tau,vdt", [(1, 1.0, "f32"), (17, 2.0, "bf16"), (300, 0.7, "f16")])
def test_distillation_loss(rows, vocab, dtype, top, tau, vdt):
    rng = np.random.default_rng(rows * vocab + top)
    x = logits_of(rng, rows, vocab, dtype)
    v = logits_of(rng, rows, top, vdt)
    idx = rng.integers(0, vocab, (rows, top))  # tokens listed twice among them
    idx[rng.random((rows, top)) < 0.1] = -1
    v[rng.random((rows, top)) < 0.05] = -np.inf
    w = rng.random(rows).astype(np.float32)
    want = op.distill(x, v.astype(np.float64), idx, w.astype(float), tau)
    xt, vt, wt = to_torch(x), to_torch(v), torch.from_numpy(w).cuda()
    it = torch.from_numpy(idx).cuda()
    lp = op.log_softmax(x, tau)
    spread = tau**2 * (2 + np.abs(lp).max(1) + np.log(top + 1)) * (2 * tol(vocab) + 2 * tol(64 * top))
    p = np.exp(lp)
    for outdt in {"f32": ("f32", "bf16")}.get(dtype, (dtype,)):
        out, grad = distillation_loss_and_grad(xt, vt, it.int() if top % 2 else it, wt, temperature=tau, grad_scale=8.0, grad_dtype=TORCH[outdt])
        close(out.per_token, want["per_token"], spread)
        close(out.loss, want["loss"], (w * spread).sum() + U * abs(want["loss"]))
        bound = 8.0 * w[:, None] * tau * (p + want["q"]) * (2 * tol(vocab) + 2 * tol(64 * top)) + 1.01 * rounding(want["grad"] * 8.0, outdt) + 1e-30
        bad = np.abs(to_numpy(grad).astype(np.float64) - want["grad"] * 8.0) > bound
        assert not bad.any(), np.argwhere(bad)[:3]
    xg = xt.clone().requires_grad_(True)
    auto = distillation_loss(xg, vt, it, wt, temperature=tau)
    assert torch.equal(auto.loss, out.loss)
    (8.0 * auto.loss).backward()
    assert torch.equal(xg.grad, distillation_loss_and_grad(xt, vt, it, wt, temperature=tau, grad_scale=8.0)[1])


# --------------------------------------------------------------------------- GPU: layouts, masks, special values


def _all_ops(xt, rng, targets=None, weights=None, live=None):
    """Every operator once on xt; a dict of its results (gradients among them)."""
    rows, vocab = xt.shape
    g = torch.Generator(device="cuda").manual_seed(7)
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g) if targets is None else targets
    f = [torch.randn(rows, device="cuda", generator=g) for _ in range(2)]
    w = torch.rand(rows, device="cuda", generator=g) + 0.1 if weights is None else weights
    old = torch.full((rows,), -7.0, device="cuda")
    idx = torch.randint(0, vocab, (rows, 5), device="cuda", generator=g)
    v = torch.randn(rows, 5, device="cuda", generator=g)
    off = torch.tensor([0, rows // 3, rows], device="cuda")
    leaf = xt.detach().requires_grad_(True)
    lp, h = token_logprobs(leaf, t, entropy=True)
    (gl,) = torch.autograd.grad([lp, h], [leaf], f)
    po, gp = policy_loss_and_grad(xt, t, old, f[0], w, ref_logprobs=old, kl_coef=0.01, entropy_coef=0.1)
    pr, gr = preference_loss_and_grad(xt, t, old, off)
    di, gd = distillation_loss_and_grad(xt, v, idx, w)
    return {"logp": lp.detach(), "h": h.detach(), "gl": gl, "gp": gp, "gr": gr, "gd": gd, **{f"po{i}": o for i, o in enumerate(po)},
            **{f"pr{i}": o for i, o in enumerate(pr)}, **{f"di{i}": o for i, o in enumerate(di)}}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab,stride,shift", [(256, 264, 0), (1000, 1001, 0), (1000, 1003, 5), (32000, 32008, 8), (32001, 32004, 1), (129, 129, 3)])
def test_strides_and_alignment(dtype, vocab, stride, shift):
    """A view of a wider, shifted buffer (NaN between the rows) gives what the dense copy gives, up to the
    order of a row's sum (which goes by the address): within the summation's tolerance."""
    rng = np.random.default_rng(vocab)
    x = logits_of(rng, 6, vocab, dtype)
    a, b = _all_ops(on_gpu(x, stride, shift), rng), _all_ops(to_torch(x), rng)
    for k in a:
        u, v = a[k].double(), b[k].double()
        step = {"f32": 0.0, "bf16": 2.0**-8, "f16": 2.0**-11}[dtype] if k in ("gl", "gp", "gr", "gd") else 0.0
        scale = v.abs().max() if v.numel() else 0.0
        assert ((u - v).abs() <= step * v.abs() + 8 * tol(vocab) * (scale + 1) + 2.0**-24).all(), k
        assert torch.isfinite(u).all(), k


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [100, 32000])
def test_masked_rows_are_not_read(dtype, vocab):
    """NaN and infinities in masked rows stay out of every result; the rows' results and gradients are zeros."""
    rng = np.random.default_rng(3)
    x = logits_of(rng, 8, vocab, dtype)
    hide = np.array([0, 1, 0, 0, 1, 1, 0, 1], bool)
    t = rng.integers(0, vocab, 8)
    t[hide] = IGN
    w = np.where(hide, 0.0, 0.25).astype(np.float32)
    clean = _all_ops(to_torch(x), rng, torch.from_numpy(t).cuda(), torch.from_numpy(w).cuda())
    for filler in (np.nan, np.inf, -np.inf):
        y = x.copy()
        y[hide] = filler
        got = _all_ops(to_torch(y), rng, torch.from_numpy(t).cuda(), torch.from_numpy(w).cuda())
        for k in got:
            assert torch.equal(got[k], clean[k]), k
    for k in ("gl", "gp", "gr", "gd", "logp", "h", "po1", "po2", "po3", "di1"):
        assert not clean[k][torch.from_numpy(hide).cuda()].any(), k
    # everything masked
    none = _all_ops(torch.full((8, vocab), float("nan"), device="cuda", dtype=TORCH[dtype]), rng, torch.full((8,), IGN, device="cuda"), torch.zeros(8, device="cuda"))
    for k in ("po0", "di0", "gl", "gp", "gr", "gd", "logp"):
        assert not none[k].any(), k
    assert abs(none["pr0"].item() - np.log(2)) < 1e-6  # an empty pair: h = 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("low", ["inf", "lowest"])
def test_masked_vocabulary(dtype, low):
    """Columns of -inf or of the type's lowest value take no part: p = 0 there, and the gradient is 0."""
    rng = np.random.default_rng(4)
    x = logits_of(rng, 5, 1500, dtype)
    hide = np.zeros(1500, bool)
    hide[:700] = True  # whole leading vectors, so that a thread's first elements are all masked
    hide[rng.integers(700, 1490, 300)] = True
    x[:, hide] = -np.inf if low == "inf" else np.array(torch.finfo(TORCH[dtype]).min, np.float64).astype(NP[dtype])
    keep = np.flatnonzero(~hide)
    t = rng.choice(keep, 5)
    xt, tt = to_torch(x).requires_grad_(True), torch.from_numpy(t).cuda()
    lp, h = token_logprobs(xt, tt, entropy=True)
    want, wh = op.token_logprobs(x[:, ~hide], np.searchsorted(keep, t))
    close(lp, want, tol(1500) * (1 + np.abs(want)))
    close(h, wh, 2 * tol(1500) * (2 + wh + 8))
    (g,) = torch.autograd.grad([lp, h], [xt], [torch.ones(5, device="cuda"), torch.ones(5, device="cuda")])
    assert torch.isfinite(g).all() and not g[:, torch.from_numpy(hide).cuda()].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [1500, 32000])
@pytest.mark.parametrize("tau", [0.7, 0.8, 1.0, 1.4426950408889634, 3.0])
def test_masked_vocabulary_at_any_temperature(dtype, vocab, tau):
    """-inf columns, whatever sign the rounding error of log2(e) / tau has (0 for tau = log2 e)."""
    rng = np.random.default_rng(40)
    x = logits_of(rng, 4, vocab, dtype)
    hide = rng.random(vocab) < 0.4
    hide[:300] = True
    x[:, hide] = -np.inf
    keep = np.flatnonzero(~hide)
    t = rng.choice(keep, 4)
    want, wh = op.token_logprobs(x[:, ~hide], np.searchsorted(keep, t), tau)
    xt, tt = to_torch(x).requires_grad_(True), torch.from_numpy(t).cuda()
    lp = token_logprobs(xt, tt, temperature=tau)
    close(lp, want, tol(vocab) * (1 + np.abs(want)))
    both, h = token_logprobs(xt, tt, entropy=True, temperature=tau)
    close(both, want, tol(vocab) * (1 + np.abs(want)))
    close(h, wh, 2 * tol(vocab) * (2 + wh + 8))
    f = torch.ones(4, device="cuda")
    out, g = policy_loss_and_grad(xt.detach(), tt, lp.detach(), f, f, temperature=tau)
    assert torch.isfinite(out.loss) and torch.isfinite(g).all() and not g[:, torch.from_numpy(hide).cuda()].any()
    idx = torch.from_numpy(np.stack([rng.choice(keep, 20, replace=False) for _ in range(4)])).cuda()
    out, g = distillation_loss_and_grad(xt.detach(), torch.randn(4, 20, device="cuda"), idx, temperature=tau)
    assert torch.isfinite(out.per_token).all() and torch.isfinite(g).all() and not g[:, torch.from_numpy(hide).cuda()].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_of_one_value(dtype):
    """Rows whose every logit is the same -- zero, a large value, the type's lowest or highest -- are uniform."""
    big = torch.finfo(TORCH[dtype]).max
    for value in (0.0, 1000.0, -1000.0, 1e38, -1e38, big, -big):
        for vocab in (64, 1003):
            x = torch.full((2, vocab), value, device="cuda", dtype=TORCH[dtype])
            lp, h = token_logprobs(x, torch.tensor([0, vocab - 1], device="cuda"), entropy=True, temperature=1.0)
            assert (lp + np.log(vocab)).abs().max().item() <= 8 * tol(vocab), value
            assert (h - np.log(vocab)).abs().max().item() <= 8 * tol(vocab), value
            _, g = distillation_loss_and_grad(x, torch.zeros(2, 1, device="cuda"), torch.full((2, 1), 3, device="cuda"))
            want = np.full((2, vocab), 0.5 / vocab)
            want[:, 3] -= 0.5
            close(g, want, 2 * tol(vocab) + rounding(want, dtype))


@pytest.mark.gpu
def test_special_values_show():
    """NaN, +inf and a row of nothing but -inf give NaN in their own row, and only there."""
    rng = np.random.default_rng(5)
    x = logits_of(rng, 6, 777)
    x[1, 300] = np.nan
    x[2, 5] = np.inf
    x[3] = -np.inf
    x[4, :776] = -np.inf
    x[4, 776] = np.nan
    t = torch.tensor([0, 1, 2, 3, 4, 5], device="cuda")
    got = _all_ops(to_torch(x), rng, t)
    bad = torch.tensor([False, True, True, True, True, False], device="cuda")
    for k in ("logp", "h", "po1", "po2", "di1"):
        assert torch.equal(torch.isnan(got[k]), bad), k
    for k in ("gl", "gp", "gd"):
        assert torch.equal(torch.isnan(got[k]).any(1), bad), k
        assert torch.isfinite(got[k][~bad]).all(), k
    assert torch.isnan(got["po0"]) and torch.isnan(got["di0"])


@pytest.mark.gpu
def test_targets_and_indices_out_of_range():
    x = torch.randn(4, 128, device="cuda")
    t = torch.tensor([0, 128, -1, 127], device="cuda")
    lp = token_logprobs(x, t)
    assert torch.equal(torch.isnan(lp), torch.tensor([False, True, True, False], device="cuda"))
    _, g = policy_loss_and_grad(x, t, torch.zeros(4, device="cuda"), torch.ones(4, device="cuda"))
    assert torch.isnan(g[1:3]).all() and torch.isfinite(g[[0, 3]]).all()
    idx = torch.tensor([[1, 2], [128, 3], [-1, -1], [2**40, 1]], device="cuda")
    out, g = distillation_loss_and_grad(x, torch.zeros(4, 2, device="cuda"), idx)
    assert torch.equal(torch.isnan(out.per_token), torch.tensor([False, True, False, True], device="cuda"))
    assert out.per_token[2] == 0 and not g[2].any()
    assert torch.isnan(g[[1, 3]]).all() and torch.isfinite(g[[0, 2]]).all()


@pytest.mark.gpu
def test_extreme_ratios_and_margins():
    """A ratio that overflows f32 is clipped where the advantage is positive and shows as inf where it is
    not; margins far out give losses without overflow."""
    x = torch.zeros(2, 16, device="cuda")
    t = torch.zeros(2, dtype=torch.long, device="cuda")
    old = torch.full((2,), -200.0, device="cuda")
    out, g = policy_loss_and_grad(x, t, old, torch.tensor([1.0, -1.0], device="cuda"), torch.ones(2, device="cuda"))
    assert out.clipped.tolist() == [True, False] and torch.isinf(out.loss) and not g[0].any()
    off = torch.tensor([0, 1, 2], device="cuda")
    for ref, loss in (((-1000.0, 1000.0), 0.0), ((1000.0, -1000.0), 200.0)):
        out, g = preference_loss_and_grad(x, t, torch.tensor(ref, device="cuda"), off, beta=0.1)
        assert out.loss.item() == pytest.approx(loss, abs=1e-3) and torch.isfinite(g).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,dtype", [(1500, 32000, "bf16"), (2000, 8200, "bf16"), (900, 8203, "f32"), (700, 50257, "f32"), (600, 131072, "bf16"), (3000, 257, "f16"), (1111, 3001, "bf16")])
def test_many_rows(rows, vocab, dtype):
    """More rows than the GPU holds at once, some masked: every row as the plain form has it (f32 sums: the
    plain form's own error, at most V u, is allowed for besides the kernels'), and no wait of the kernels ran out."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = (3 * torch.randn(rows, vocab, device="cuda", generator=g)).to(TORCH[dtype])
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    t[torch.rand(rows, device="cuda", generator=g) < 0.2] = IGN
    w = torch.rand(rows, device="cuda", generator=g) * (torch.rand(rows, device="cuda", generator=g) > 0.2)
    old, adv = torch.full((rows,), -9.0, device="cuda"), torch.randn(rows, device="cuda", generator=g)
    idx = torch.randint(0, vocab, (rows, 40), device="cuda", generator=g)
    v = torch.randn(rows, 40, device="cuda", generator=g)
    off = torch.arange(0, rows + 1, rows // 6, device="cuda")[:7]
    e = 2 * (tol(vocab) + vocab * U) * (1 + np.log(vocab) + 20)

    def near(a, b, scale=1.0):
        step = rounding(b.float().cpu().numpy().astype(np.float64), dtype) if a.ndim == 2 else 0.0
        close(a.float(), b.float().cpu().numpy().astype(np.float64), e * scale + 1.01 * step)

    ref = x.detach().float().requires_grad_(True)
    lp, h = token_logprobs_reference(ref, t)
    leaf = x.detach().requires_grad_(True)
    glp, gh = token_logprobs(leaf, t, entropy=True)
    near(glp.detach(), lp.detach())
    near(gh.detach(), h.detach())
    (gr,) = torch.autograd.grad([lp, h], [ref], [adv, 0.1 * adv])
    (gg,) = torch.autograd.grad([glp, gh], [leaf], [adv, 0.1 * adv])
    near(gg, gr, 10.0)
    want = policy_loss_reference(ref, t, old, adv, w, ref_logprobs=old, kl_coef=0.001)
    (gr,) = torch.autograd.grad(want.loss, ref)
    got, gg = policy_loss_and_grad(x, t, old, adv, w, ref_logprobs=old, kl_coef=0.001)
    size = 1 + gr.abs().max().item()
    near(got.logprobs * (w != 0), want.logprobs)
    near(gg, gr, 10.0 * size)
    want = preference_loss_reference(ref, t, old, off)
    (gr,) = torch.autograd.grad(want.loss, ref)
    got, gg = preference_loss_and_grad(x, t, old, off)
    near(gg, gr, 10.0)
    want = distillation_loss_reference(ref, v, idx, w, temperature=2.0)
    (gr,) = torch.autograd.grad(want.loss, ref)
    got, gg = distillation_loss_and_grad(x, v, idx, w, temperature=2.0)
    near(got.per_token, want.per_token, 10.0)
    near(gg, gr, 10.0 * size)
    nat.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,top", [(700, 100, 1024), (700, 3, 1000), (650, 20000, 1024), (900, 1, 1024), (640, 9000, 700)])
def test_long_lists(rows, vocab, top):
    """The longest lists, over vocabularies much smaller than they are (every token listed many times) and larger."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = 3 * torch.randn(rows, vocab, device="cuda", generator=g)
    v, idx = torch.randn(rows, top, device="cuda", generator=g), torch.randint(-1, vocab, (rows, top), device="cuda", generator=g)
    idx[5] = -1
    ref = x.clone().requires_grad_(True)
    want = distillation_loss_reference(ref, v, idx)
    (gr,) = torch.autograd.grad(want.loss, ref)
    got, gg = distillation_loss_and_grad(x, v, idx)
    e = 4 * (tol(vocab) + tol(64 * top) + (vocab + top) * U) * (1 + np.log(vocab + 1) + np.log(top))
    close(got.per_token, want.per_token.cpu().numpy().astype(np.float64), e)
    close(gg, gr.cpu().numpy().astype(np.float64), e / rows * 2)
    assert not gg[5].any() and got.per_token[5] == 0
    nat.device_status()


@pytest.mark.gpu
def test_a_row_has_the_same_bits_in_every_batch():
    """With 16-byte aligned rows a row's results and gradient depend on nothing but the row."""
    for vocab, dtype in ((4096, torch.bfloat16), (32000, torch.bfloat16), (50304, torch.float32)):
        g = torch.Generator(device="cuda").manual_seed(vocab)
        x = (3 * torch.randn(1200, vocab, device="cuda", generator=g)).to(dtype)
        t = torch.randint(0, vocab, (1200,), device="cuda", generator=g)
        f = torch.randn(1200, device="cuda", generator=g)
        w = torch.full((1200,), 0.5, device="cuda")
        whole, grad = policy_loss_and_grad(x, t, f - 9, f, w, ref_logprobs=f - 9, kl_coef=0.01)
        for a, b in ((0, 1), (7, 8), (300, 317), (1000, 1200)):
            part, pg = policy_loss_and_grad(x[a:b].clone(), t[a:b], f[a:b] - 9, f[a:b], w[a:b], ref_logprobs=f[a:b] - 9, kl_coef=0.01)
            assert torch.equal(part.logprobs, whole.logprobs[a:b]) and torch.equal(pg, grad[a:b]) and torch.equal(part.kl, whole.kl[a:b])
        assert torch.equal(token_logprobs(x[300:317].clone(), t[300:317]), whole.logprobs[300:317])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,dtype", [(6000, 32000, "bf16"), (6000, 8192, "bf16"), (8000, 4096, "f16"), (3000, 32000, "f32"), (2500, 50264, "f16"), (1200, 131072, "bf16"), (500, 200000, "f32")])
def test_full_gpu_repeats_and_matches_small_batches(rows, vocab, dtype):
    """With every SM busy, calls back to back give the same bits each time, and those of a few rows alone: no
    entry comes from a piece of a row that was overwritten while it was in use."""
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    x = (3 * torch.randn(rows, vocab, device="cuda", generator=g)).to(TORCH[dtype])
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    f, dlp = torch.randn(2, rows, device="cuda", generator=g)
    w = torch.full((rows,), 1.0 / rows, device="cuda")
    v, idx = torch.randn(rows, 4096, device="cuda", generator=g).topk(64)
    off = torch.arange(0, rows + 1, rows // 10, device="cuda")

    def logprobs(a, b):
        leaf = x[a:b].detach().requires_grad_(True)
        lp, h = token_logprobs(leaf, t[a:b], entropy=True)
        (grad,) = torch.autograd.grad([lp, h], [leaf], [dlp[a:b], 0.1 * dlp[a:b]])
        return lp.detach(), h.detach(), grad

    def policy(a, b):
        out, grad = policy_loss_and_grad(x[a:b], t[a:b], f[a:b] - 9, dlp[a:b], w[a:b], ref_logprobs=f[a:b] - 9, kl_coef=0.01)
        return out.logprobs, out.kl, grad

    def distill(a, b):
        out, grad = distillation_loss_and_grad(x[a:b], v[a:b], idx[a:b], w[a:b])
        return out.per_token, grad

    for fn in (logprobs, policy, distill):
        first = fn(0, rows)
        for _ in range(6):
            assert all(torch.equal(p, q) for p, q in zip(fn(0, rows), first))
        for a in range(0, rows, rows // 5):
            part = fn(a, a + 60)
            assert all(torch.equal(p, q[a:a + 60]) for p, q in zip(part, first))
    out, first = preference_loss_and_grad(x, t, f - 9, off)
    for _ in range(6):
        again, grad = preference_loss_and_grad(x, t, f - 9, off)
        assert torch.equal(grad, first) and torch.equal(again.loss, out.loss)


@pytest.mark.gpu
def test_no_rows():
    x = torch.empty(0, 100, device="cuda")
    t, f = torch.empty(0, dtype=torch.long, device="cuda"), torch.empty(0, device="cuda")
    assert token_logprobs(x, t).shape == (0,)
    out, g = policy_loss_and_grad(x, t, f, f)
    assert out.loss.item() == 0.0 and g.shape == (0, 100)
    out, g = distillation_loss_and_grad(x, torch.empty(0, 3, device="cuda"), torch.empty(0, 3, dtype=torch.int32, device="cuda"))
    assert out.loss.item() == 0.0 and g.shape == (0, 100)
    out, g = preference_loss_and_grad(x, t, f, torch.zeros(3, dtype=torch.long, device="cuda"))
    assert out.loss.item() == pytest.approx(np.log(2), rel=1e-6) and g.shape == (0, 100)


@pytest.mark.gpu
def test_offsets_are_clamped():
    """Offsets outside the rows, and sequences that run backwards, reach nothing outside the tensors."""
    x, t, f = torch.randn(5, 64, device="cuda"), torch.zeros(5, dtype=torch.long, device="cuda"), torch.zeros(5, device="cuda")
    for off in ([-7, 2, 99], [0, 5, 3], [9, 9, 9]):
        out, g = preference_loss_and_grad(x, t, f, torch.tensor(off, device="cuda"))
        assert torch.isfinite(out.loss) and g.shape == (5, 64)


@pytest.mark.gpu
def test_repeatable_and_on_another_stream():
    g = torch.Generator(device="cuda").manual_seed(1)
    x = 3 * torch.randn(300, 5001, device="cuda", generator=g)
    a = _all_ops(x, None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = _all_ops(x, None)
    torch.cuda.current_stream().wait_stream(side)
    for k in a:
        assert torch.equal(a[k], b[k]), k


@pytest.mark.gpu
def test_captured_in_a_graph():
    g = torch.Generator(device="cuda").manual_seed(2)
    x = 3 * torch.randn(64, 4000, device="cuda", generator=g)
    t, f = torch.randint(0, 4000, (64,), device="cuda", generator=g), torch.randn(64, device="cuda", generator=g) - 8
    policy_loss_and_grad(x, t, f, f)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grad = policy_loss_and_grad(x, t, f, f)
    x.copy_(2 * torch.randn(64, 4000, device="cuda", generator=g))
    graph.replay()
    want, wg = policy_loss_and_grad(x, t, f, f)
    assert torch.equal(out.loss, want.loss) and torch.equal(grad, wg)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows that start beyond 2^31 elements: the last rows of a tensor of 2.2e9 elements."""
    rows, vocab = 68000, 32768
    x = torch.empty(rows, vocab, dtype=torch.bfloat16, device="cuda")
    x[: rows - 4].fill_(float("nan"))
    g = torch.Generator(device="cuda").manual_seed(3)
    x[rows - 4 :] = torch.randn(4, vocab, device="cuda", generator=g)
    t = torch.full((rows,), IGN, device="cuda")
    t[rows - 4 :] = torch.tensor([0, 5, 32767, 77], device="cuda")
    w = torch.ones(rows, device="cuda")
    old = torch.full((rows,), -10.0, device="cuda")
    out, grad = policy_loss_and_grad(x, t, old, w, w)
    small, sg = policy_loss_and_grad(x[rows - 4 :].clone(), t[rows - 4 :], old[:4], w[:4], w[:4])
    assert torch.equal(out.loss, small.loss) and torch.equal(grad[rows - 4 :], sg)
    assert not grad[1000].any() and not grad[rows - 5].any()
