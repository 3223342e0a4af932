"""Oracle of the post-training losses (numpy, 64 bits) -- test infrastructure only.

From the definitions: token log-probabilities and entropies, the clipped policy loss with its
KL term and entropy bonus, the preference loss of paired sequences, and distillation from a
teacher's top logits, each with the derivative of its formula in the logits.  The reference
has no counterpart (its loss is the mean cross-entropy of src/ferrite/model/gpt.py:147-152).
"""

from __future__ import annotations

import numpy as np

F64 = np.float64


def log_softmax(x: np.ndarray, tau: float = 1.0) -> np.ndarray:
    z = x.astype(F64) / tau
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        z = z - np.max(z, axis=-1, keepdims=True)
        return z - np.log(np.sum(np.exp(z), axis=-1, keepdims=True))


def _plogp(lp: np.ndarray) -> np.ndarray:
    p = np.exp(lp)
    return np.where(p > 0, p * np.where(p > 0, lp, 0.0), 0.0)


def token_logprobs(x, t, tau=1.0, ignore=-100):
    """(logp, H) per row; zeros where the target is ``ignore``."""
    live = t != ignore
    lp = log_softmax(x, tau)
    logp = np.take_along_axis(lp, np.where(live, t, 0)[:, None], 1)[:, 0]
    return np.where(live, logp, 0.0), np.where(live, -_plogp(lp).sum(1), 0.0)


def logits_grad(x, t, a, b, tau=1.0, ignore=-100):
    """d/dx of sum_r a_r logp_r + b_r H_r."""
    live = t != ignore
    lp = log_softmax(x, tau)
    p = np.exp(lp)
    h = -_plogp(lp).sum(1, keepdims=True)
    one = np.zeros_like(p)
    one[np.arange(len(t)), np.where(live, t, 0)] = 1.0
    with np.errstate(invalid="ignore"):
        g = a[:, None] * (one - p) - b[:, None] * (_plogp(lp) + p * h)
    return np.where(live[:, None], g / tau, 0.0)


def policy(x, t, old, adv, w, ref=None, lo=0.2, hi=0.2, beta=0.0, c=0.0, tau=1.0, ignore=-100):
    """dict of loss, logp, entropy, kl, clipped, grad and the coefficients a = dL/dlogp, b = dL/dH."""
    live = (t != ignore) & (w != 0)
    t = np.where(live, t, ignore)
    logp, h = token_logprobs(x, t, tau, ignore)
    with np.errstate(over="ignore", invalid="ignore"):
        ratio = np.exp(logp - old)
        free, held = ratio * adv, np.clip(ratio, 1 - lo, 1 + hi) * adv
        d = np.zeros_like(logp) if ref is None else ref - logp
        kl = np.expm1(d) - d
        per = -np.minimum(free, held) + beta * kl - c * h
        a = w * (np.where(held < free, 0.0, -free) + beta * (0.0 if ref is None else -np.expm1(d)))
    keep = lambda v: np.where(live, v, 0.0)  # noqa: E731
    a, b = keep(a), keep(-w * c)
    return {"loss": keep(w * per).sum(), "logp": logp, "entropy": h, "kl": keep(kl), "clipped": live & (held < free), "a": a, "b": b,
            "grad": logits_grad(x, t, a, b, tau, ignore)}


def pair_value(h, beta, kind, e=0.0):
    """(loss, dloss/dh) of pairs with difference h."""
    if kind == "sigmoid":
        return (1 - e) * np.logaddexp(0, -beta * h) + e * np.logaddexp(0, beta * h), beta * (1 / (1 + np.exp(-beta * h)) - (1 - e))
    if kind == "squared":
        return (h - 0.5 / beta) ** 2, 2 * (h - 0.5 / beta)
    return np.maximum(0, 1 - beta * h), np.where(1 - beta * h > 0, -beta, 0.0)


def preference(x, t, ref, offsets, beta=0.1, kind="sigmoid", e=0.0, average=False, tau=1.0, ignore=-100):
    """dict of loss, margins, logp, the rows' dloss/dlogp a, and grad."""
    live = t != ignore
    logp, _ = token_logprobs(x, t, tau, ignore)
    pairs = len(offsets) // 2
    d, n = np.zeros(2 * pairs), np.ones(2 * pairs)
    for j in range(2 * pairs):
        s = slice(offsets[j], offsets[j + 1])
        if average:
            n[j] = max(1, live[s].sum())
        d[j] = np.where(live[s], logp[s] - ref[s], 0.0).sum() / n[j]
    h = d[0::2] - d[1::2]
    loss, dh = pair_value(h, beta, kind, e)
    a = np.zeros(len(t))
    for j in range(2 * pairs):
        a[offsets[j] : offsets[j + 1]] = (1 if j % 2 == 0 else -1) * dh[j // 2] / pairs / n[j]
    a = np.where(live, a, 0.0)
    return {"loss": loss.mean(), "margins": beta * h, "logp": logp, "a": a, "grad": logits_grad(x, t, a, np.zeros_like(a), tau, ignore)}


def distill(x, values, indices, w, tau=1.0):
    """dict of loss, per_token, q (dense weights over the vocabulary), grad."""
    rows, vocab = x.shape
    per, grad, dense = np.zeros(rows), np.zeros((rows, vocab)), np.zeros((rows, vocab))
    lp = log_softmax(x, tau)
    for r in range(rows):
        on = (indices[r] >= 0) & (values[r] > -np.inf)
        if w[r] == 0 or not on.any():
            continue
        lq = log_softmax(values[r][on][None].astype(F64), tau)[0]
        q, at = np.exp(lq), indices[r][on]
        use = q > 0
        per[r] = tau**2 * np.sum(q[use] * (lq[use] - lp[r, at[use]]))
        np.add.at(dense[r], at, q)
        grad[r] = w[r] * tau * (np.exp(lp[r]) - dense[r])
    live = per != 0
    return {"loss": np.sum(np.where(live, w, 0.0) * per), "per_token": per, "q": dense, "grad": grad}
