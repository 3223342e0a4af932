"""Post-training of the GPT: preference pairs, a clipped policy loss, distillation from a larger model.

The reference stops at next-token pre-training (src/ferrite/model/train.py:102-177); these are the steps
that follow it, on the same model, optimiser and parameter layout.  Each objective is one function of
``(params, batch, cfg)`` whose loss runs on the tied head with its gradient fused
(:mod:`ferrite.kernels.tied_head`); what a step needs besides -- log-probabilities under the policy that sampled
or under a frozen reference, a teacher's top logits -- comes from :func:`score` and :func:`top_logits`.

``python -m ferrite.model.posttrain --objective policy`` (``preference``, ``distill``) runs an objective on a
small byte-level model and prints its course.
"""

from __future__ import annotations

import dataclasses
import json
from typing import Any

import numpy as np
import torch

from ferrite.kernels.logprobs import IGNORE_INDEX, token_logprobs
from ferrite.kernels.matmul import gemm
from ferrite.kernels.tied_head import tied_head_distillation_loss, tied_head_policy_loss, tied_head_preference_loss
from ferrite.model import data as data_lib
from ferrite.model.gpt import GPTConfig, hidden, init_params, param_leaves
from ferrite.model.train import TrainConfig, make_optimizer


def _head(params, tokens, cfg: GPTConfig):
    """(y [rows, d_model], embedding [vocab, d_model]) in the compute type: what the tied head multiplies."""
    return hidden(params, tokens, cfg), params["tok_emb"].to(cfg.dtype)


@torch.no_grad()
def logits_of(params, tokens, cfg: GPTConfig) -> torch.Tensor:
    """f32 logits ``[rows, vocab]`` of ``tokens [B, S]``."""
    y, e = _head(params, tokens, cfg)
    return gemm(y, e, trans_b=True, out_dtype=torch.float32)


def score(params, tokens, targets, cfg: GPTConfig, temperature: float = 1.0) -> torch.Tensor:
    """Log-probabilities ``[rows]`` of ``targets`` after ``tokens``; zeros where a target is ``IGNORE_INDEX``."""
    return token_logprobs(logits_of(params, tokens, cfg), targets.reshape(-1), temperature=temperature)


def top_logits(params, tokens, cfg: GPTConfig, top: int) -> tuple[torch.Tensor, torch.Tensor]:
    """A teacher's ``top`` best tokens of each row and their logits: ``(values, indices)``, ``[rows, top]``."""
    best = logits_of(params, tokens, cfg).topk(top)
    return best.values, best.indices.int()


def policy_objective(params, batch, cfg: GPTConfig, **kw):
    """batch: tokens [B, S], targets [B, S], old_logprobs, advantages [rows], optionally weights, ref_logprobs [rows]."""
    y, e = _head(params, batch["tokens"], cfg)
    return tied_head_policy_loss(y, e, batch["targets"].reshape(-1), batch["old_logprobs"], batch["advantages"], batch.get("weights"),
                                 ref_logprobs=batch.get("ref_logprobs"), **kw)


def preference_objective(params, batch, cfg: GPTConfig, **kw):
    """batch: tokens [2 pairs, S] (chosen and rejected in turn), targets likewise, ref_logprobs [rows]."""
    tokens = batch["tokens"]
    y, e = _head(params, tokens, cfg)
    offsets = torch.arange(0, tokens.numel() + 1, tokens.shape[1], device=tokens.device)
    return tied_head_preference_loss(y, e, batch["targets"].reshape(-1), batch["ref_logprobs"], offsets, **kw)


def distillation_objective(params, batch, cfg: GPTConfig, **kw):
    """batch: tokens [B, S], teacher_values and teacher_indices [rows, top], optionally weights [rows]."""
    y, e = _head(params, batch["tokens"], cfg)
    return tied_head_distillation_loss(y, e, batch["teacher_values"], batch["teacher_indices"], batch.get("weights"), **kw)


OBJECTIVES = {"policy": policy_objective, "preference": preference_objective, "distill": distillation_objective}


def build_step(objective, params, leaves, cfg: GPTConfig, train_cfg: TrainConfig, **kw):
    """``step(batch) -> the objective's result``: forward, backward and AdamW on ``leaves``."""
    opt, flat = make_optimizer(leaves, train_cfg)

    def step(batch):
        flat.zero()
        out = objective(params, batch, cfg, **kw)
        out.loss.backward()
        opt.update() if hasattr(opt, "grads") else opt.update(flat.views)
        return out

    return step


# ---------------------------------------------------------------- the command


@dataclasses.dataclass(frozen=True)
class PosttrainConfig:
    objective: str = "policy"
    steps: int = 40
    batch: int = 16
    lr: float = 1e-3
    seed: int = 0
    top: int = 16
    temperature: float = 1.0


def _windows(rng, corpus, n, seq, device):
    x, y = data_lib.get_batch(rng, corpus, n, seq)
    return torch.from_numpy(x).to(device), torch.from_numpy(y).to(device)


def _sampled(params, x, cfg, gen, temperature):
    """One token sampled after every position of ``x``."""
    p = torch.softmax(logits_of(params, x, cfg) / temperature, dim=-1)
    return torch.multinomial(p, 1, generator=gen).reshape(x.shape)


def posttrain(cfg: GPTConfig, pc: PosttrainConfig, *, verbose: bool = True) -> dict[str, Any]:
    """Runs an objective on synthetic text; returns its loss curve and what the objective is about: the mean
    reward of sampled tokens (policy), the share of pairs in the right order (preference), the mean KL to the
    teacher (distill)."""
    device = torch.device("cuda", torch.cuda.current_device())
    rng, gen = np.random.default_rng(pc.seed), torch.Generator(device=device).manual_seed(pc.seed)
    corpus = data_lib.synthetic(100_000, seed=pc.seed)
    params = init_params(pc.seed, cfg, device=device)
    leaves = param_leaves(params)
    for p in leaves:
        p.requires_grad_(True)
    frozen = init_params(pc.seed, cfg, device=device)  # the reference policy: the model as it was at the start
    teacher_cfg = cfg.replace(d_model=2 * cfg.d_model, n_head=2 * cfg.n_head, d_ff=2 * cfg.d_ff)
    teacher = init_params(pc.seed + 1, teacher_cfg, device=device) if pc.objective == "distill" else None
    if teacher is not None:  # an embedding wide enough that the teacher's logits are not all alike
        teacher["tok_emb"] *= 10.0
    kw = {"policy": {"kl_coef": 0.02, "entropy_coef": 0.001, "temperature": pc.temperature}, "preference": {"beta": 0.1, "average": False},
          "distill": {"temperature": pc.temperature}}[pc.objective]
    train_cfg = TrainConfig(steps=pc.steps, lr=pc.lr, warmup=5, weight_decay=0.0)
    step = build_step(OBJECTIVES[pc.objective], params, leaves, cfg, train_cfg, **kw)

    def batch():
        x, y = _windows(rng, corpus, pc.batch, cfg.seq_len, device)
        if pc.objective == "distill":
            values, indices = top_logits(teacher, x, teacher_cfg, pc.top)
            return {"tokens": x, "teacher_values": values, "teacher_indices": indices}
        if pc.objective == "preference":  # chosen: the text; rejected: the same windows with random second halves
            half = cfg.seq_len // 2
            bad_x, bad_y = x.clone(), y.clone()
            bad_y[:, half:] = torch.randint(0, cfg.vocab_size, bad_y[:, half:].shape, device=device, generator=gen)
            bad_x[:, half + 1 :] = bad_y[:, half:-1]
            tokens, targets = (torch.stack([a, b], 1).reshape(-1, cfg.seq_len) for a, b in ((x, bad_x), (y, bad_y)))
            targets[:, :half] = IGNORE_INDEX  # the prompt
            return {"tokens": tokens, "targets": targets, "ref_logprobs": score(frozen, tokens, targets, cfg)}
        actions = _sampled(params, x, cfg, gen, pc.temperature)  # reward: a byte below 64, as all of the text is
        reward = (actions < 64).float().reshape(-1)
        return {"tokens": x, "targets": actions, "reward": reward, "advantages": (reward - reward.mean()) / (reward.std() + 1e-4),
                "old_logprobs": score(params, x, actions, cfg, pc.temperature), "ref_logprobs": score(frozen, x, actions, cfg, pc.temperature)}

    losses, course = [], []
    for i in range(pc.steps):
        b = batch()
        for _ in range(2 if pc.objective == "policy" else 1):  # a policy's batch is used twice: the second time off-policy
            out = step(b)
        losses.append(float(out.loss.detach()))
        course.append(float({"policy": lambda: b["reward"].mean(), "preference": lambda: (out.margins > 0).float().mean(),
                             "distill": lambda: out.per_token.mean()}[pc.objective]()))
        if verbose and (i % 10 == 0 or i == pc.steps - 1):
            print(f"step {i:4d} loss {losses[-1]:.4f} {pc.objective} {course[-1]:.4f}")
    return {"objective": pc.objective, "loss": losses, "course": course, "loss_first": losses[0], "loss_last": losses[-1],
            "course_first": course[0], "course_last": float(np.mean(course[-5:]))}


def main(argv=None):
    import argparse

    ap = argparse.ArgumentParser(description="Post-train a small byte-level GPT on the B200 kernels.")
    ap.add_argument("--objective", choices=sorted(OBJECTIVES), default="policy")
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--seq", type=int, default=128)
    ap.add_argument("--lr", type=float, default=1e-3)
    a = ap.parse_args(argv)
    cfg = GPTConfig(seq_len=a.seq, d_model=256, n_head=4, n_layer=2, d_ff=1024, linear="pallas")
    res = posttrain(cfg, PosttrainConfig(objective=a.objective, steps=a.steps, batch=a.batch, lr=a.lr))
    print(json.dumps({k: v for k, v in res.items() if not isinstance(v, list)}, indent=2))


if __name__ == "__main__":
    main()
