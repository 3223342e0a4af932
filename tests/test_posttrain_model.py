"""The post-training losses on the tied head and in the model's training step.

CPU: refusals of the tied-head entry points.
GPU (``-m gpu``): loss and gradients of the fused node against the same chain in torch f32 (the plain forms
of the losses on ``y @ e^T``), and a short run of each objective, which has to move what it is about.

Tolerances: y and e are bf16, the logits f32; the logits' gradient and the products' results are rounded to
bf16, 2^-8 each, and the products sum terms of mixed sign, so gradients are held to 2^-6 of their largest entry.
"""

import pytest
import torch

from ferrite.kernels.distillation import distillation_loss_reference
from ferrite.kernels.policy_loss import policy_loss_reference
from ferrite.kernels.preference_loss import preference_loss_reference
from ferrite.kernels.tied_head import tied_head_distillation_loss, tied_head_policy_loss, tied_head_preference_loss


def test_refusals():
    y, e, t, f = torch.zeros(4, 8), torch.zeros(16, 8), torch.zeros(4, dtype=torch.long), torch.zeros(4)
    with pytest.raises(ValueError):
        tied_head_policy_loss(y, torch.zeros(16, 9), t, f, f)
    with pytest.raises(ValueError):
        tied_head_policy_loss(y, e.bfloat16(), t, f, f)
    with pytest.raises(TypeError):
        tied_head_preference_loss(y.bfloat16(), e.bfloat16(), t, f, torch.tensor([0, 2, 4]), logits_dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        tied_head_distillation_loss(y, e, torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [4096, 1003])
@pytest.mark.parametrize("logits_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("which", ["policy", "preference", "distill"])
def test_tied_head_matches_the_unfused_chain(which, logits_dtype, vocab):
    g = torch.Generator(device="cuda").manual_seed(3)
    rows, d = 512, 256
    y = torch.randn(rows, d, device="cuda", generator=g).bfloat16().requires_grad_(True)
    e = (0.1 * torch.randn(vocab, d, device="cuda", generator=g)).bfloat16().requires_grad_(True)
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    old, adv = torch.full((rows,), -8.5, device="cuda"), torch.randn(rows, device="cuda", generator=g)
    off = torch.tensor([0, 100, 250, 380, 512], device="cuda")
    v, i = torch.randn(rows, 8, device="cuda", generator=g), torch.randint(0, vocab, (rows, 8), device="cuda", generator=g)
    y2, e2 = y.detach().clone().requires_grad_(True), e.detach().clone().requires_grad_(True)
    logits = y2.float() @ e2.float().t()
    if logits_dtype != torch.float32:
        logits = logits + (logits.to(logits_dtype).float() - logits).detach()  # the rounding, passed straight through
    if which == "policy":
        got = tied_head_policy_loss(y, e, t, old, adv, ref_logprobs=old, kl_coef=0.01, entropy_coef=0.01, logits_dtype=logits_dtype)
        want = policy_loss_reference(logits, t, old, adv, ref_logprobs=old, kl_coef=0.01, entropy_coef=0.01)
    elif which == "preference":
        got = tied_head_preference_loss(y, e, t, old, off, average=True, logits_dtype=logits_dtype)
        want = preference_loss_reference(logits, t, old, off, average=True)
    else:
        got = tied_head_distillation_loss(y, e, v, i, temperature=2.0, logits_dtype=logits_dtype)
        want = distillation_loss_reference(logits, v, i, temperature=2.0)
    (3.0 * got.loss).backward()
    (3.0 * want.loss).backward()
    # bf16 logits may round the other way than the chain's where its sum lies next to a tie
    torch.testing.assert_close(got.loss, want.loss, rtol=1e-4 if logits_dtype == torch.float32 else 5e-3, atol=1e-4 if logits_dtype == torch.float32 else 5e-3)
    for a, b in ((y.grad, y2.grad), (e.grad, e2.grad)):
        assert (a.float() - b.float()).abs().max().item() <= 2.0**-6 * b.float().abs().max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("objective", ["policy", "preference", "distill"])
def test_objectives_move_what_they_are_about(objective):
    from ferrite.model.gpt import GPTConfig
    from ferrite.model.posttrain import PosttrainConfig, posttrain

    cfg = GPTConfig(seq_len=128, d_model=128, n_head=2, n_layer=2, d_ff=512, linear="pallas")
    res = posttrain(cfg, PosttrainConfig(objective=objective, steps=30, batch=8, lr=2e-3), verbose=False)
    if objective == "policy":
        assert res["course_last"] > res["course_first"] + 0.2  # a quarter of random bytes are below 64
    elif objective == "preference":
        assert res["course_last"] > 0.9 and res["loss_last"] < 0.6 < res["loss_first"] < 0.75
    else:
        assert res["course_last"] < 0.8 * res["course_first"]
