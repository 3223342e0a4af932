"""The tied-head losses where the embedding's gradient cannot be taken for granted: f16 operands, scaled losses,
evaluation without a gradient, arguments that a gradient does not reach.

Tolerance of the f16 gradients: the logits' gradient and the products' results are rounded to f16, 2^-11 each, and the
products sum terms of mixed sign; held to 2^-9 of the largest entry.
"""

import pytest
import torch

from ferrite.kernels.distillation import distillation_loss_reference
from ferrite.kernels.policy_loss import policy_loss_reference
from ferrite.kernels.preference_loss import preference_loss_reference
from ferrite.kernels.tied_head import tied_head_distillation_loss, tied_head_policy_loss, tied_head_preference_loss


@pytest.mark.gpu
@pytest.mark.parametrize("logits_dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("which", ["policy", "preference", "distill"])
def test_f16_gradients_have_the_upstream_scale_before_they_are_rounded(which, logits_dtype):
    """Rows of so small a weight that f16 has none of their logits' gradient, under a loss scale that makes up for it."""
    g = torch.Generator(device="cuda").manual_seed(13)
    rows, d, vocab, small = 512, 128, 2048, 2.0**-26
    y = torch.randn(rows, d, device="cuda", generator=g).half().requires_grad_(True)
    e = (0.2 * torch.randn(vocab, d, device="cuda", generator=g)).half().requires_grad_(True)
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    y2, e2 = y.detach().float().requires_grad_(True), e.detach().float().requires_grad_(True)
    logits = y2 @ e2.t()
    if logits_dtype != torch.float32:
        logits = logits + (logits.to(logits_dtype).float() - logits).detach()  # the rounding, passed straight through
    old = torch.log_softmax(logits.detach(), 1).gather(1, t[:, None])[:, 0] - 0.05
    adv, w = torch.randn(rows, device="cuda", generator=g), torch.full((rows,), small, device="cuda")
    off = torch.tensor([0, 100, 250, 380, 512], device="cuda")
    v, i = torch.randn(rows, 8, device="cuda", generator=g), torch.randint(0, vocab, (rows, 8), device="cuda", generator=g)
    if which == "policy":
        got = tied_head_policy_loss(y, e, t, old, adv, w, ref_logprobs=old, kl_coef=0.1, logits_dtype=logits_dtype)
        want = policy_loss_reference(logits, t, old, adv, w, ref_logprobs=old, kl_coef=0.1)
    elif which == "preference":
        got = tied_head_preference_loss(y, e, t, old, off, beta=4 * small, logits_dtype=logits_dtype)
        want = preference_loss_reference(logits, t, old, off, beta=4 * small)
    else:
        got = tied_head_distillation_loss(y, e, v, i, w, logits_dtype=logits_dtype)
        want = distillation_loss_reference(logits, v, i, w)
    (got.loss / small).backward()
    (want.loss / small).backward()
    assert got.loss.item() == pytest.approx(want.loss.item(), rel=1e-3)
    for a, b in ((y.grad, y2.grad), (e.grad, e2.grad)):
        assert a.dtype == torch.float16
        assert (a.float() - b).abs().max().item() <= 2.0**-9 * b.abs().max().item()


def test_scales_of_the_logits_gradient_are_refused():
    """The node's gradient is autograd's: what scales or rounds the logits' own is not an argument of these."""
    y, e, t, f = torch.zeros(4, 8), torch.zeros(16, 8), torch.zeros(4, dtype=torch.long), torch.zeros(4)
    for kw in ({"grad_scale": 1024.0}, {"grad_dtype": torch.float32}):
        with pytest.raises(TypeError, match=next(iter(kw))):
            tied_head_policy_loss(y, e, t, f, f, **kw)
        with pytest.raises(TypeError, match=next(iter(kw))):
            tied_head_preference_loss(y, e, t, f, torch.tensor([0, 2, 4]), **kw)
        with pytest.raises(TypeError, match=next(iter(kw))):
            tied_head_distillation_loss(y, e, torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["policy", "preference", "distill"])
def test_no_gradient_is_computed_where_none_is_wanted(which):
    """Under no_grad, and with operands that need none, the logits are all that is allocated; the results are the same."""
    g = torch.Generator(device="cuda").manual_seed(17)
    rows, d, vocab = 1024, 64, 32000
    y = torch.randn(rows, d, device="cuda", generator=g).bfloat16()
    e = (0.2 * torch.randn(vocab, d, device="cuda", generator=g)).bfloat16()
    t, f = torch.randint(0, vocab, (rows,), device="cuda", generator=g), torch.full((rows,), -10.0, device="cuda")
    off = torch.tensor([0, 500, rows], device="cuda")
    v, i = torch.randn(rows, 8, device="cuda", generator=g), torch.randint(0, vocab, (rows, 8), device="cuda", generator=g)

    def call(y, e):
        return {"policy": lambda: tied_head_policy_loss(y, e, t, f, f, kl_coef=0.1, ref_logprobs=f), "preference": lambda: tied_head_preference_loss(y, e, t, f, off),
                "distill": lambda: tied_head_distillation_loss(y, e, v, i)}[which]()

    yg, eg = y.clone().requires_grad_(True), e.clone().requires_grad_(True)
    want = call(yg, eg)
    assert want.loss.requires_grad
    kept = [o.detach().clone() for o in want]
    del want
    with torch.no_grad():
        evaluated = lambda: call(yg, eg)  # noqa: E731
        for fn in (evaluated, lambda: call(y, e)):
            torch.cuda.synchronize()
            before = torch.cuda.memory_allocated()
            torch.cuda.reset_peak_memory_stats()
            got = fn()
            assert torch.cuda.max_memory_allocated() - before < rows * vocab * 5  # f32 logits; with a 16-bit gradient 6 bytes
            assert not got.loss.requires_grad and all(torch.equal(a, b) for a, b in zip(got, kept))
            del got
    got = call(y, e)
    assert not got.loss.requires_grad and torch.equal(got.loss, kept[0])
