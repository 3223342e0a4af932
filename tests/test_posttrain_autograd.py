"""What autograd may ask of the post-training losses, and what they refuse: they have a first derivative, in the logits."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from ferrite.kernels.distillation import distillation_loss, distillation_loss_and_grad
from ferrite.kernels.logprobs import token_logprobs
from ferrite.kernels.policy_loss import policy_loss, policy_loss_and_grad
from ferrite.kernels.preference_loss import preference_loss, preference_loss_and_grad
from ferrite.kernels.tied_head import tied_head_distillation_loss, tied_head_policy_loss, tied_head_preference_loss


def _inputs(device, grad=True):
    x = torch.randn(4, 64, device=device).requires_grad_(grad)
    t = torch.zeros(4, dtype=torch.long, device=device)
    f = torch.full((4,), -4.0, device=device)
    off, v = torch.tensor([0, 2, 4], device=device), torch.zeros(4, 2, device=device)
    return x, t, f, off, v, torch.zeros(4, 2, dtype=torch.int32, device=device)


def _calls(x, t, f, off, v, i, y=None, e=None):
    """(argument, call with that argument passed through ``on``)"""
    calls = [
        ("old_logprobs", lambda on: policy_loss(x, t, on(f), f)),
        ("advantages", lambda on: policy_loss(x, t, f, on(f))),
        ("weights", lambda on: policy_loss(x, t, f, f, on(f))),
        ("ref_logprobs", lambda on: policy_loss(x, t, f, f, ref_logprobs=on(f), kl_coef=0.1)),
        ("ref_logprobs", lambda on: preference_loss(x, t, on(f), off)),
        ("teacher_values", lambda on: distillation_loss(x, on(v), i)),
        ("weights", lambda on: distillation_loss(x, v, i, on(f))),
    ]
    if y is not None:
        calls += [
            ("argument", lambda on: tied_head_policy_loss(y, e, t, f, on(f))),
            ("argument", lambda on: tied_head_policy_loss(y, e, t, f, f, ref_logprobs=on(f))),
            ("argument", lambda on: tied_head_preference_loss(y, e, t, on(f), off)),
            ("argument", lambda on: tied_head_distillation_loss(y, e, on(v), i)),
        ]
    return calls


def _leaf(a):
    return a.clone().requires_grad_(True)


def test_other_arguments_that_ask_for_a_gradient_are_refused():
    y, e = torch.zeros(4, 8, requires_grad=True), torch.zeros(64, 8)
    for name, call in _calls(*_inputs("cpu"), y, e):
        with pytest.raises(ValueError, match=f"{name} requires a gradient"):
            call(_leaf)


@pytest.mark.gpu
def test_other_arguments_without_a_record_are_taken():
    """Under no_grad, or where the logits are not recorded, nothing is lost; detached arguments are always taken."""
    y, e = torch.randn(4, 64, device="cuda", requires_grad=True), torch.randn(64, 64, device="cuda")
    for _, call in _calls(*_inputs("cuda"), y, e):
        with torch.no_grad():
            assert not call(_leaf).loss.requires_grad
        assert call(lambda a: a).loss.requires_grad
    for _, call in _calls(*_inputs("cuda", grad=False)):
        assert not call(_leaf).loss.requires_grad


@pytest.mark.gpu
def test_forward_mode_tangents_are_refused():
    """A tangent raises whether or not the logits also ask for a gradient; a dual level without one changes nothing."""
    x, t, f, off, v, i = _inputs("cuda", grad=False)
    y, e = torch.randn(4, 64, device="cuda"), torch.randn(64, 64, device="cuda")
    calls = [
        (x, lambda z: token_logprobs(z, t)),
        (x, lambda z: policy_loss(z, t, f, f)),
        (x, lambda z: preference_loss(z, t, f, off)),
        (x, lambda z: distillation_loss(z, v, i)),
        (y, lambda z: tied_head_policy_loss(z, e, t, f, f)),
        (e, lambda z: tied_head_policy_loss(y, z, t, f, f)),
    ]
    with fwd.dual_level():
        for n, (at, call) in enumerate(calls):
            call(at)
            for grad in (False, True):
                with pytest.raises(RuntimeError, match="jvp|forward AD"):
                    call(fwd.make_dual(at.clone().requires_grad_(grad), torch.ones_like(at)))
                    pytest.fail(f"call {n} dropped the tangent")


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    """Of a term with no second derivative in it the gradient's own would be all that is left, without a word."""
    x, t, f, off, v, i = _inputs("cuda")
    y, e = torch.randn(4, 64, device="cuda", requires_grad=True), torch.randn(64, 64, device="cuda")
    losses = [
        (x, lambda: token_logprobs(x, t).sum()),
        (x, lambda: policy_loss(x, t, f, f).loss),
        (x, lambda: preference_loss(x, t, f, off).loss),
        (x, lambda: distillation_loss(x, v, i).loss),
        (y, lambda: tied_head_policy_loss(y, e, t, f, f).loss),
    ]
    for n, (at, loss) in enumerate(losses):
        (g,) = torch.autograd.grad(loss(), at, create_graph=True)
        with pytest.raises(RuntimeError, match="no second derivative"):
            (g.pow(2).sum() + at.sum()).backward()
            pytest.fail(f"loss {n}: the second derivative was dropped")


@pytest.mark.gpu
def test_upstream_scalars():
    """``upstream`` is a number on the logits' device, and multiplies the gradient like ``grad_scale``."""
    x, t, f, off, v, i = _inputs("cuda", grad=False)
    calls = [
        lambda **kw: policy_loss_and_grad(x, t, f, f, **kw),
        lambda **kw: preference_loss_and_grad(x, t, f, off, **kw),
        lambda **kw: distillation_loss_and_grad(x, v, i, **kw),
    ]
    for call in calls:
        for bad in (torch.tensor(2.0), torch.ones(2, device="cuda"), torch.ones((), device="cuda", dtype=torch.long)):
            with pytest.raises((ValueError, RuntimeError)):
                call(upstream=bad)
        out, grad = call(upstream=torch.tensor([4.0], device="cuda", dtype=torch.float64))
        want, scaled = call(grad_scale=4.0)
        assert torch.equal(grad, scaled) and torch.equal(out.loss, want.loss)
