from ferrite.kernels.distillation import distillation_loss, distillation_loss_and_grad, distillation_loss_reference
from ferrite.kernels.flash_attention import flash_attention, flash_attention_reference
from ferrite.kernels.logprobs import token_logprobs, token_logprobs_reference
from ferrite.kernels.matmul import matmul, matmul_reference
from ferrite.kernels.policy_loss import policy_loss, policy_loss_and_grad, policy_loss_reference
from ferrite.kernels.preference_loss import preference_loss, preference_loss_and_grad, preference_loss_reference
from ferrite.kernels.rmsnorm import rmsnorm, rmsnorm_reference
from ferrite.kernels.tied_head import tied_head_distillation_loss, tied_head_policy_loss, tied_head_preference_loss

__all__ = [
    "distillation_loss",
    "distillation_loss_and_grad",
    "distillation_loss_reference",
    "flash_attention",
    "flash_attention_reference",
    "matmul",
    "matmul_reference",
    "policy_loss",
    "policy_loss_and_grad",
    "policy_loss_reference",
    "preference_loss",
    "preference_loss_and_grad",
    "preference_loss_reference",
    "rmsnorm",
    "rmsnorm_reference",
    "tied_head_distillation_loss",
    "tied_head_policy_loss",
    "tied_head_preference_loss",
    "token_logprobs",
    "token_logprobs_reference",
]
