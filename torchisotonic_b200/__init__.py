"""Batched isotonic regression for PyTorch on NVIDIA B200 (sm_100a): a drop-in for
``torchisotonic.isotonic`` over hand-written CUDA kernels behind a C ABI (include/tiso.h); and the
losses and the optimizer step of a language model whose answers it calibrates (losses.py,
optim.py)."""

from torchisotonic_b200._api import isotonic, isotonic_varlen
from torchisotonic_b200.calibration import calibrate, fit_calibration
from torchisotonic_b200.losses import PolicyLoss, policy_loss, preference_loss, token_logprobs
from torchisotonic_b200.optim import AdamW, adamw_step
from torchisotonic_b200.soft_rank import soft_rank

__all__ = ["isotonic", "isotonic_varlen", "fit_calibration", "calibrate", "soft_rank",
           "token_logprobs", "preference_loss", "policy_loss", "PolicyLoss", "adamw_step", "AdamW"]
__version__ = "0.1.0"
