"""mlp_megakernel_b200 -- B200-native (sm_100a) fused softplus MLP.

Drop-in for the fused-MLP path of Marcelo5444/mlp-megakernel: the functional
forward ``_fused_mlp_fwd`` / ``ModelNew`` (kernel.py:130-180) and the module API
``FusedMLPSoftplus`` / ``FusedMLPSoftplusWN`` (README.md:58-70).  Around it, what a training or serving step of a block of
such MLPs needs: the RMS norm with the residual's addition, rows sorted by
expert and back, a block of MLP experts, the AdamW step, and feed-forward layers
of any width (plain and gated) with activations kept in 8 bits.  All compute
runs in hand-written CUDA kernels (libmlpk.so, C ABI in include/mlpk.h).
"""
from .functional import ModelNew, _fused_mlp_fwd, fused_mlp_fwd, fused_mlp_fwd_host  # noqa: F401
from .modules import FusedMLPSoftplus, FusedMLPSoftplusWN  # noqa: F401
from .feedforward import (FusedGatedMLP, FusedLinear, fp8_checkpoint, fp8_restore, fused_gated_mlp,  # noqa: F401
                          fused_linear)
from .experts import ExpertPlan, FusedMLPExperts, expert_combine, expert_dispatch, expert_sort  # noqa: F401
from .norm import FusedRMSNorm, fused_rms_norm, fused_rms_norm_fp8  # noqa: F401
from .optim import FusedAdamW  # noqa: F401

__all__ = ["fused_mlp_fwd", "fused_mlp_fwd_host", "_fused_mlp_fwd", "ModelNew", "FusedMLPSoftplus",
           "FusedMLPSoftplusWN", "fused_rms_norm", "fused_rms_norm_fp8", "FusedRMSNorm", "expert_sort",
           "expert_dispatch", "expert_combine", "ExpertPlan", "FusedMLPExperts", "FusedAdamW", "fused_linear",
           "fused_gated_mlp", "fp8_checkpoint", "fp8_restore", "FusedLinear", "FusedGatedMLP"]
