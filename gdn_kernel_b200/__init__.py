"""B200-native (sm_100a) Gated DeltaNet hot path: T=1 decode and chunked
(C=64) variable-length prefill behind the reference's ``kernel`` API, plus the
serving forms of the decode step (state pool with indices, multi-token
decode), and the operators that stand around it: short causal convolution,
selective state space scan, gated norm, residual add and norm."""

from .kernel import (decode, gdn_decode, gdn_decode_pool, gdn_mtp, gdn_prefill,  # noqa: F401
                     load_tvm_kernel, mtp, prefill)
from .mixer import (add_norm, gated_norm, gdn_add_norm, gdn_gated_norm, gdn_short_conv,  # noqa: F401
                    gdn_short_conv_step, gdn_ssm_prefill, gdn_ssm_step, short_conv,
                    short_conv_step, ssm_prefill, ssm_prefill_workspace_bytes, ssm_step)
from ._lib import device_status  # noqa: F401

__all__ = ["decode", "prefill", "gdn_decode", "gdn_prefill", "gdn_decode_pool", "gdn_mtp", "mtp",
           "gdn_short_conv", "gdn_short_conv_step", "short_conv", "short_conv_step",
           "gdn_ssm_prefill", "gdn_ssm_step", "ssm_prefill", "ssm_step",
           "ssm_prefill_workspace_bytes", "gdn_gated_norm", "gated_norm", "gdn_add_norm",
           "add_norm", "load_tvm_kernel", "device_status"]
