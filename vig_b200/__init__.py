"""B200-native bi-directional gated linear attention and ViG block kernels behind the reference's operator API."""
from .ops import (bi_gla, bi_gla_backward, bid_fused_recurrent_gla, fused_chunk_gla, chunk_gla, fused_recurrent_gla,  # noqa: F401
                  dwconv3x3, gate_inject, add_rmsnorm, layernorm_act, swiglu, swiglu_linear, linear_swiglu,
                  gated_recurrence, gated_recurrence_step, add_rmsnorm_8bit, add_rmsnorm_train, add_rmsnorm_backward, adamw_step,
                  selective_scan, selective_scan_step, causal_conv, causal_conv_step, add_layernorm_train, add_layernorm_backward, linear_int8,
                  check_status, status_word)
from .modules import RMSNorm, GatedLinearAttention, GLAMLP, GLABlock  # noqa: F401
from .vig import ViG, build_vig  # noqa: F401
from .hier import HierViG, GLA2D, VSSBlock  # noqa: F401
from .recurrent import GatedRecurrence  # noqa: F401
from .state_space import SelectiveStateSpace  # noqa: F401
from .optim import AdamW  # noqa: F401
from . import native  # noqa: F401  (imported here so that it knows the operators as they are before anyone wraps them)
