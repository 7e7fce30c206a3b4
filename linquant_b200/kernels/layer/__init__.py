"""Operators around the recurrence of a layer, for prompts (``*_fwd``) and single tokens (``*_step``): short causal
convolution, selective scan, linear attention, INT8 product of the projections, norms with residual, gate and quantisation."""

from .group_norm import group_norm_fwd  # noqa: F401
from .int8_linear import int8_linear_fwd, quantize_rows_fwd  # noqa: F401
from .linear_attention import linear_attention_fwd, linear_attention_step  # noqa: F401
from .lora_linear import lora_linear_fwd, stack_adapters  # noqa: F401
from .rms_norm import gated_rms_norm_fwd, rms_norm_fwd  # noqa: F401
from .selective_scan import selective_scan_fwd, selective_scan_step  # noqa: F401
from .short_conv import short_conv_fwd, short_conv_step  # noqa: F401
