"""Norms around a block: residual add and norms in one pass, the gated norm behind a mixer, and their INT8 codes.

    norm(v) = v / sqrt(mean(v^2) + eps)"""

from __future__ import annotations

import torch

from . import _layer
from ... import _cabi


def _out_dtype(t):
    if t is not None and t not in _layer.ACTIVATIONS:
        raise NotImplementedError(f"out_dtype {t} is not supported by the CUDA kernels")
    return t


def rms_norm_fwd(x, weight, residual=None, residual_scale=1.0, post_weight=None, eps=1e-5, quantize=False, out_dtype=None):
    """    r = residual + residual_scale P(x),   P(x) = x, or norm(x) post_weight
        y = norm(r) weight                       (norm(x) weight without a residual)

    x (.., D) f16/bf16/f32, D up to 16384; ``residual`` of x's type or fp32; ``residual_scale`` a number or (D,); weight,
    post_weight (D,). ``weight=None`` stops at r (a norm behind the last block). With ``quantize`` y comes as (codes, scale)
    of its rows, ready for ``int8_linear_fwd``. r enters the norm unrounded. Returns y, or (y, r) with a residual."""
    r = _cabi.host().rms_norm(x, weight, residual, residual_scale, post_weight, eps, quantize, out_dtype)
    if r is None:
        _layer.require_cuda(x, "rms_norm_fwd")
        D = x.shape[-1]
        if residual is not None and residual.dtype not in (x.dtype, torch.float32):
            raise NotImplementedError(f"residual must be {x.dtype} or float32 (got {residual.dtype})")
        scale = _layer.parameter("residual_scale", residual_scale, (D,), x) if torch.is_tensor(residual_scale) and residual_scale.dim() else float(residual_scale)
        r = _cabi.host().rms_norm(
            _layer.rows("x", x), _layer.parameter("weight", weight, (D,), x), None if residual is None else _layer.rows("residual", residual, x), scale,
            _layer.parameter("post_weight", post_weight, (D,), x), float(eps), bool(quantize), _out_dtype(out_dtype))
    y, res = _layer.result(r, "rms_norm_fwd")
    return y if residual is None else (y, res)


def gated_rms_norm_fwd(x, gate, weight, group_size=None, gate_first=True, eps=1e-5, quantize=False, out_dtype=None):
    """y = norm(x silu(gate)) weight, or norm(x) weight silu(gate) with ``gate_first=False``; the norm over each
    ``group_size`` channels, at most 16384 (all of them without it). x, gate (.., D) of one type, the gate a slice of a wider projection
    if need be; weight (D,). With ``quantize`` y comes as (codes, scale) of its rows."""
    r = _cabi.host().gated_rms_norm(x, gate, weight, group_size, gate_first, eps, quantize, out_dtype)
    if r is None:
        _layer.require_cuda(x, "gated_rms_norm_fwd")
        if gate.dtype != x.dtype:
            raise NotImplementedError(f"gate must be {x.dtype} (got {gate.dtype})")
        r = _cabi.host().gated_rms_norm(
            _layer.rows("x", x), _layer.rows("gate", gate, x), _layer.parameter("weight", weight, (x.shape[-1],), x),
            None if group_size is None else int(group_size), bool(gate_first), float(eps), bool(quantize), _out_dtype(out_dtype))
    return _layer.result(r, "gated_rms_norm_fwd")
