"""INT8 matrix product with a scale per token and per output channel, and the row quantiser that feeds it.

    y[m,n] = (sum_k x[m,k] w[n,k]) x_scale[m] w_scale[n] + bias[n]"""

from __future__ import annotations

import torch

from . import _layer
from ... import _cabi


def quantize_rows_fwd(x):
    """Symmetric INT8 codes of the rows of x (.., K) f16/bf16/f32, of any length: scale = amax / 127 in fp32, codes = x / scale rounded half
    away from zero. Returns (codes (.., K) int8, scale (..) fp32); the rows of the codes lie at a pitch of K rounded up to 16
    bytes, as ``int8_linear_fwd`` reads them in place. Also lays out a weight (N, K) once, its scales per output channel. A
    row of zeros has scale 0; one with an infinity or NaN a scale that is not finite, and so has its product."""
    r = _cabi.host().quantize_rows(x)
    if r is None:
        _layer.require_cuda(x, "quantize_rows_fwd")
        r = _cabi.host().quantize_rows(_layer.rows("x", x))
    return _layer.result(r, "quantize_rows_fwd")


def _codes(name, t):
    """Rows of codes on 16-byte boundaries: copied where they are not."""
    if t.dtype != torch.int8:
        raise NotImplementedError(f"{name} must be int8 codes (got {t.dtype})")
    K = t.shape[-1]
    buf = torch.empty(*t.shape[:-1], (K + 15) // 16 * 16, device=t.device, dtype=torch.int8)
    out = buf[..., :K]
    out.copy_(t)
    return out


def int8_linear_fwd(x, w, w_scale, x_scale=None, bias=None, out_dtype=None):
    """x (.., K): INT8 codes with ``x_scale`` (..), or f16/bf16/f32 values that are quantised row by row first; w (N,K) int8,
    w_scale, bias (N,). K up to 131071; sums are exact in INT32. Codes are read in place where their rows start on 16-byte
    boundaries and are copied otherwise: lay weights out once with ``quantize_rows_fwd``. Returns y (.., N) in ``out_dtype``
    (x's type; bf16 for codes)."""
    r = _cabi.host().int8_linear(x, w, w_scale, x_scale, bias, out_dtype)
    if r is None:
        _layer.require_cuda(x, "int8_linear_fwd")
        assert w.dim() == 2 and x.dim() >= 1 and x.shape[-1] == w.shape[1], f"x (.., K) and w (N, K) do not fit: {tuple(x.shape)}, {tuple(w.shape)}"
        if w.device != x.device:
            raise _cabi.LinQuantError(f"w must be on {x.device} (got {w.device})")
        assert (x.dtype == torch.int8) == (x_scale is not None), "x_scale goes with INT8 codes, and only with them"
        if out_dtype is not None and out_dtype not in _layer.ACTIVATIONS:
            raise NotImplementedError(f"out_dtype {out_dtype} is not supported by the CUDA kernels")
        N = w.shape[0]
        r = _cabi.host().int8_linear(
            _codes("x", x) if x_scale is not None else _layer.rows("x", x), _codes("w", w), _layer.parameter("w_scale", w_scale, (N,), x),
            _layer.parameter("x_scale", x_scale, x.shape[:-1], x), _layer.parameter("bias", bias, (N,), x), out_dtype)
    return _layer.result(r, "int8_linear_fwd")
