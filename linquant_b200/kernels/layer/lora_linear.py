"""INT8 matrix product with low-rank adapters of many requests at once: each token's own beside the shared projection.

    y[m,n] = (sum_k c[m,k] w[n,k]) x_scale[m] w_scale[n] + bias[n] + scaling[l] sum_r (sum_k x[m,k] a[l,r,k]) b[l,n,r],   l = adapters[m]"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from . import _layer
from .int8_linear import _codes
from ... import _cabi


def stack_adapters(pairs):
    """[(a (r,K), b (N,r)), ..] of any ranks up to 128 as the (L,R,K) and (L,N,R) that ``lora_linear_fwd`` reads in place, R the
    largest rank rounded up to 8: zeros add nothing. Lay adapters out once."""
    pairs = list(pairs)
    assert pairs, "no adapters"
    (a0, b0), R = pairs[0], (max(a.shape[0] for a, _ in pairs) + 7) // 8 * 8
    for a, b in pairs:
        assert a.dim() == 2 and b.dim() == 2 and a.shape[0] == b.shape[1] and a.shape[1] == a0.shape[1] and b.shape[0] == b0.shape[0], (
            f"a (r, K) and b (N, r) do not fit: {tuple(a.shape)}, {tuple(b.shape)}")
    return (torch.stack([F.pad(a, (0, 0, 0, R - a.shape[0])) for a, _ in pairs]), torch.stack([F.pad(b, (0, R - b.shape[1])) for _, b in pairs]))


def lora_linear_fwd(x, w, w_scale, lora_a, lora_b, adapters, scaling=None, x_scale=None, bias=None, out_dtype=None):
    """``int8_linear_fwd`` (x (.., K): codes with ``x_scale``, or values that are quantised row by row for the shared product; w (N,K)
    int8, w_scale, bias (N,)) and to each row its adapter's share, added before y is rounded. The adapters see x as it is
    given: the values, or codes times their scale.

    lora_a (L,R,K), lora_b (L,N,R) of one type, f16/bf16/f32; R up to 128, a multiple of 8 is read in place, others are copied:
    lay adapters out once with ``stack_adapters``. ``adapters`` (..): which of the L each row has; one outside 0..L-1 has none.
    ``scaling`` a number, one on the device or (L,). Rows that lie next to one another with one adapter share its reads. Returns y (.., N) in
    ``out_dtype`` (x's type; bf16 for codes).

    The share is an fp32 sum whatever y's type, and joins the shared product's before either is rounded: it may be larger than y's type holds. With
    16-bit outputs of more than 16 rows x a and b go into it as two bf16 numbers each (16 bits), and it takes up to 1 GiB of scratch."""
    r = _cabi.host().lora_linear(x, w, w_scale, lora_a, lora_b, adapters, scaling, x_scale, bias, out_dtype)
    if r is None:
        _layer.require_cuda(x, "lora_linear_fwd")
        assert w.dim() == 2 and x.dim() >= 1 and x.shape[-1] == w.shape[1], f"x (.., K) and w (N, K) do not fit: {tuple(x.shape)}, {tuple(w.shape)}"
        N, K = w.shape
        assert lora_a.dim() == 3 and lora_b.dim() == 3 and lora_a.shape[2] == K and tuple(lora_b.shape) == (lora_a.shape[0], N, lora_a.shape[1]), (
            f"lora_a (L, R, K) and lora_b (L, N, R) do not fit: {tuple(lora_a.shape)}, {tuple(lora_b.shape)}")
        for name, t in (("w", w), ("lora_a", lora_a), ("lora_b", lora_b)):
            if t.device != x.device:
                raise _cabi.LinQuantError(f"{name} must be on {x.device} (got {t.device})")
        if lora_a.dtype != lora_b.dtype or lora_a.dtype not in _layer.ACTIVATIONS:
            raise NotImplementedError(f"lora_a and lora_b must be of one type out of float16, bfloat16 and float32 (got {lora_a.dtype}, {lora_b.dtype})")
        assert (x.dtype == torch.int8) == (x_scale is not None), "x_scale goes with INT8 codes, and only with them"
        if out_dtype is not None and out_dtype not in _layer.ACTIVATIONS:
            raise NotImplementedError(f"out_dtype {out_dtype} is not supported by the CUDA kernels")
        lead, pad = x.shape[:-1], -lora_a.shape[1] % 8
        adapters = torch.as_tensor(adapters)
        assert adapters.shape == lead, f"adapters has shape {tuple(adapters.shape)}, {tuple(lead)} expected"
        if torch.is_tensor(scaling) and scaling.dim() == 0:  # on the device it is read there
            scaling = scaling.expand(lora_a.shape[0]) if scaling.is_cuda else float(scaling)
        if pad:
            lora_a, lora_b = F.pad(lora_a, (0, 0, 0, pad)), F.pad(lora_b, (0, pad))
        lora_b = lora_b.contiguous()
        r = _cabi.host().lora_linear(
            _codes("x", x) if x_scale is not None else _layer.rows("x", x), _codes("w", w), _layer.parameter("w_scale", w_scale, (N,), x),
            lora_a.contiguous(), lora_b if lora_b.data_ptr() % 16 == 0 else lora_b.clone(), _layer.integers("adapters", adapters.reshape(-1), lead.numel(), x).view(lead),
            _layer.parameter("scaling", scaling, (lora_a.shape[0],), x) if torch.is_tensor(scaling) else None if scaling is None else float(scaling),
            _layer.parameter("x_scale", x_scale, lead, x), _layer.parameter("bias", bias, (N,), x), out_dtype)
    return _layer.result(r, "lora_linear_fwd")
