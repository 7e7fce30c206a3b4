"""What the layer operators share. Each hands its arguments to the native host module; where that finds one in another form
than the kernels read (strides, integer types, devices), the wrapper checks and converts here and calls once more."""

from __future__ import annotations

import torch

from ... import _cabi

ACTIVATIONS = (torch.float16, torch.bfloat16, torch.float32)


def require_cuda(t, what):
    if not (torch.is_tensor(t) and t.is_cuda):
        raise _cabi.LinQuantError(f"{what} runs on CUDA tensors only (no CPU path)")


def activation(name, t, shape, like):
    """Type and device of ``like``, the extents, and contiguous channels (copied where they are not)."""
    if t is None:
        return None
    assert tuple(t.shape) == tuple(shape), f"{name} has shape {tuple(t.shape)}, {tuple(shape)} expected"
    if t.dtype != like.dtype or t.dtype not in ACTIVATIONS:
        raise NotImplementedError(f"{name} must be {like.dtype} out of float16, bfloat16 and float32 (got {t.dtype})")
    if t.device != like.device:
        raise _cabi.LinQuantError(f"{name} must be on {like.device} (got {t.device})")
    return t if t.stride(-1) == 1 else t.contiguous()


def dense(name, t, shape, like):
    t = activation(name, t, shape, like)
    return None if t is None else t.contiguous()


def parameter(name, t, shape, like):
    if t is None:
        return None
    assert tuple(t.shape) == tuple(shape), f"{name} has shape {tuple(t.shape)}, {tuple(shape)} expected"
    return _cabi.f32c(t, like.device)


def integers(name, t, n, like):
    """Lengths and slots as the kernels read them: int32, dense, on the device. What int32 does not hold stays outside every
    range on its side (behind the longest prompt, no slot)."""
    if t is None:
        return None
    t = torch.as_tensor(t)
    assert tuple(t.shape) == (n,), f"{name} has shape {tuple(t.shape)}, {(n,)} expected"
    if t.dtype.is_floating_point or t.dtype == torch.bool:
        raise NotImplementedError(f"{name} must be integers (got {t.dtype})")
    if t.dtype == torch.int64:
        t = t.clamp(-1, 2**31 - 1)
    return t.to(device=like.device, dtype=torch.int32).contiguous()


def cache(name, t, shape, dtypes, like):
    """A state that is updated in place: nothing can be converted on its way."""
    assert t.dim() == len(shape) + 1 and tuple(t.shape[1:]) == tuple(shape), f"{name} has shape {tuple(t.shape)}, (slots, {', '.join(map(str, shape))}) expected"
    if t.dtype not in dtypes:
        raise NotImplementedError(f"{name} must be one of {dtypes} (got {t.dtype})")
    if t.device != like.device:
        raise _cabi.LinQuantError(f"{name} must be on {like.device} (got {t.device})")
    assert t.is_contiguous(), f"{name} is updated in place and must be contiguous"
    return t


def rows(name, t, like=None):
    """A tensor whose leading axes are rows at one pitch, copied where they are not."""
    if like is not None:
        assert t.shape == like.shape, f"{name} has shape {tuple(t.shape)}, {tuple(like.shape)} expected"
        if t.device != like.device:
            raise _cabi.LinQuantError(f"{name} must be on {like.device} (got {t.device})")
    if t.dtype not in ACTIVATIONS:
        raise NotImplementedError(f"{name}: dtype {t.dtype} is not supported by the CUDA kernels")
    return t.contiguous()


def result(r, what):
    if r is None:
        raise _cabi.LinQuantError(f"{what}: the arguments have no form that the kernels read")
    if type(r) is int:
        _cabi.check(r, what)
    return r
