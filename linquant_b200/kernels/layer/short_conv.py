"""Short causal convolution over the tokens of each channel (two to four taps), with its activation.

    y[t] = act(bias + sum_i weight[i] x[t - W + 1 + i])"""

from __future__ import annotations

from . import _layer
from ... import _cabi

_ACTIVATION = {None: False, "silu": True}


def _silu(activation):
    if activation not in _ACTIVATION:
        raise NotImplementedError(f"activation must be 'silu' or None (got {activation!r})")
    return _ACTIVATION[activation]


def short_conv_fwd(x, weight, bias=None, activation="silu", initial_state=None, lengths=None, output_final_state=False):
    """x (B,T,D) f16/bf16/f32 with any batch and token stride; weight (D,W), the last tap on the current token, W = 2..4;
    bias (D,). ``initial_state`` (B,W-1,D): the inputs ahead of the first token, oldest first (zeros without it).
    ``lengths`` (B,): tokens of each sequence that count; y is zero behind them and nothing there is read.

    Returns (y (B,T,D), final_state (B,W-1,D) or None): the last W-1 inputs of each sequence, which the next call or
    ``short_conv_step`` starts from."""
    silu = _silu(activation)
    r = _cabi.host().short_conv(x, weight, bias, silu, initial_state, lengths, output_final_state)
    if r is None:
        _layer.require_cuda(x, "short_conv_fwd")
        assert x.dim() == 3 and weight.dim() == 2, "x is (B,T,D) and weight (D,W)"
        B, T, D = x.shape
        W = weight.shape[1]
        r = _cabi.host().short_conv(
            _layer.activation("x", x, (B, T, D), x), _layer.parameter("weight", weight, (D, W), x), _layer.parameter("bias", bias, (D,), x), silu,
            _layer.dense("initial_state", initial_state, (B, W - 1, D), x), _layer.integers("lengths", lengths, B, x), bool(output_final_state))
    return _layer.result(r, "short_conv_fwd")


def short_conv_step(x, state, weight, bias=None, activation="silu", slots=None):
    """One token of each sequence: x (B,D); ``state`` (S,W-1,D) in x's type, shifted in place. ``slots`` (B,): the row of the
    state that belongs to each sequence, no row twice (row b without it); one outside 0..S-1 marks an idle entry, whose y is
    zero and which touches no state. Returns y (B,D)."""
    silu = _silu(activation)
    r = _cabi.host().short_conv_step(x, state, weight, bias, silu, slots)
    if r is None:
        _layer.require_cuda(x, "short_conv_step")
        assert x.dim() == 2 and weight.dim() == 2, "x is (B,D) and weight (D,W)"
        B, D = x.shape
        W = weight.shape[1]
        r = _cabi.host().short_conv_step(
            _layer.activation("x", x, (B, D), x), _layer.cache("state", state, (W - 1, D), (x.dtype,), x), _layer.parameter("weight", weight, (D, W), x),
            _layer.parameter("bias", bias, (D,), x), silu, _layer.integers("slots", slots, B, x))
    return _layer.result(r, "short_conv_step")
