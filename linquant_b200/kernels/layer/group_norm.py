"""Group norm with an activation, channels last: of single tokens (behind a mixer, a group a head) or over a sequence's tokens.

    y = act((x - mean) / sqrt(var + eps) weight + bias) silu(gate)"""

from __future__ import annotations

from . import _layer
from .short_conv import _silu
from ... import _cabi


def group_norm_fwd(x, num_groups, weight=None, bias=None, activation=None, gate=None, eps=1e-5, over_tokens=False, lengths=None):
    """x (.., D) f16/bf16/f32; mean and variance over the D / num_groups channels of each group, for each token by itself. With
    ``over_tokens`` x is (B,T,D) and they are taken over all tokens of a sequence as well (for encoders: later tokens reach earlier ones);
    ``lengths`` (B,): tokens of each sequence that count, y is zero behind them and nothing there is read. weight, bias (D,). ``activation`` "silu" or None. ``gate``, shaped
    and typed like x, may be a slice of a wider projection: y is multiplied by its SiLU, after the activation.

    Returns y, dense, in x's type. Sums are fp32, around each group's own mean."""
    silu = _silu(activation)
    r = _cabi.host().group_norm(x, num_groups, weight, bias, silu, gate, eps, over_tokens, lengths)
    if r is None:
        _layer.require_cuda(x, "group_norm_fwd")
        D = x.shape[-1]
        assert not over_tokens or x.dim() == 3, "x is (B,T,D) over tokens"
        assert over_tokens or lengths is None, "lengths go with over_tokens"
        if gate is not None and gate.dtype != x.dtype:
            raise NotImplementedError(f"gate must be {x.dtype} (got {gate.dtype})")
        r = _cabi.host().group_norm(
            _layer.rows("x", x), int(num_groups), _layer.parameter("weight", weight, (D,), x), _layer.parameter("bias", bias, (D,), x), silu,
            None if gate is None else _layer.rows("gate", gate, x), float(eps), bool(over_tokens),
            _layer.integers("lengths", lengths, x.shape[0] if over_tokens else 0, x))
    return _layer.result(r, "group_norm_fwd")
