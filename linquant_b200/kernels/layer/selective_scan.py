"""Selective scan: a state space recurrence whose step, input and read-out depend on the token.

    dt  = clamp(softplus(dt + dt_bias), *dt_limit)
    h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t,   y_t = C_t . h_t + D u_t,   y_t *= silu(z_t)

The prompt form has one decay rate per channel and state. Prompts of the form with one rate per head are the INT8 SSD ops of
``linquant_b200.kernels.mamba2``; its single tokens are here."""

from __future__ import annotations

import torch

from . import _layer
from ... import _cabi

_INF = float("inf")


def selective_scan_fwd(u, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=True, dt_limit=(0.0, _INF), initial_state=None,
                       lengths=None, output_final_state=False):
    """u, dt, z (b,T,d) and B, C (b,T,G,N) of one type, f16/bf16/f32, with any batch and token stride (B and C serve the
    d/G channels of their group); A (d,N) negative, D, dt_bias (d,); N up to 256. ``initial_state`` (b,d,N) fp32.
    ``lengths`` (b,): tokens of each sequence that count; y is zero behind them and nothing there is read.

    Returns (y (b,T,d), final_state (b,d,N) fp32 or None). States are fp32 throughout."""
    r = _cabi.host().selective_scan(u, dt, A, B, C, D, z, dt_bias, dt_softplus, dt_limit[0], dt_limit[1], initial_state, lengths, output_final_state)
    if r is None:
        _layer.require_cuda(u, "selective_scan_fwd")
        assert u.dim() == 3 and B.dim() == 4, "u is (b,T,d), B and C are (b,T,G,N)"
        (b, T, d), (G, N) = u.shape, B.shape[2:]
        r = _cabi.host().selective_scan(
            _layer.activation("u", u, (b, T, d), u), _layer.activation("dt", dt, (b, T, d), u), _layer.parameter("A", A, (d, N), u),
            _layer.activation("B", B, (b, T, G, N), u), _layer.activation("C", C, (b, T, G, N), u), _layer.parameter("D", D, (d,), u),
            _layer.activation("z", z, (b, T, d), u), _layer.parameter("dt_bias", dt_bias, (d,), u), bool(dt_softplus), float(dt_limit[0]),
            float(dt_limit[1]), _layer.parameter("initial_state", initial_state, (b, d, N), u), _layer.integers("lengths", lengths, b, u),
            bool(output_final_state))
    return _layer.result(r, "selective_scan_fwd")


def selective_scan_step(state, u, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=True, dt_limit=(0.0, _INF), slots=None):
    """One token of each sequence, ``state`` updated in place (f32, or rounded to f16 / bf16 once a token; the sum and the
    product with C are fp32).

    One decay rate per channel and state: u, dt, z (b,d), A (d,N), D, dt_bias (d,), state (S,d,N). One per head: u, z
    (b,H,P), dt (b,H), A, dt_bias (H,), D (H,) or (H,P), state (S,H,P,N). B, C (b,G,N). ``slots`` (b,): the row of the state
    that belongs to each sequence, no row twice (row i without it); one outside 0..S-1 marks an idle entry, whose y is zero
    and which touches no state. Returns y shaped like u."""
    r = _cabi.host().selective_scan_step(state, u, dt, A, B, C, D, z, dt_bias, dt_softplus, dt_limit[0], dt_limit[1], slots)
    if r is None:
        _layer.require_cuda(u, "selective_scan_step")
        assert u.dim() in (2, 3) and B.dim() == 3, "u is (b,d) or (b,H,P), B and C are (b,G,N)"
        b, (G, N), ch = u.shape[0], B.shape[1:], tuple(u.shape[1:])
        heads = u.dim() == 3
        flat = lambda name, t: None if t is None else _layer.activation(name, t, u.shape, u).flatten(1).view(u.shape)  # noqa: E731
        if D is not None and heads and D.dim() == 2:
            D = D.expand(ch)
        r = _cabi.host().selective_scan_step(
            _layer.cache("state", state, (*ch, N), (torch.float32, torch.bfloat16, torch.float16), u), flat("u", u),
            _layer.activation("dt", dt, (b, ch[0]), u), _layer.parameter("A", A, ch[:1] if heads else (*ch, N), u),
            _layer.activation("B", B, (b, G, N), u), _layer.activation("C", C, (b, G, N), u),
            _layer.parameter("D", D, ch if heads and D is not None and D.dim() == 2 else ch[:1], u), flat("z", z),
            _layer.parameter("dt_bias", dt_bias, ch[:1], u), bool(dt_softplus), float(dt_limit[0]), float(dt_limit[1]),
            _layer.integers("slots", slots, b, u))
    return _layer.result(r, "selective_scan_step")
