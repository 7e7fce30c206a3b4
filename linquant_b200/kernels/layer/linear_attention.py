"""Linear attention with a decay for each head, in floating point: prompts of any length and single tokens.

    S_t = exp(g_t) S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t

The state has the layout of the INT8 chunk op's carry (``linquant_b200.kernels.zoo.chunk_simple_gla_int8``): what that call
leaves, these calls continue, and the other way round."""

from __future__ import annotations

import torch

from . import _layer
from ... import _cabi


def _decay(g, like, lead, H):
    """fp32 on the device, one for each token and head or one a head, in place where it can be."""
    if g is None:
        return None
    g = torch.as_tensor(g)
    assert tuple(g.shape) in ((H,), (*lead, H)), f"g has shape {tuple(g.shape)}, {(*lead, H)} or {(H,)} expected"
    if not g.dtype.is_floating_point:
        raise NotImplementedError(f"g must be floating point (got {g.dtype})")
    return g.to(device=like.device, dtype=torch.float32)


def _heads(what, q, k, v, dims):
    _layer.require_cuda(q, what)
    assert q.dim() == dims and v.dim() == dims, f"{what}: q, k and v have {dims} axes"
    lead, (H, V) = tuple(q.shape[:-2]), v.shape[-2:]
    assert H % max(q.shape[-2], 1) == 0, f"{what}: the {H} heads of v share the {q.shape[-2]} of q and k evenly"
    return lead, H, V, _layer.activation("q", q, q.shape, q), _layer.activation("k", k, q.shape, q), _layer.activation("v", v, (*lead, H, V), q)


def linear_attention_fwd(q, k, v, g=None, scale=None, initial_state=None, lengths=None, output_final_state=False):
    """q, k (B,T,Hk,K), v (B,T,H,V) of one type, f16/bf16/f32, with any strides of batch, token and head; K up to 256, any V; H a
    multiple of Hk, whose heads are shared by H/Hk heads of v each. g (B,T,H) or, constant, (H,): log-decays, read as fp32
    (none: no decay). ``scale``: 1/sqrt(K) without one. ``initial_state`` (B,H,K,V) fp32. ``lengths`` (B,): tokens of each sequence that
    count; o is zero behind them and nothing there is read.

    An infinity or NaN in q, k, v or g may reach every token of its chunk of 64, the ones before it too, and those that follow. Log-decays may be
    minus infinity (what came before is forgotten) or positive, up to 88 in all between two tokens of a chunk.

    Returns (o (B,T,H,V), final_state (B,H,K,V) fp32 or None). States are fp32 throughout; outputs are rounded once. In fp16 what a chunk leaves to the state is kept to 2^-39 of the chunk's largest decayed value."""
    r = _cabi.host().linear_attention(q, k, v, g, scale, initial_state, lengths, output_final_state)
    if r is None:
        lead, H, V, q, k, v = _heads("linear_attention_fwd", q, k, v, 4)
        r = _cabi.host().linear_attention(
            q, k, v, _decay(g, q, lead, H), None if scale is None else float(scale), _layer.parameter("initial_state", initial_state, (lead[0], H, q.shape[-1], V), q),
            _layer.integers("lengths", lengths, lead[0], q), bool(output_final_state))
    return _layer.result(r, "linear_attention_fwd")


def linear_attention_step(state, q, k, v, g=None, scale=None, slots=None):
    """One token of each sequence, ``state`` (S,H,K,V) updated in place (f32, or rounded to f16 / bf16 once a token; the products with
    k and q are fp32). q, k (B,Hk,K), v (B,H,V), g (B,H) or (H,). ``slots`` (B,): the row of the state that belongs to each
    sequence, no row twice (row i without it); one outside 0..S-1 marks an idle entry, whose o is zero and which touches no
    state. Returns o (B,H,V)."""
    r = _cabi.host().linear_attention_step(state, q, k, v, g, scale, slots)
    if r is None:
        lead, H, V, q, k, v = _heads("linear_attention_step", q, k, v, 3)
        r = _cabi.host().linear_attention_step(
            _layer.cache("state", state, (H, q.shape[-1], V), (torch.float32, torch.bfloat16, torch.float16), q), q, k, v, _decay(g, q, lead, H),
            None if scale is None else float(scale), _layer.integers("slots", slots, lead[0], q))
    return _layer.result(r, "linear_attention_step")
