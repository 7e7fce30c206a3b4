"""Linear-attention layer with a decay a head, INT8 projections and low-rank adapters of its own for each sequence.

A layer call is one residual block: residual add and norm whose kernel writes INT8 codes, the INT8 in-projection, linear attention,
a norm of each head with the gate, and the INT8 out-projection. Queries, keys, values and gate stay slices of the in-projection's
rows. Both projections may carry adapters: ``adapters`` names each sequence's, one outside the stack is none. ``prefill`` takes
prompts of different lengths (right-padded) from their first token or, with ``resume``, from the state in the cache, so that a long
prompt may come in parts; ``step`` advances any of the cached sequences by one token. A slot outside the cache marks an idle entry
of the batch, which leaves no state."""

from __future__ import annotations

import torch
import torch.nn.functional as F

from ..kernels.layer import (group_norm_fwd, int8_linear_fwd, linear_attention_fwd, linear_attention_step, lora_linear_fwd, rms_norm_fwd,
                             stack_adapters)
from .mamba import Int8Linear, _Cache, _randn

_DECAY_UNIT = 16.0  # the logarithm of a decay is logsigmoid over it


class _AdaptedLinear(Int8Linear):
    """The shared projection and, once it has some, adapters beside it."""

    def __init__(self, weight):
        super().__init__(weight)
        self.a = self.b = self.scaling = None

    def adapt(self, pairs, scaling, dtype):
        self.a, self.b = (t.to(device="cuda", dtype=dtype) for t in stack_adapters(pairs))
        self.scaling = scaling

    def __call__(self, x, x_scale=None, out_dtype=None, adapters=None):
        if adapters is None or self.a is None:
            return int8_linear_fwd(x, self.codes, self.scale, x_scale=x_scale, out_dtype=out_dtype)
        return lora_linear_fwd(x, self.codes, self.scale, self.a, self.b, adapters, scaling=self.scaling, x_scale=x_scale, out_dtype=out_dtype)


class LinearAttentionLayer:
    """``heads`` of values (head_v wide) share ``kv_heads`` of queries and keys (head_k wide, up to 256) evenly. Random weights
    (seeded); ``slots`` sequences in the cache."""

    def __init__(self, d_model, heads, head_k=128, head_v=128, kv_heads=None, slots=1, dtype=torch.bfloat16, seed=0):
        gen = torch.Generator("cuda").manual_seed(seed)
        self.H, self.Hk, self.K, self.V, self.dtype = heads, kv_heads or heads, head_k, head_v, dtype
        self.parts = [self.Hk * head_k, self.Hk * head_k, heads * head_v, heads * head_v, heads]  # q, k, v, gate, decay
        self.parts.append(-sum(self.parts) % 8)  # rows of whole 16 bytes: the operators' fast paths take them
        self.norm, self.head_norm = torch.ones(d_model, device="cuda"), torch.ones(heads * head_v, device="cuda")
        self.in_proj = _AdaptedLinear(_randn(gen, sum(self.parts), d_model, scale=d_model**-0.5))
        self.out_proj = _AdaptedLinear(_randn(gen, d_model, heads * head_v, scale=(heads * head_v) ** -0.5))
        self.decay_bias = torch.rand(heads, generator=gen, device="cuda") * 4.0
        self._cache = _Cache(slots, heads, head_k, head_v)
        self.state = self._cache.rows

    def adapt(self, in_pairs=None, out_pairs=None, scaling=None):
        """[(a (r, inputs), b (outputs, r)), ..] of the in- and the out-projection, laid out once."""
        for proj, pairs in ((self.in_proj, in_pairs), (self.out_proj, out_pairs)):
            if pairs is not None:
                proj.adapt(pairs, scaling, self.dtype)
        return self

    def _in(self, x, residual, adapters):
        (codes, scale), residual = rms_norm_fwd(x, self.norm, residual=residual, quantize=True)
        q, k, v, z, a, _ = self.in_proj(codes, scale, self.dtype, adapters).split(self.parts, -1)
        g = F.logsigmoid(a.float() + self.decay_bias) / _DECAY_UNIT
        return q.unflatten(-1, (self.Hk, self.K)), k.unflatten(-1, (self.Hk, self.K)), v.unflatten(-1, (self.H, self.V)), g, z, residual

    def _out(self, o, z, adapters):
        return self.out_proj(group_norm_fwd(o.flatten(-2), self.H, self.head_norm, gate=z), None, self.dtype, adapters)

    @torch.no_grad()
    def prefill(self, x, residual, slots, lengths=None, adapters=None, resume=False):
        """x, residual (B,T,d_model); slots, lengths, adapters (B,) int32. Returns (out, residual)."""
        which = None if adapters is None else adapters.unsqueeze(1).expand(x.shape[:2]).contiguous()
        q, k, v, g, z, residual = self._in(x, residual, which)
        o, last = linear_attention_fwd(q, k, v, g, initial_state=self._cache.take(slots) if resume else None, lengths=lengths, output_final_state=True)
        self._cache.put(slots, last)
        return self._out(o, z, which), residual

    @torch.no_grad()
    def step(self, x, residual, slots, adapters=None):
        """x, residual (B,d_model): one token of each of the sequences in ``slots``. Returns (out, residual)."""
        q, k, v, g, z, residual = self._in(x, residual, adapters)
        return self._out(linear_attention_step(self.state, q, k, v, g, slots=slots), z, adapters), residual
