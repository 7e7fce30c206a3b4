"""Mamba-2 and Mamba layers with INT8 projections, prompts and single tokens, on the package's operators.

A layer call is one residual block: residual add and norm whose kernel writes INT8 codes, the INT8 in-projection, the short
convolution, the recurrence, the gated norm (Mamba-2; again to codes) and the INT8 out-projection. ``prefill`` takes prompts of
different lengths (right-padded), each from its first token, and leaves each sequence's convolution and recurrence state in the
layer's cache; ``step`` advances any of the cached sequences by one token. In both, a slot outside the cache marks an idle entry
of the batch, which leaves no state.

The Mamba-2 prompt runs through the INT8 SSD ops (static scales from ``calibrate``); its state, an integer carry on the
state scale, becomes the fp32 state of the token step, in the rotated basis of B and C."""

from __future__ import annotations

import torch
import torch.nn.functional as F

from ..kernels.hadamard import kronecker_hadamard_fwd
from ..kernels.layer import (gated_rms_norm_fwd, int8_linear_fwd, quantize_rows_fwd, rms_norm_fwd, selective_scan_fwd,
                             selective_scan_step, short_conv_fwd, short_conv_step)
from ..kernels.mamba2.bmm_chunk import _quant_bmm_chunk_fwd
from ..kernels.mamba2.calibration import SsdObservers
from ..kernels.mamba2.chunk_cumsum import _quant_chunk_cumsum_fwd
from ..kernels.mamba2.chunk_scan_v2 import _quant_chunk_scan_fwd
from ..kernels.mamba2.chunk_state import _quant_chunk_state_fwd_xfp_static_int8
from ..kernels.mamba2.fused_split_rotate_xBC import fused_split_rotate_quant_xBC
from ..kernels.mamba2.state_passing import _fixedpoint_state_passing_fwd

_NO_STEP = -1e4  # softplus of it is 0: a token that neither decays nor writes the state


class Int8Linear:
    """A weight (N, K) as INT8 codes with a scale per output channel, laid out once."""

    def __init__(self, weight, bias=None):
        self.codes, self.scale = quantize_rows_fwd(weight)
        self.bias = bias

    def __call__(self, x, x_scale=None, out_dtype=None):
        return int8_linear_fwd(x, self.codes, self.scale, x_scale=x_scale, bias=self.bias, out_dtype=out_dtype)


def _randn(gen, *shape, scale=1.0):
    return torch.randn(*shape, generator=gen, device="cuda") * scale


class _Cache:
    """Rows of a state, one a slot, and one behind them that takes what idle entries leave: no wait for the slots' values."""

    def __init__(self, slots, *shape, dtype=torch.float32):
        self.all = torch.zeros(slots + 1, *shape, device="cuda", dtype=dtype)
        self.rows = self.all[:slots]

    def put(self, slots, values):
        at = slots.long()
        self.all[torch.where((at >= 0) & (at < self.rows.shape[0]), at, self.rows.shape[0])] = values


class Mamba2Layer:
    """headdim 64; d_state 64 or 128; chunk 128 or 256. Random weights (seeded); ``slots`` sequences in the cache."""

    def __init__(self, d_model, nheads, d_state=128, ngroups=1, chunk=256, taps=4, slots=1, dtype=torch.float16, seed=0):
        gen = torch.Generator("cuda").manual_seed(seed)
        self.H, self.P, self.N, self.G, self.chunk, self.dtype = nheads, 64, d_state, ngroups, chunk, dtype
        self.d = nheads * 64
        self.width = self.d + 2 * ngroups * d_state  # of xBC
        self.norm, self.gate_norm = torch.ones(d_model, device="cuda"), torch.ones(self.d, device="cuda")
        self.in_proj = Int8Linear(_randn(gen, self.d + self.width + nheads, d_model, scale=d_model**-0.5))
        self.out_proj = Int8Linear(_randn(gen, d_model, self.d, scale=self.d**-0.5))
        self.conv, self.conv_bias = _randn(gen, self.width, taps, scale=taps**-0.5), _randn(gen, self.width, scale=0.1)
        self.A_log = torch.rand(nheads, generator=gen, device="cuda") * 2.0
        self.A = -torch.exp(self.A_log)
        self.D = torch.ones(nheads, device="cuda")
        want = torch.exp(torch.rand(nheads, generator=gen, device="cuda") * 4.6 - 6.9)  # steps of 0.001 to 0.1
        self.dt_bias = want + torch.log(-torch.expm1(-want))
        self.signs = torch.randint(0, 2, (ngroups, d_state), generator=gen, device="cuda").float() * 2 - 1
        self._conv_cache, self._cache = _Cache(slots, taps - 1, self.width, dtype=dtype), _Cache(slots, nheads, 64, d_state)
        self.conv_state, self.state = self._conv_cache.rows, self._cache.rows
        self.scales = None

    def _in(self, x, residual):
        """Residual add, norm and in-projection: (z, xBC, dt) as slices of one buffer, and the new residual."""
        (codes, scale), residual = rms_norm_fwd(x, self.norm, residual=residual, quantize=True)
        zxbcdt = self.in_proj(codes, scale, out_dtype=self.dtype)
        return (*zxbcdt.split([self.d, self.width, self.H], -1), residual)

    def _out(self, y, z):
        codes, scale = gated_rms_norm_fwd(y.to(self.dtype), z, self.gate_norm, quantize=True)
        return self.out_proj(codes, scale, out_dtype=self.dtype)

    def _pad(self, xBC, dt, lengths):
        """Whole chunks, and no step behind each sequence's end."""
        B, T = dt.shape[:2]
        pad = -T % self.chunk
        dt = F.pad(dt.float(), (0, 0, 0, pad), value=_NO_STEP)
        if lengths is not None:
            behind = torch.arange(T + pad, device=dt.device) >= lengths.unsqueeze(1)
            dt = torch.where(behind.unsqueeze(-1), _NO_STEP, dt)
        return F.pad(xBC, (0, 0, 0, pad)) if pad else xBC, dt

    @torch.no_grad()
    def calibrate(self, x, residual=None, lengths=None):
        """Static scales of the SSD ops from prompts (B, T, d_model) that end as the ones to come do: a prompt that ends inside a
        chunk writes its last tokens undecayed, which is more than the same tokens write at the end of a full one. Without
        ``lengths`` the prompts are also cut at every eighth of a chunk."""
        residual = torch.zeros_like(x) if residual is None else residual
        _, xBC, dt, _ = self._in(x, residual)
        xBC = short_conv_fwd(xBC, self.conv, self.conv_bias, lengths=lengths)[0]
        B, T = dt.shape[:2]
        ends = [lengths]
        if lengths is None:
            ends += [torch.full((B,), n, device=x.device) for n in range(max(1, T - self.chunk), T, self.chunk // 8)]
        obs = SsdObservers()
        for n in ends:
            xp, dp = self._pad(xBC, dt, n)
            rot = [kronecker_hadamard_fwd(t.unflatten(-1, (self.G, self.N)).contiguous(), self.signs, self.G)
                   for t in xp[..., self.d:].split(self.G * self.N, -1)]
            obs.observe(xp[..., :self.d].unflatten(-1, (self.H, self.P)), dp, self.A_log, *rot, self.chunk, dt_bias=self.dt_bias)
        self.scales = {k: v.contiguous() for k, v in obs.scales().items()}
        return self

    @torch.no_grad()
    def prefill(self, x, residual, slots, lengths=None):
        """x, residual (B,T,d_model); slots (B,) int32 rows of the cache; lengths (B,) int32 or None. Returns (out, residual)."""
        assert self.scales is not None, "calibrate() first: the SSD ops take static scales"
        S, (B, T) = self.scales, x.shape[:2]
        z, xBC, dt, residual = self._in(x, residual)
        xBC, last = short_conv_fwd(xBC, self.conv, self.conv_bias, lengths=lengths, output_final_state=True)
        self._conv_cache.put(slots, last)
        xBC, dt = self._pad(xBC, dt, lengths)
        xs, qB, qC = fused_split_rotate_quant_xBC(xBC, self.signs, self.H, self.G, self.N, self.P, 1 / S["B_scale"], 1 / S["C_scale"])
        dA, step = _quant_chunk_cumsum_fwd(dt, 1.0, self.A_log, 1.0, self.chunk, dt_bias=self.dt_bias, dt_softplus=True)
        states = _quant_chunk_state_fwd_xfp_static_int8(xs, qB, step, dA, S["alpha_hp"], S["B_scale"], S["state_scale"])
        passed, _, carry = _fixedpoint_state_passing_fwd(states.flatten(3), dA[..., -1], return_carry=True)
        self._cache.put(slots, carry.view(B, self.H, self.P, self.N) * S["state_scale"].view(1, self.H, self.P, 1))
        cb = _quant_bmm_chunk_fwd(qC, S["C_scale"], qB, S["B_scale"], self.chunk, S["cb_scale"])
        y = _quant_chunk_scan_fwd(cb, xs, step, dA, qC, S["C_scale"], passed.view_as(states), self.D, 1.0, S["state_scale"], S["cb_scale"])
        return self._out(y[:, :T].flatten(2), z), residual

    @torch.no_grad()
    def step(self, x, residual, slots):
        """x, residual (B,d_model): one token of each of the sequences in ``slots``. Returns (out, residual)."""
        z, xBC, dt, residual = self._in(x, residual)
        return self._out(self._mix_step(xBC, dt, slots), z), residual

    def _mix_step(self, xBC, dt, slots):
        xBC = short_conv_step(xBC, self.conv_state, self.conv, self.conv_bias, slots=slots)
        BC = xBC[:, None, self.d:].unflatten(-1, (2 * self.G, self.N))
        BC = kronecker_hadamard_fwd(BC, torch.cat([self.signs, self.signs]), 2 * self.G)[:, 0]  # the state's basis
        x = xBC[:, :self.d].unflatten(-1, (self.H, self.P))
        y = selective_scan_step(self.state, x, dt, self.A, BC[:, :self.G], BC[:, self.G:], D=self.D, dt_bias=self.dt_bias, slots=slots)
        return y.flatten(1)


class MambaLayer:
    """One decay rate per channel and state; the gate rides the scan. Random weights (seeded)."""

    def __init__(self, d_model, d_inner, d_state=16, dt_rank=None, taps=4, slots=1, dtype=torch.bfloat16, seed=0):
        gen = torch.Generator("cuda").manual_seed(seed)
        self.d, self.N, self.R, self.dtype = d_inner, d_state, dt_rank or max(1, d_model // 16), dtype
        self.norm = torch.ones(d_model, device="cuda")
        self.in_proj = Int8Linear(_randn(gen, 2 * d_inner, d_model, scale=d_model**-0.5))
        self.x_proj = Int8Linear(_randn(gen, self.R + 2 * d_state, d_inner, scale=d_inner**-0.5))
        self.dt_proj = Int8Linear(_randn(gen, d_inner, self.R, scale=self.R**-0.5))
        self.out_proj = Int8Linear(_randn(gen, d_model, d_inner, scale=d_inner**-0.5))
        self.conv, self.conv_bias = _randn(gen, d_inner, taps, scale=taps**-0.5), _randn(gen, d_inner, scale=0.1)
        self.A = -torch.arange(1, d_state + 1, device="cuda").float().expand(d_inner, d_state).contiguous()
        self.D = torch.ones(d_inner, device="cuda")
        want = torch.exp(torch.rand(d_inner, generator=gen, device="cuda") * 4.6 - 6.9)
        self.dt_bias = want + torch.log(-torch.expm1(-want))
        self._conv_cache, self._cache = _Cache(slots, taps - 1, d_inner, dtype=dtype), _Cache(slots, d_inner, d_state)
        self.conv_state, self.state = self._conv_cache.rows, self._cache.rows

    def _in(self, x, residual):
        (codes, scale), residual = rms_norm_fwd(x, self.norm, residual=residual, quantize=True)
        return (*self.in_proj(codes, scale, out_dtype=self.dtype).split(self.d, -1), residual)

    def _operands(self, u):
        """dt, B, C of the convolved inputs; B and C as groups of one."""
        dt, B, C = self.x_proj(u).split([self.R, self.N, self.N], -1)
        return self.dt_proj(dt), B.unsqueeze(-2), C.unsqueeze(-2)

    @torch.no_grad()
    def prefill(self, x, residual, slots, lengths=None):
        u, z, residual = self._in(x, residual)
        u, last = short_conv_fwd(u, self.conv, self.conv_bias, lengths=lengths, output_final_state=True)
        self._conv_cache.put(slots, last)
        dt, B, C = self._operands(u)
        y, last = selective_scan_fwd(u, dt, self.A, B, C, D=self.D, z=z, dt_bias=self.dt_bias, lengths=lengths, output_final_state=True)
        self._cache.put(slots, last)
        return self.out_proj(y), residual

    @torch.no_grad()
    def step(self, x, residual, slots):
        u, z, residual = self._in(x, residual)
        u = short_conv_step(u, self.conv_state, self.conv, self.conv_bias, slots=slots)
        dt, B, C = self._operands(u)
        y = selective_scan_step(self.state, u, dt, self.A, B, C, D=self.D, z=z, dt_bias=self.dt_bias, slots=slots)
        return self.out_proj(y), residual
