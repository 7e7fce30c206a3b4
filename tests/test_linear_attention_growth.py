"""Linear attention of fp16 and bf16 prompts whose decays grow, fall and grow again, or forget what was larger, against the recurrence in
64 bits, element by element."""

import pytest
import torch

from tests import layer_reference as ref
from tests.test_linear_attention import BF16, CHUNK, F16, F32, inputs, recurrence

gpu = pytest.mark.gpu

# Decayed q.k and the state that q reads are two pieces of the type, fp32 operands three: half a step squared, or 2^-24 for each of four products
OUT = {BF16: 2.0**-16, F16: 2.0**-22, F32: 2.0**-22}


@pytest.fixture(autouse=True)
def seed():
    torch.manual_seed(17)


def lost(q, k, v, g, scale, dtype, initial=None):
    """What fp16 does not hold beside the largest value of a set that goes under one power of two: the largest is 2^14 at least, half the
    distance of the smallest numbers 2^-25, so 2^-39 of the largest at most for each value, times the other operand. The sets: a row of
    decayed q k^T; what a chunk adds to the state, decayed to the chunk's end (v on tcgen05, k on warp MMA: the larger bound of both); the state
    that q reads. Of the outputs and of the final state, in 64 bits."""
    B, T, H, V = v.shape
    K = q.shape[-1]
    o, h = torch.zeros(B, T, H, V, device="cuda", dtype=torch.float64), torch.zeros(B, H, K, V, device="cuda", dtype=torch.float64)
    if dtype != F16:
        return o, h
    q, k, v = (x.double().repeat_interleave(H // x.shape[2], 2).movedim(2, 1) for x in (q, k, v))
    g, state, part = g.double().movedim(2, 1).clamp(min=-1e3), h.clone() if initial is None else initial.double(), 2.0**-39
    for t in range(0, T, 64):
        qc, kc, vc, G = q[:, :, t:t + 64], k[:, :, t:t + 64], v[:, :, t:t + 64], g[:, :, t:t + 64].cumsum(-1)
        C = G.shape[-1]
        below = torch.ones(C, C, device="cuda", dtype=torch.bool).tril()
        decay = torch.exp(torch.where(below, G.unsqueeze(-1) - G.unsqueeze(-2), -torch.inf))
        row = ((qc @ kc.mT) * decay).abs().amax(-1, keepdim=True)
        read = torch.exp(G).unsqueeze(-1) * (state.abs().amax((2, 3), keepdim=True) * part + h.amax((2, 3), keepdim=True)) * qc.abs().sum(-1, keepdim=True)
        here = part * row * ((decay > 0).double() @ vc.abs())  # a decay of zero leaves nothing to round
        o[:, t:t + 64] = abs(scale) * (here + read).movedim(1, 2)
        out = torch.exp(G[..., -1:] - G).unsqueeze(-1)
        end = torch.exp(G[..., -1])[..., None, None]
        on = (out > 0).double()
        a = (out * vc).abs().amax((2, 3), keepdim=True) * (on * kc).abs().sum(2).unsqueeze(-1)
        b = (out * kc).abs().amax((2, 3), keepdim=True) * (on * vc).abs().sum(2).unsqueeze(-2)
        h = end * h + part * torch.maximum(a, b)
        state = end * state + (out * kc).mT @ vc
    return o, h


def outputs(o, want, mag, rel):
    """What rounds to an infinity of the type may be one: where the bound reaches the type's largest value on that side."""
    reach = torch.where(o > 0, want, -want) + rel * mag
    over = torch.isinf(o) & (reach >= torch.finfo(o.dtype).max)
    ref.check(torch.where(over, 0.0, o), torch.where(over, 0.0, want), torch.where(over, 0.0, mag), rel)


def steps(what, T, H):
    g = torch.full((1, T, H), -0.1, device="cuda")
    if what == "turns":
        g = torch.where(torch.arange(T, device="cuda") % 2 == 0, -1.0, 1.0).view(1, T, 1).expand(1, T, H).contiguous()
    elif what == "walk":
        g = torch.randn(1, T, H, device="cuda")
    elif what == "rise":
        g[:] = 0.5
    elif what == "up and down":
        g[0, 20], g[0, 40] = 30.0, -30.0
        g[0, 90], g[0, 91] = 30.0, -30.0
    elif what == "down and up":
        g[0, 20], g[0, 40] = -30.0, 30.0
        g[0, 90], g[0, 91] = -30.0, 30.0
    elif what == "up and down later":
        g[0, 20], g[0, 100] = 30.0, -30.0
    return g


@gpu
@pytest.mark.parametrize("what", ["turns", "walk", "rise", "up and down", "down and up", "up and down later"])
@pytest.mark.parametrize("dtype,K,V,pad", [(F16, 128, 128, 0), (F16, 64, 72, 0), (F16, 128, 64, 1), (BF16, 128, 128, 0), (BF16, 64, 64, 1)])
def test_decays_that_grow(what, dtype, K, V, pad):
    """Rows on 16-byte boundaries run on tcgen05, those of ``pad`` on warp MMA."""
    from linquant_b200.kernels.layer import linear_attention_fwd

    T, H = 130, 3
    q, k, v, _ = inputs(1, T, H, H, K, V, dtype, pad)
    k /= K**0.5
    g = steps(what, T, H)
    scale = K**-0.5
    wo, mag, h, m = recurrence(q, k, v, g, scale, None, None)
    o, state = linear_attention_fwd(q, k, v, g, scale=scale, output_final_state=True)
    lo, lh = lost(q, k, v, g, scale, dtype)
    chunks = T // 64 + 2
    rel = OUT[dtype] + chunks * CHUNK
    outputs(o, wo, mag + lo / rel, rel)
    ref.check(state, h, m + lh / (chunks * CHUNK), chunks * CHUNK)


@gpu
@pytest.mark.parametrize("large", ["k", "v"])
@pytest.mark.parametrize("K,V,pad", [(128, 128, 0), (64, 64, 0), (72, 64, 1)])
def test_a_reset_behind_large_values(K, V, pad, large):
    """fp16: before a step of minus infinity keys (values) are 2^35 times those behind it. What a row, or the state, keeps has its own precision."""
    from linquant_b200.kernels.layer import linear_attention_fwd

    T = 200
    q, k, v, _ = inputs(1, T, 1, 1, K, V, F32)
    g = torch.full((1, T, 1), -0.05, device="cuda")
    size = torch.full((T, 1, 1), 2.0**-20, device="cuda")
    for at in (40, 101, 190):
        g[0, at] = -torch.inf
        size[at - 30:at] = 2.0**13
    q = q * 2.0**9
    k, v = (k * size, v * 2.0**9) if large == "k" else (k * 2.0**9, v * size)
    q, k, v = (torch.cat([x.new_zeros(1, T, 1, pad), x], -1).half()[..., pad:] for x in (q, k, v))
    wo, mag, h, m = recurrence(q, k, v, g, 1.0, None, None)
    o, state = linear_attention_fwd(q, k, v, g, scale=1.0, output_final_state=True)
    lo, lh = lost(q, k, v, g, 1.0, F16)
    chunks = T // 64 + 2
    rel = OUT[F16] + chunks * CHUNK
    outputs(o, wo, mag + lo / rel, rel)
    ref.check(state, h, m + lh / (chunks * CHUNK), chunks * CHUNK)


@gpu
@pytest.mark.parametrize("start", [0.0, 1e-36])
@pytest.mark.parametrize("dtype,K", [(F16, 128), (BF16, 128), (BF16, 200), (F32, 64)])
def test_a_segment_that_grows_by_more_than_fp32_holds(dtype, K, start):
    """e^102 over 128 tokens, where the state is nothing, or so little that what comes of it is a number."""
    from linquant_b200.kernels.layer import linear_attention_fwd

    T, V = 2000, 64
    q, k, v, _ = inputs(1, T, 1, 1, K, V, dtype)
    g = torch.full((1, T, 1), -0.05, device="cuda")
    g[0, 256:384] = 0.8
    k[:, :400] = 0
    s0 = torch.randn(1, 1, K, V, device="cuda") * start
    scale = 1e-7 if start else 1.0
    wo, mag, h, m = recurrence(q, k, v, g, scale, s0, None)
    o, state = linear_attention_fwd(q, k, v, g, scale=scale, initial_state=s0, output_final_state=True)
    lo, lh = lost(q, k, v, g, scale, dtype, s0)
    chunks = T // 64 + 2
    rel = OUT[dtype] + chunks * CHUNK
    # A state of 1e-36 has come down to 3e-42 when it starts to grow, below what fp32 (2^-126) and its bf16 pieces hold in full: an fp32 product or sum there
    # is off by 2^-150, four of them a chunk, and what q reads by half of bf16's smallest number, 2^-134. Both grow from there like the state itself. Outputs in front
    # of the growth, 1e-43, are off by half of their type's smallest number.
    G, low_state, low_read = g.double().flatten(), 0.0, torch.zeros(1, T, 1, 1, device="cuda", dtype=torch.float64)
    for t in range(0, T, 64):
        up = torch.exp(G[t:t + 64].cumsum(0))
        low_read[0, t:t + 64, 0, 0] = up * (low_state + 2.0**-134)
        low_state = float(up[-1]) * low_state + 2.0**-148
    lo = lo + abs(scale) * low_read * q.double().abs().sum(-1, keepdim=True) + {F16: 0.0, BF16: 2.0**-134, F32: 2.0**-150}[dtype]
    ref.check(o, wo, mag + lo / rel, rel)
    ref.check(state, h, m + (lh + low_state) / (chunks * CHUNK), chunks * CHUNK)
