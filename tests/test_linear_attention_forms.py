"""The forms of linear attention's prompts, held to what their pieces leave: on tcgen05 (16-bit operands of more than 64 tokens, K <= 128, rows
on 16-byte boundaries) and on warp MMA (the others)."""

import pytest
import torch

from tests import layer_reference as ref
from tests.test_linear_attention import BF16, CHUNK, F16, F32, ints, randn, recurrence
from tests.test_linear_attention_growth import lost

gpu = pytest.mark.gpu

# Beside its own rounding an output has those of the terms it is summed of. A term goes through a decayed q.k or through the state that q
# reads, each in two pieces of the type: half a step squared; three pieces of fp32 operands leave 2^-24 a product, four of which meet.
TERMS = {BF16: 2.0**-16, F16: 2.0**-22, F32: 2.0**-22}


@pytest.fixture(autouse=True)
def seed():
    torch.manual_seed(11)


def rows(B, T, heads, width, pitch, dtype):
    """Heads of ``width`` values, ``pitch`` apart; what lies between them is no number."""
    x = torch.full((B, T, heads, pitch), float("nan"), device="cuda", dtype=dtype)
    x[..., :width] = randn(B, T, heads, width, dtype=dtype)
    return x[..., :width]


def compare(q, k, v, g, s0, n):
    from linquant_b200.kernels.layer import linear_attention_fwd

    B, T, H, V = v.shape
    K, dtype = q.shape[-1], q.dtype
    want = recurrence(q, k, v, g, None, s0, n)
    on = torch.ones(B, T, 1, 1, device="cuda", dtype=torch.bool) if n is None else (n.view(B, 1) > torch.arange(T, device="cuda"))[..., None, None]
    lo, lh = lost(*(torch.where(on, x, 0.0) for x in (q, k, v)), torch.where(on[..., 0], g, 0.0), K**-0.5, dtype, s0)
    if n is not None:  # what lies behind a sequence takes no part
        for b in range(B):
            for x in (q, k, v, g):
                x[b, max(int(n[b]), 0):] = float("nan")
    o, state = linear_attention_fwd(q, k, v, g, initial_state=s0, lengths=n, output_final_state=True)
    chunks = T // 64 + 2
    rel = TERMS[dtype] + chunks * CHUNK
    ref.check(o, want[0], want[1] + lo / rel, rel)
    ref.check(state, want[2], want[3] + lh / (chunks * CHUNK), chunks * CHUNK)
    for b in range(B):
        if n is not None:
            assert not o[b, max(int(n[b]), 0):].any()
    again, _ = linear_attention_fwd(q, k, v, g, initial_state=s0, lengths=n)
    assert torch.equal(o, again)


def decays(B, T, H):
    return -2 * torch.rand(B, T, H, device="cuda")**4


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,T,Hk,H,K,V,lengths,initial", [
    (1, 1500, 1, 1, 128, 128, None, False),                              # six segments
    (1, 2500, 1, 2, 64, 64, None, True),
    (4, 1600, 1, 1, 128, 64, (1600, 700, 65, 0), True),                  # sequences that end inside segments and before them
    (3, 900, 1, 2, 128, 128, (257, 900, 256), False),                    # and at a segment's end
    (2, 130, 2, 2, 128, 128, (129, 64), True),                           # one segment
])
def test_segments_on_tcgen05(B, T, Hk, H, K, V, lengths, initial, dtype):
    q, k, v = rows(B, T, Hk, K, K, dtype), rows(B, T, Hk, K, K, dtype), rows(B, T, H, V, V, dtype)
    compare(q, k, v, decays(B, T, H), randn(B, H, K, V) if initial else None, None if lengths is None else ints(*lengths))


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,K,V,lengths", [
    (200, 32, 64, None), (130, 8, 64, None), (200, 1, 64, None), (200, 72, 128, (131,)), (130, 100, 64, None), (1500, 100, 64, None), (130, 127, 64, None),
    (200, 64, 70, None), (200, 128, 77, (140,)), (1500, 128, 70, (1130,)), (130, 40, 1, None), (1500, 33, 130, None),  # outputs off 16-byte boundaries
])
def test_widths_on_tcgen05(T, K, V, lengths, dtype):
    """Channels of q, k and v that end inside their tiles, heads on 16-byte boundaries all the same."""
    B, Hk, H = 1, 1, 2
    up = lambda n: (n + 7) // 8 * 8  # noqa: E731
    q, k, v = rows(B, T, Hk, K, up(K), dtype), rows(B, T, Hk, K, up(K) + 8, dtype), rows(B, T, H, V, up(V), dtype)
    compare(q, k, v, decays(B, T, H), None, None if lengths is None else ints(*lengths))


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("T,K,V,pitch", [
    (1, 128, 128, 128), (8, 128, 128, 128), (64, 128, 128, 128), (64, 64, 72, 64),  # calls of one chunk
    (130, 128, 128, 129), (200, 64, 64, 65), (1500, 100, 70, 101),                   # heads off 16-byte boundaries
    (130, 200, 64, 200), (200, 256, 32, 256), (1500, 136, 40, 136),                  # wide heads
])
def test_warp_mma(T, K, V, pitch, dtype):
    """Calls of one chunk among them."""
    q, k, v = rows(1, T, 2, K, pitch, dtype), rows(1, T, 2, K, pitch, dtype), rows(1, T, 2, V, V, dtype)
    compare(q, k, v, decays(1, T, 2), None, None)
