"""Layers: tokens one by one continue a prompt as the longer prompt does; ragged prompts leave every sequence's own state."""

import pytest
import torch

from tests.helpers import rel_l2

pytestmark = pytest.mark.gpu


def inputs(B, T, d, dtype, seed=3):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(B, T, d, generator=g, device="cuda", dtype=dtype), torch.randn(B, T, d, generator=g, device="cuda", dtype=dtype)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def drive(layer, x, r, lengths, extra):
    """The prompts up to ``lengths``, then ``extra`` tokens each; outputs of those, (B, extra, d)."""
    B = x.shape[0]
    slots = ints(*range(B - 1, -1, -1))
    T = max(lengths)
    layer.prefill(x[:, :T], r[:, :T], slots, ints(*lengths))
    out = []
    for i in range(extra):
        at = torch.tensor([n + i for n in lengths], device="cuda")
        pick = lambda t: t[torch.arange(B, device="cuda"), at]  # noqa: E731
        out.append(layer.step(pick(x), pick(r), slots)[0])
    return torch.stack(out, 1)


def mamba2_recurrence(layer, xBC, dt, h):
    """The recurrence of the layer's heads in 64 bits over tokens xBC (T, width), dt (T, H) from state h (H,P,N): outputs, the
    magnitudes of their terms, the state, and for the INT8 prompt path a bound of what its codes may be off by."""
    from linquant_b200.kernels.hadamard import kronecker_hadamard_fwd

    H, P, N, G, S = layer.H, layer.P, layer.N, layer.G, layer.scales
    x = xBC[:, :layer.d].double().view(-1, H, P)
    BC = kronecker_hadamard_fwd(xBC[None, :, layer.d:].unflatten(-1, (2 * G, N)).contiguous(), torch.cat([layer.signs, layer.signs]), 2 * G)[0].double()
    B, C = (t.repeat_interleave(H // G, 1) for t in (BC[:, :G], BC[:, G:]))  # (T,H,N)
    step = torch.nn.functional.softplus(dt.double() + layer.dt_bias.double())
    a = torch.exp(step * layer.A.double())
    alpha, sB, sS = S["alpha_hp"].double(), S["B_scale"].double().repeat_interleave(H // G), S["state_scale"].double()
    ys, mags, bound, bound_B = [], [], torch.zeros_like(h), torch.zeros_like(h)
    mag = h.abs()
    for t in range(x.shape[0]):
        w = step[t, :, None] * x[t]
        term = w[:, :, None] * B[t, :, None]
        h, mag = a[t, :, None, None] * h + term, a[t, :, None, None] * mag + term.abs()
        # a code of x dt is made at the chunk's end: its error does not decay within the chunk (not at all, to be short)
        bound = bound + 0.51 * alpha[:, :, None] * (B[t, :, None].abs() + sB[:, None, None])
        bound_B = a[t, :, None, None] * bound_B + 0.51 * w[:, :, None].abs() * sB[:, None, None]
        ys.append((h * C[t, :, None]).sum(-1) + layer.D.double()[:, None] * x[t])
        mags.append((mag * C[t, :, None].abs()).sum(-1) + (layer.D.double()[:, None] * x[t]).abs())
    return torch.stack(ys), torch.stack(mags), h, mag, bound + bound_B + sS[:, :, None]


@pytest.mark.parametrize("lengths", [(256, 256), (100, 301)])
def test_mamba2_layer(lengths):
    """The prompt's state is the recurrence's to within the codes of x, B and the chunk states; each token step from there is the
    recurrence itself.

    State: every code is at most half a step off (0.51 with the fp32 rounding), a token's part x dt decayed to the chunk's end is
    a code on alpha, B one on its scale; a chunk state is a code on the state scale (one step for the two chunks of the longest
    prompt, the earlier one decayed); the gate between chunks is a multiple of 2^-7, half of that off, on what it multiplies.
    Codes that saturate would add to this: calibration covers the tokens themselves. Step: the rounding of its fp16 output and
    300 fp32 roundings of its terms."""
    from linquant_b200.kernels.layer import short_conv_fwd
    from linquant_b200.models import Mamba2Layer
    from tests import layer_reference as ref

    B, extra, d = 2, 12, 512
    layer = Mamba2Layer(d, 16, slots=B, seed=1)
    x, r = inputs(B, max(lengths) + extra, d, torch.float16)
    slots, n = ints(1, 0), ints(*lengths)
    layer.calibrate(x[:, :max(lengths)], r[:, :max(lengths)], n)
    layer.prefill(x[:, :max(lengths)], r[:, :max(lengths)], slots, n)
    z, xBC, dt, _ = layer._in(x, r)
    conv, _ = short_conv_fwd(xBC, layer.conv, layer.conv_bias)
    start = layer.state[slots.long()].clone()
    for b in range(B):
        zero = torch.zeros(layer.H, layer.P, layer.N, device="cuda", dtype=torch.float64)
        _, _, h, mag, bound = mamba2_recurrence(layer, conv[b, :lengths[b]], dt[b, :lengths[b]], zero)
        assert ((start[b].double() - h).abs() <= bound + mag * 2.0**-8 + mag * 2.0**-16).all()
    got = []
    for i in range(extra):
        at = [torch.arange(B, device="cuda"), n.long() + i]
        got.append(layer._mix_step(xBC[at[0], at[1]], dt[at[0], at[1]], slots))
    got = torch.stack(got, 1)
    for b in range(B):
        s = slice(lengths[b], lengths[b] + extra)
        y, mag, h, hmag, _ = mamba2_recurrence(layer, conv[b, s], dt[b, s], start[b].double())
        ref.check(got[b], y.flatten(1), mag.flatten(1), 300 * 2.0**-24)
        ref.check(layer.state[slots[b]], h, hmag, extra * 64 * 2.0**-24)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_mamba_layer(dtype):
    """Prompt and token run the same arithmetic up to the order of fp32 sums: what differs is roundings of 16-bit values (and codes
    of them) that fall to the other side, one unit each."""
    from linquant_b200.models import MambaLayer

    B, extra, d, lengths = 3, 9, 256, (70, 1, 33)
    layer = MambaLayer(d, 640, slots=B, dtype=dtype, seed=2)
    x, r = inputs(B, max(lengths) + extra, d, dtype)
    got = drive(layer, x, r, lengths, extra)
    slots = ints(0, 1, 2)
    for b, n in enumerate(lengths):
        whole, _ = layer.prefill(x[b:b + 1, :n + extra], r[b:b + 1, :n + extra], slots[:1])
        assert rel_l2(got[b], whole[0, n:]) <= (2.0**-8 if dtype == torch.bfloat16 else 2.0**-11) * 4


def test_example_runs():
    import subprocess
    import sys

    from tests.conftest import ROOT

    for kind in ("mamba2", "mamba"):
        p = subprocess.run([sys.executable, "examples/serve_mamba.py", "--kind", kind, "--layers", "2", "--batch", "3", "--prompt", "300", "--tokens", "4"],
                           cwd=ROOT, capture_output=True, text=True, timeout=300)
        assert p.returncode == 0, p.stderr[-2000:]
        assert "us a step" in p.stdout
