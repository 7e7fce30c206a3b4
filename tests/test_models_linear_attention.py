"""Linear attention, norms of heads and adapted projections run together: prompts, their parts and single tokens."""

import pytest
import torch

from tests import layer_reference as ref
from tests.helpers import rel_l2

gpu = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
D, T, EXTRA = 256, 150, 7


def randn(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda", dtype=dtype)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def pairs(N, K, ranks, seed):
    return [(randn(r, K, seed=seed + i) / K**0.5, randn(N, r, seed=seed + i + 50) / r**0.5) for i, r in enumerate(ranks)]


def make(dtype=F16, kv=None, slots=4, heads=4, K=64, V=48):
    from linquant_b200.models import LinearAttentionLayer

    layer = LinearAttentionLayer(D, heads, K, V, kv_heads=kv, slots=slots, dtype=dtype, seed=5)
    return layer.adapt(pairs(*layer.in_proj.codes.shape, (8, 16), 100), pairs(*layer.out_proj.codes.shape, (4, 12), 200), scaling=0.5)


def batch(B, dtype, n=T + EXTRA):
    return randn(B, n, D, dtype=dtype, seed=1), randn(B, n, D, dtype=dtype, seed=2)


def projection(proj, x, dtype, which):
    """64 bits, then the operator's one or two roundings to its type; x: values that the shared part takes as codes."""
    from linquant_b200.kernels.layer import quantize_rows_fwd

    codes, scale = x if isinstance(x, tuple) else quantize_rows_fwd(x)
    seen = codes.double() * scale.double().unsqueeze(-1) if isinstance(x, tuple) else x.double()
    y = (codes.double() @ proj.codes.double().t()) * scale.double().unsqueeze(-1) * proj.scale.double()
    for l in range(proj.a.shape[0]):
        share = proj.scaling * (seen @ proj.a[l].double().t()) @ proj.b[l].double().t()
        y = y + torch.where((which == l).unsqueeze(-1), share, torch.zeros_like(share))
    return y.to(dtype)


def plain(layer, x, r, which):
    """The layer over whole prompts, one token after the other in 64 bits."""
    from linquant_b200.kernels.layer import rms_norm_fwd

    B, n = x.shape[:2]
    which = which.unsqueeze(1).expand(B, n)
    (codes, scale), _ = rms_norm_fwd(x, layer.norm, residual=r, quantize=True)  # an operator with tests of its own
    q, k, v, z, a, _ = projection(layer.in_proj, (codes, scale), layer.dtype, which).split(layer.parts, -1)
    q, k = (t.unflatten(-1, (layer.Hk, layer.K)).double().repeat_interleave(layer.H // layer.Hk, 2) for t in (q, k))
    v = v.unflatten(-1, (layer.H, layer.V)).double()
    decay = torch.exp(torch.nn.functional.logsigmoid(a.double() + layer.decay_bias.double()) / 16)
    S, o = torch.zeros(B, layer.H, layer.K, layer.V, device="cuda", dtype=torch.float64), []
    states = []
    for t in range(n):
        S = decay[:, t, :, None, None] * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        o.append((q[:, t, :, :, None] * S).sum(-2) * layer.K**-0.5)
        states.append(S)
    o = torch.stack(o, 1).to(layer.dtype).double()
    o = (o - o.mean(-1, keepdim=True)) / torch.sqrt(o.var(-1, unbiased=False, keepdim=True) + 1e-5)
    o = (o.flatten(2) * torch.nn.functional.silu(z.double())).to(layer.dtype)
    return projection(layer.out_proj, o, layer.dtype, which), torch.stack(states, 1)


# Two runs differ by roundings to 16 bits (of the projection's outputs, twice with adapters, of o and of the normed rows) that fall to
# the other side, at most a whole step each, 2 units: relative to a row of independent values as much. The codes of the normed rows, one
# of 127 steps of a row's largest value, flip where a 16-bit step crosses their half: a share of 127 times 2 units of them, by 1 / 127
# of the largest, which is below 4 times a row's norm a channel: squared below 127 2 unit (4 / 127)^2 = 0.25 unit.
def tolerance(dtype):
    u = ref.UNIT[dtype]
    return 4 * 2 * u + (0.25 * u) ** 0.5


@gpu
@pytest.mark.parametrize("dtype,kv", [(F16, None), (BF16, 2), (F16, 1)])
def test_prompts_then_tokens(dtype, kv):
    """Ragged prompts with an adapter each (one with none), a part of them continued, then tokens: the plain layer."""
    layer, B = make(dtype, kv), 4
    x, r = batch(B, dtype)
    lengths, which, slots = (T, 1, 97, 64), ints(1, 0, -1, 1), ints(2, 0, 3, 1)
    want, states = plain(layer, x, r, which)
    out, res = layer.prefill(x[:, :T], r[:, :T], slots, ints(*lengths), which)
    assert torch.equal(res, x[:, :T] + r[:, :T])
    tol = tolerance(dtype)
    for b, n in enumerate(lengths):
        assert rel_l2(out[b, :n], want[b, :n]) <= tol
        assert rel_l2(layer.state[slots[b]], states[b, n - 1]) <= tol
    for i in range(EXTRA):
        at = torch.tensor([n + i for n in lengths], device="cuda")
        rows = torch.arange(B, device="cuda")
        out, _ = layer.step(x[rows, at], r[rows, at], slots, which)
        for b in range(B):
            assert rel_l2(out[b], want[b, at[b]]) <= 2 * tol  # a single row, not the mean over many
    for b, n in enumerate(lengths):
        assert rel_l2(layer.state[slots[b]], states[b, n + EXTRA - 1]) <= tol


@gpu
def test_a_prompt_in_parts_and_idle_entries():
    """Parts of a prompt leave what the whole of it leaves; entries outside the cache leave the others' states as they are."""
    layer, B = make(), 3
    x, r = batch(B, F16)
    which, slots = ints(0, 1, 5), ints(3, 1, 0)
    whole, _ = layer.prefill(x, r, slots, None, which)
    state = layer.state.clone()
    layer.state.zero_()
    parts, at = [], 0
    for n in (64, 1, 30, x.shape[1] - 95):
        parts.append(layer.prefill(x[:, at:at + n], r[:, at:at + n], slots, None, which, resume=at > 0)[0])
        at += n
    # The projections' rows are not the same bits: the parts have 192, 3, 90 and 186 rows, whose fp32 sums are made in other orders, and
    # few rows round once where many round the adapters' share too. A step of k and v each moves the state by 4 units; one of a
    # decay's logit, below 4 in magnitude, its logarithm by 2 units 4 / 16, independent over at most 157 tokens: 0.5 units 157^0.5.
    assert rel_l2(torch.cat(parts, 1), whole) <= tolerance(F16) and rel_l2(layer.state, state) <= (4 + 0.5 * 157**0.5) * ref.UNIT[F16]
    before = layer.state.clone()
    layer.prefill(x, r, ints(-1, 4, 2), ints(5, 0, 9), which)
    assert torch.equal(layer.state[[0, 1, 3]], before[[0, 1, 3]]) and layer.state[2].any()
    before = layer.state.clone()
    layer.step(x[:, 0], r[:, 0], ints(-1, 7, 1), which)
    assert torch.equal(layer.state[[0, 2, 3]], before[[0, 2, 3]]) and not torch.equal(layer.state[1], before[1])


@gpu
def test_tokens_in_a_graph():
    """A captured step, replayed on other tokens, adapters and slots, is the step itself."""
    layer, B = make(), 3
    x, r = batch(B, F16)
    layer.prefill(x, r, ints(0, 1, 2))
    start = layer.state.clone()
    token, res, which, slots = x[:, 0].clone(), r[:, 0].clone(), ints(0, 0, 0), ints(0, 1, 2)
    layer.step(token, res, slots, which)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.step(token, res, slots, which)[0]
    for i, (w, s) in enumerate(((ints(1, -1, 0), ints(2, 0, 1)), (ints(0, 1, 1), ints(3, -1, 0)))):
        token.copy_(x[:, i + 1]), which.copy_(w), slots.copy_(s)
        layer.state.copy_(start)
        graph.replay()
        got, state = out.clone(), layer.state.clone()
        layer.state.copy_(start)
        assert torch.equal(got, layer.step(token, res, slots, which)[0]) and torch.equal(state, layer.state)


@gpu
def test_example_runs():
    import subprocess
    import sys

    from tests.conftest import ROOT

    p = subprocess.run([sys.executable, "examples/serve_mamba.py", "--kind", "attention", "--layers", "2", "--batch", "3", "--prompt", "300", "--tokens", "4"],
                       cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stderr[-2000:]
    assert "us a step" in p.stdout
