"""Linear attention with a decay for each head (prompts, single tokens) against the recurrence in 64 bits."""

import ctypes

import pytest
import torch

from linquant_b200 import _cabi
from tests import layer_reference as ref
from tests.test_layer_host import call, filled

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
ULP = 2.0**-24
gpu = pytest.mark.gpu

# A term of a state is off by 24 roundings of the chunk's sum (four steps of 16 tokens, three pieces, the tensor core cuts off
# below 2^-23), by its decay's exponential (2) and by the exponent's rounding (log-decays of 2 x 64 at most: 89): 128 ulps a chunk.
# An output has besides the rounding of the decayed products q.k to the type (half a step) and of the state to two pieces
# (2^-16 bf16, 2^-22 fp16, nothing for fp32); fp16 products below 2^-25 of a row's largest are lost: 2^-24 of the terms' sum.
CHUNK = 128 * ULP
OUT = {F32: 2**-22, BF16: 2.0**-8 + 2.0**-14, F16: 2.0**-11 + 2.0**-16}


@pytest.fixture(autouse=True)
def seed():
    torch.manual_seed(5)


def randn(*shape, dtype=F32):
    return torch.randn(*shape, device="cuda").to(dtype)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def recurrence(q, k, v, g, scale, initial, lengths):
    """o, the sum of its terms' magnitudes, the final state and its magnitudes; in 64 bits."""
    B, T, H, V = v.shape
    K, rep = q.shape[-1], H // q.shape[2]
    scale = K**-0.5 if scale is None else scale
    h = torch.zeros(B, H, K, V, device="cuda", dtype=torch.float64) if initial is None else initial.double()
    m, o, mag = h.abs(), torch.zeros(B, T, H, V, device="cuda", dtype=torch.float64), torch.zeros(B, T, H, V, device="cuda", dtype=torch.float64)
    a = torch.ones(B, T, H, device="cuda", dtype=torch.float64) if g is None else torch.exp(g.double()).expand(B, T, H)
    for t in range(T):
        on = torch.ones(B, device="cuda", dtype=torch.bool) if lengths is None else lengths > t
        qt, kt = (x[:, t].double().repeat_interleave(rep, 1) for x in (q, k))
        kv = torch.where(on[:, None, None, None], kt.unsqueeze(-1) * v[:, t].double().unsqueeze(-2), 0.0)
        qt = torch.where(on[:, None, None], qt, 0.0)
        at = torch.where(on[:, None], a[:, t], 1.0)[..., None, None]
        h, m = at * h + kv, at * m + kv.abs()
        o[:, t] = scale * torch.einsum("bhk,bhkv->bhv", qt, h)
        mag[:, t] = abs(scale) * torch.einsum("bhk,bhkv->bhv", qt.abs(), m)
    return o, mag, h, m


def inputs(B, T, Hk, H, K, V, dtype, pad=0, decay="token"):
    def rows(heads, width):
        x = randn(B, T, heads * width + pad, dtype=dtype)
        return x[..., pad:].unflatten(-1, (heads, width))

    q, k, v = rows(Hk, K), rows(Hk, K), rows(H, V)
    g = {"none": None, "head": -torch.rand(H, device="cuda") * 0.2, "token": -2 * torch.rand(B, T, H, device="cuda")**4}[decay]
    return q, k, v, g


def agree(o, state, want, dtype, T):
    wo, mag, h, m = want
    chunks = T // 64 + 2
    rel = OUT[dtype] + chunks * CHUNK
    # what the type does not hold (fp16: from 65520, halfway behind its largest value) is an infinity of its sign
    over = torch.isinf(o) & (wo.abs() + rel * mag >= torch.finfo(dtype).max) & (o.sign() == wo.sign())
    ref.check(torch.where(over, 0.0, o), torch.where(over, 0.0, wo), mag, rel)
    if state is not None:
        ref.check(state, h, m, chunks * CHUNK)


@gpu
@pytest.mark.parametrize("B,T,Hk,H,K,V,dtype,pad,decay,initial,lengths", [
    (1, 1, 1, 1, 1, 1, F32, 0, "token", False, None),
    (2, 3, 2, 2, 8, 8, BF16, 0, "token", True, (3, 0)),            # an empty sequence
    (1, 64, 1, 1, 64, 64, F16, 0, "none", False, None),
    (1, 65, 2, 2, 128, 128, BF16, 0, "token", False, None),
    (2, 63, 1, 2, 128, 64, F16, 8, "token", True, (63, 17)),        # shared heads, rows at a pitch
    (1, 130, 1, 4, 100, 77, BF16, 0, "head", True, None),
    (2, 129, 3, 3, 33, 130, F16, 1, "token", False, (128, 129)),    # nothing aligned
    (2, 100, 2, 2, 72, 100, F32, 3, "token", True, (99, 64)),
    (1, 70, 2, 4, 256, 96, BF16, 0, "token", True, None),
    (1, 70, 1, 1, 200, 33, F16, 2, "head", True, None),
    (1, 70, 1, 2, 256, 40, F32, 0, "token", True, None),
    (1, 70, 1, 2, 129, 7, F32, 1, "none", False, None),
    (3, 150, 2, 2, 64, 257, BF16, 0, "token", True, (150, -3, 999)),  # lengths outside 0..T
    (1, 1500, 1, 1, 128, 128, BF16, 0, "token", True, None),       # cut into segments
    (2, 1101, 1, 2, 128, 70, F16, 0, "head", True, (1101, 520)),
    (1, 1300, 1, 2, 60, 64, F32, 0, "token", False, (700,)),
    (2, 700, 1, 1, 256, 32, BF16, 0, "token", True, (513, 0)),
    (0, 5, 1, 1, 16, 16, BF16, 0, "token", True, None),
    (2, 0, 1, 1, 16, 16, BF16, 0, "token", True, None),
])
def test_prompts(B, T, Hk, H, K, V, dtype, pad, decay, initial, lengths):
    from linquant_b200.kernels.layer import linear_attention_fwd

    q, k, v, g = inputs(B, T, Hk, H, K, V, dtype, pad, decay)
    s0 = randn(B, H, K, V) if initial else None
    n = None if lengths is None else ints(*lengths)
    want = recurrence(q, k, v, g, None, s0, n)
    if n is not None:  # what lies behind a sequence takes no part
        for b in range(B):
            for x in (q, k, v) + ((g,) if g is not None and g.dim() == 3 else ()):
                x[b, max(int(n[b]), 0):] = float("nan")
    o, state = linear_attention_fwd(q, k, v, g, initial_state=s0, lengths=n, output_final_state=True)
    assert o.dtype == dtype and o.is_contiguous() and state.dtype == F32
    agree(o, state, want, dtype, T)
    for b in range(B):
        if n is not None:
            assert not o[b, max(int(n[b]), 0):].any()
    again, none = linear_attention_fwd(q, k, v, g, initial_state=s0, lengths=n)
    assert none is None and torch.equal(again, o)


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_decays_at_the_ends(dtype):
    """Steps of minus infinity forget everything before them, growing decays and a scale of one's own are taken, strong ones lose
    no precision behind them."""
    from linquant_b200.kernels.layer import linear_attention_fwd

    q, k, v, _ = inputs(1, 200, 1, 3, 64, 64, dtype)
    g = -0.1 * torch.rand(1, 200, 3, device="cuda")
    g[0, [5, 64, 127, 130], 0] = float("-inf")
    g[0, ::3, 1] = -90.0
    g[0, :, 2] = 0.05
    o, state = linear_attention_fwd(q, k, v, g, scale=-0.3, output_final_state=True)
    agree(o, state, recurrence(q, k, v, g, -0.3, None, None), dtype, 200)


@gpu
@pytest.mark.parametrize("qs,ks,vs,dtype", [(1e-3, 1e-3, 1e-3, F16), (60.0, 200.0, 1e-4, F16), (1e-4, 300.0, 100.0, F16), (3.0, 1e-6, 1e4, F16),
                                            (1e15, 1e-20, 1e10, BF16), (1e-18, 1e12, 1e8, F32)])
def test_ranges(qs, ks, vs, dtype):
    """Values far from 1: neither the decayed products nor the state leave the operands' type on their way."""
    from linquant_b200.kernels.layer import linear_attention_fwd

    q, k, v, g = inputs(1, 150, 2, 2, 64, 64, F32)
    q, k, v = (q * qs).to(dtype), (k * ks).to(dtype), (v * vs).to(dtype)
    k[:, 64:128] = 0  # a chunk without keys
    o, state = linear_attention_fwd(q, k, v, g, scale=1.0 if dtype != F16 else min(1.0, 100 / (qs * ks * vs)), output_final_state=True)
    agree(o, state, recurrence(q, k, v, g, 1.0 if dtype != F16 else min(1.0, 100 / (qs * ks * vs)), None, None), dtype, 150)


@gpu
def test_forms_of_arguments():
    """Log-decays in half precision, transposed operands, lengths of 64 bits: converted; a fp64 state as well."""
    from linquant_b200.kernels.layer import linear_attention_fwd

    q, k, v, g = inputs(2, 90, 2, 2, 32, 48, BF16)
    s0 = randn(2, 2, 32, 48)
    n = torch.tensor([90, 2**40], device="cuda")
    o, s = linear_attention_fwd(q, k, v, g.half(), initial_state=s0.double(), lengths=n, output_final_state=True)
    qt = q.transpose(2, 3).contiguous().transpose(2, 3)
    o2, s2 = linear_attention_fwd(qt, k.transpose(1, 2).contiguous().transpose(1, 2), v, g.half().float(), initial_state=s0, output_final_state=True)
    assert torch.equal(o, o2) and torch.equal(s, s2)


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_in_pieces_and_token_by_token(dtype):
    """Segments that hand their state on, and single tokens through a cache, agree with the recurrence."""
    from linquant_b200.kernels.layer import linear_attention_fwd, linear_attention_step

    q, k, v, g = inputs(2, 77, 2, 4, 64, 96, dtype)
    want = recurrence(q, k, v, g, None, None, None)
    st, parts = None, []
    for a, b in ((0, 1), (1, 40), (40, 77)):
        o, st = linear_attention_fwd(q[:, a:b], k[:, a:b], v[:, a:b], g[:, a:b], initial_state=st, output_final_state=True)
        parts.append(o)
    agree(torch.cat(parts, 1), st, want, dtype, 77)
    cache, slots = torch.zeros(5, 4, 64, 96, device="cuda"), ints(3, 1)
    o = torch.stack([linear_attention_step(cache, q[:, t], k[:, t], v[:, t], g[:, t], slots=slots) for t in range(77)], 1)
    agree(o, cache[slots.long()], want, dtype, 77)
    assert not cache[[0, 2, 4]].any()


# A step: the decay's expf (2), products and sums of the state (2) and of up to 256 channels (256 in sequence at most)
STEP = 300 * ULP


@gpu
@pytest.mark.parametrize("B,Hk,H,K,V,dtype,state,decay,pad", [
    (1, 1, 1, 1, 1, F32, F32, "token", 0), (3, 2, 4, 64, 64, BF16, F32, "token", 8), (5, 16, 16, 128, 128, F16, F32, "head", 0),
    (2, 1, 3, 100, 77, BF16, F32, "none", 1), (2, 1, 2, 256, 260, F32, BF16, "token", 0), (4, 1, 2, 33, 36, F16, F16, "token", 3),
    (300, 4, 8, 16, 8, BF16, BF16, "token", 0), (1, 2, 2, 17, 1000, F32, F16, "head", 0), (0, 1, 1, 8, 8, F16, F32, "token", 0),
])
def test_tokens(B, Hk, H, K, V, dtype, state, decay, pad):
    from linquant_b200.kernels.layer import linear_attention_step

    q, k, v, g = inputs(B, 1, Hk, H, K, V, dtype, pad, decay)
    q, k, v = q[:, 0], k[:, 0], v[:, 0]
    g = g[:, 0] if decay == "token" else g
    S = B + 3
    cache = randn(S, H, K, V, dtype=state)
    before = cache.clone()
    slots = torch.randperm(S, device="cuda")[:B].int()
    if B > 2:
        slots[1], slots[2] = -1, S  # idle entries
    live = (slots >= 0) & (slots < S)
    rows = slots[live].long()
    o = linear_attention_step(cache, q, k, v, g, slots=slots)
    gl = None if g is None else (g if g.dim() == 1 else g[live].unsqueeze(1))
    wo, mag, h, m = recurrence(q[live].unsqueeze(1), k[live].unsqueeze(1), v[live].unsqueeze(1), gl, None, before[rows].float(), None)
    ref.check(o[live], wo[:, 0], mag[:, 0], STEP)
    ref.check(cache[rows], h, m, 4 * ULP)
    assert not o[~live].any()
    rest = torch.ones(S, dtype=torch.bool, device="cuda")
    rest[rows] = False
    assert torch.equal(cache[rest], before[rest])
    if B and decay != "token":
        c2 = before[:B].clone()
        assert torch.equal(linear_attention_step(c2, q, k, v, g), linear_attention_step(before[:B].clone(), q, k, v, g, slots=torch.arange(B, device="cuda")))


@gpu
def test_the_int8_prefill_hands_its_state_on():
    """A prompt through the INT8 chunk op, its last tokens and the ones behind it here: the carry has the same layout."""
    from linquant_b200.kernels.layer import linear_attention_fwd
    from linquant_b200.kernels.zoo.simple_gla import chunk_simple_gla_int8
    from tests.helpers import OracleRun, rel_l2, zoo_inputs

    q, k, v, g, _ = zoo_inputs(1, 192, 2, 64, 128, decay="scalar", dtype=BF16, seed=3)
    orc = OracleRun(q[:, :128], k[:, :128], v[:, :128], g[:, :128], None, family="linear", decay="scalar", policy="kernel_pt")
    q, k, v, g = (t.cuda() for t in (q, k, v, g))
    first = tuple(t[:, :128].contiguous() for t in (q, k, v, g))
    _, carry = chunk_simple_gla_int8(*first, orc.scales("cuda"), eta=1.0, output_final_state=True)
    o, state = linear_attention_fwd(q[:, 128:], k[:, 128:], v[:, 128:], g[:, 128:], initial_state=carry, output_final_state=True)
    agree(o, state, recurrence(q[:, 128:], k[:, 128:], v[:, 128:], g[:, 128:], None, carry, None), BF16, 64)
    whole, _, last, _ = recurrence(q, k, v, g, None, None, None)
    # what INT8 codes leave of the state: steps of 1/127 of the largest value, of which half are off on average
    assert rel_l2(state, last) < 0.05 and rel_l2(o, whole[:, 128:]) < 0.05


@gpu
def test_captured_and_on_other_streams():
    """Two graphs with a workspace each, replayed at once on two streams, with inputs that change."""
    from linquant_b200.kernels.layer import linear_attention_fwd

    sets = [inputs(1, 1200, 1, 1, 64, 64, BF16) for _ in range(2)]
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for s, (q, k, v, g) in zip(streams, sets):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            linear_attention_fwd(q, k, v, g, output_final_state=True)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(linear_attention_fwd(q, k, v, g, output_final_state=True))
        graphs.append(graph)
    for round_ in range(3):
        for q, k, v, g in sets:
            v.copy_(randn(*v.shape, dtype=BF16))
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (q, k, v, g), (o, state) in zip(sets, outs):
            o2, state2 = linear_attention_fwd(q, k, v, g, output_final_state=True)
            assert torch.equal(o, o2) and torch.equal(state, state2)


# ------------------------------------------------------------------------------------------------------- without a GPU
def test_layout_matches_the_compiled_struct():
    L = _cabi.lib()
    L.lq_struct_bytes.restype = ctypes.c_ulonglong
    L.lq_struct_bytes.argtypes = [ctypes.c_int]
    assert L.lq_struct_bytes(7) == ctypes.sizeof(_cabi.AttentionProblem)


def fwd(p, ws=None, n=0):
    fn = _cabi.lib().lq_linear_attention_fwd
    fn.argtypes = [ctypes.POINTER(type(p)), ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    return fn(ctypes.byref(p), ws, n, None)


@pytest.mark.parametrize("over,want", [({"B": 0}, 0), ({"K": 257}, 4), ({"K": 0}, 2), ({"Hk": 3}, 2), ({"dtype": 3}, 4), ({"q": None}, 1), ({"T": -1}, 2),
                                       ({"T": 4096}, 7)])  # a long prompt of few heads without its workspace
def test_prompt_entry(over, want):
    p = filled(_cabi.AttentionProblem, **{**dict(B=1, T=3, H=4, Hk=2, K=64, V=64, dtype=1), **over})
    assert fwd(p) == want


@pytest.mark.parametrize("over,want", [({}, 0), ({"T": 2}, 2), ({"state_dtype": 5}, 4), ({"slots": None, "n_slots": -1}, 2), ({"B": 3, "slots": None, "n_slots": 2}, 2),
                                       ({"B": 1, "n_slots": 1, "state": None}, 1), ({"H": 70000, "Hk": 70000, "B": 1}, 2)])
def test_step_entry(over, want):
    p = filled(_cabi.AttentionProblem, **{**dict(B=0, T=1, H=4, Hk=2, K=64, V=64, dtype=1, state_dtype=2, n_slots=0), **over})
    assert call("lq_linear_attention_step", p) == want


def test_cpu_tensors_are_refused():
    from linquant_b200.kernels import layer

    x = torch.zeros(2, 3, 1, 16)
    with pytest.raises(_cabi.LinQuantError):
        layer.linear_attention_fwd(x, x, x)
    with pytest.raises(_cabi.LinQuantError):
        layer.linear_attention_step(torch.zeros(2, 1, 16, 16), x[:, 0], x[:, 0], x[:, 0])


@gpu
@pytest.mark.parametrize("what", ["k", "v", "heads", "g", "g_int", "initial", "lengths", "dtype", "wide", "state", "state_view", "slots"])
def test_refusals(what):
    from linquant_b200.kernels.layer import linear_attention_fwd, linear_attention_step

    q, k, v, g = inputs(2, 5, 2, 4, 16, 24, BF16)
    error = {"g_int": NotImplementedError, "dtype": NotImplementedError, "wide": NotImplementedError}.get(what, AssertionError)
    with pytest.raises(error):
        if what == "k":
            linear_attention_fwd(q, k[:, :4], v, g)
        elif what == "v":
            linear_attention_fwd(q, k, v[:1], g)
        elif what == "heads":
            linear_attention_fwd(q, k, v[:, :, :3], g[..., :3])
        elif what == "g":
            linear_attention_fwd(q, k, v, g[:, :, :2])
        elif what == "g_int":
            linear_attention_fwd(q, k, v, g.int())
        elif what == "initial":
            linear_attention_fwd(q, k, v, g, initial_state=randn(2, 4, 24, 16))
        elif what == "lengths":
            linear_attention_fwd(q, k, v, g, lengths=ints(1))
        elif what == "dtype":
            linear_attention_fwd(q, k.float(), v, g)
        elif what == "wide":
            x = randn(1, 2, 1, 257, dtype=BF16)
            linear_attention_fwd(x, x, x)
        elif what == "state":
            linear_attention_step(randn(2, 4, 24, 16), q[:, 0], k[:, 0], v[:, 0], g[:, 0])
        elif what == "state_view":
            linear_attention_step(randn(2, 4, 24, 16).transpose(2, 3), q[:, 0], k[:, 0], v[:, 0], g[:, 0])
        else:
            linear_attention_step(randn(1, 4, 16, 24), q[:, 0], k[:, 0], v[:, 0], g[:, 0])  # a row fewer than sequences


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("what", ["batch", "heads", "tokens", "all"])
def test_operands_that_repeat(dtype, what):
    """Broadcast operands, whose strides are zero."""
    from linquant_b200.kernels.layer import linear_attention_fwd, linear_attention_step

    B, T, H, K, V = 2, 90, 3, 64, 72
    one = {"batch": (1, T, H), "heads": (B, T, 1), "tokens": (B, 1, H), "all": (1, 1, 1)}[what]
    q, k, v = (randn(*one, n, dtype=dtype).expand(B, T, H, n) for n in (K, K, V))
    g = (-torch.rand(*one, device="cuda")).expand(B, T, H)
    o, state = linear_attention_fwd(q, k, v, g, output_final_state=True)
    agree(o, state, recurrence(q, k, v, g, None, None, None), dtype, T)
    cache = randn(B, H, K, V)
    want = recurrence(q[:, :1], k[:, :1], v[:, :1], g[:, :1], None, cache.clone(), None)
    o = linear_attention_step(cache, q[:, 0], k[:, 0], v[:, 0], g[:, 0])
    agree(o.unsqueeze(1), cache, want, dtype, 1)


@gpu
@pytest.mark.parametrize("K,dtype", [(64, BF16), (136, F16)])
def test_outputs_behind_32_bits(K, dtype):
    """2.3e9 outputs and values; the last sequence counts its first tokens only."""
    from linquant_b200.kernels.layer import linear_attention_fwd

    B, T, H, V = 2, 70000, 128, 128
    n = ints(65, 130)
    q, k = randn(B, T, 1, K, dtype=dtype), randn(B, T, 1, K, dtype=dtype)
    v = torch.empty(B, T, H, V, device="cuda", dtype=dtype)
    v[:, :130] = randn(B, 130, H, V, dtype=dtype)
    g = -torch.rand(H, device="cuda")
    o, state = linear_attention_fwd(q, k, v, g, lengths=n, output_final_state=True)
    agree(o[:, :130], state, recurrence(q[:, :130], k[:, :130], v[:, :130], g, None, None, n), dtype, 130)
    assert not o[:, 130:].any()


@gpu
def test_from_two_threads():
    """Calls whose kernels differ in shared memory and workspaces, each on a stream of its own: every one has its own result."""
    import threading

    from linquant_b200.kernels.layer import group_norm_fwd, linear_attention_fwd, lora_linear_fwd, quantize_rows_fwd

    def calls(dtype, K, T, M, R):
        q, k, v, g = inputs(1, T, 2, 2, K, 64, dtype)
        x = randn(M, 320, dtype=dtype)
        w, ws = quantize_rows_fwd(randn(96, 320))
        a, b, which = randn(3, R, 320, dtype=dtype), randn(3, 96, R, dtype=dtype), torch.randint(-1, 3, (M,), device="cuda").int()
        return lambda: (linear_attention_fwd(q, k, v, g)[0], lora_linear_fwd(x, w, ws, a, b, which), group_norm_fwd(x.unsqueeze(0), 5, over_tokens=True))

    jobs = [calls(F32, 100, 300, 90, 128), calls(BF16, 64, 1500, 3, 8), calls(F16, 200, 90, 700, 40)]
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    bad, start = [], threading.Barrier(len(jobs))

    def work(job, expected):
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait()
            for _ in range(200):
                got = job()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, expected)):
                    bad.append(expected[0].dtype)

    threads = [threading.Thread(target=work, args=z) for z in zip(jobs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert bad == []
