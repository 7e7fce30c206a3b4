"""Layer operators at the ends of what they take: long rows, empty batches, integers and shapes that do not fit."""

import pytest
import torch

from tests import layer_reference as ref

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
ULP = 2.0**-24
INF = float("inf")
gpu = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seed():
    torch.manual_seed(11)


def randn(*shape, dtype=F32):
    return torch.randn(*shape, device="cuda").to(dtype)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def int_codes(n, k):
    return torch.randint(-128, 128, (n, k), device="cuda", dtype=torch.int8)


# ------------------------------------------------------------------------------------- rows of more than 16384 channels
@gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,K,pad", [(5, 16385, 0), (700, 16392, 0), (4, 20000, 1), (3, 28672, 8), (2, 131071, 0)])
def test_codes_of_long_rows(rows, K, pad, dtype):
    from linquant_b200.kernels.layer import quantize_rows_fwd

    x = randn(rows, K + pad, dtype=dtype)[:, :K]
    x[0] = 0
    codes, scale = quantize_rows_fwd(x)
    ref.check_codes(codes, scale, x.double().cpu())
    x[1, 3], x[1, K - 1] = INF, float("nan")
    _, scale = quantize_rows_fwd(x)
    assert not torch.isfinite(scale[1]) and torch.isfinite(scale[2:]).all() and scale[0] == 0


@gpu
@pytest.mark.parametrize("K", [16385, 20000, 131071])
@pytest.mark.parametrize("M", [1, 7, 8, 9, 40])
def test_product_of_long_rows_from_values(M, K):
    """Whatever kernel makes the codes, the product is the one of codes that were made ahead."""
    from linquant_b200.kernels.layer import int8_linear_fwd, quantize_rows_fwd

    x, (w, sw) = randn(M, K, dtype=BF16), quantize_rows_fwd(randn(24, K))
    codes, scale = quantize_rows_fwd(x)
    y = int8_linear_fwd(x, w, sw, out_dtype=F32)
    assert torch.equal(y, int8_linear_fwd(codes, w, sw, x_scale=scale, out_dtype=F32))
    want = (codes.double() @ w.double().t()) * scale.double()[:, None] * sw.double()
    ref.check(y, want, want.abs(), 4 * ULP)


# --------------------------------------------------------------------------------------------- extents near 2^31 - 1
@pytest.mark.parametrize("entry,cls,axis", [
    ("lq_short_conv_fwd", "ConvProblem", "T"), ("lq_short_conv_fwd", "ConvProblem", "D"), ("lq_short_conv_step", "ConvProblem", "D"),
    ("lq_selective_scan_fwd", "ScanProblem", "T"), ("lq_selective_scan_fwd", "ScanProblem", "D"), ("lq_selective_scan_step", "ScanProblem", "D"),
    ("lq_int8_linear", "LinearProblem", "M"), ("lq_int8_linear", "LinearProblem", "N"), ("lq_rms_norm", "NormProblem", "D")])
def test_extents_that_tiles_would_overflow(entry, cls, axis):
    """The number of an axis' tiles, and what is requested behind them, has to fit an int: refused ahead of any launch."""
    import ctypes

    from linquant_b200 import _cabi

    p = getattr(_cabi, cls)()
    for name, t in p._fields_:
        if t is ctypes.c_void_p:
            setattr(p, name, 4096)
    values = dict(B=0, T=1, D=8, W=4, N=8, G=1, dtype=1, state_dtype=2, M=1, K=16, x_stride=16, w_stride=16, rows=0, group=8, out_dtype=1, codes_stride=16)
    for name in values.keys() & {n for n, _ in p._fields_}:
        setattr(p, name, values[name])
    setattr(p, axis, 2**31 - 1)
    if cls == "NormProblem":
        p.group = p.D
    fn = getattr(_cabi.lib(), entry)
    fn.argtypes = [ctypes.POINTER(type(p)), ctypes.c_void_p]
    assert fn(ctypes.byref(p), None) == 2


# ------------------------------------------------------------------------------------------------- integers of 64 bits
@gpu
def test_lengths_and_slots_that_int32_does_not_hold():
    """A length behind 2^31 is the whole prompt, one below 0 none of it; such slots are idle entries."""
    from linquant_b200.kernels.layer import selective_scan_step, short_conv_fwd, short_conv_step

    x, w = randn(3, 9, 32), randn(32, 4)
    y, state = short_conv_fwd(x, w, lengths=torch.tensor([2**31 + 5, 2**32 + 4, -2**32 + 4], device="cuda"), output_final_state=True)
    want, last = short_conv_fwd(x, w, lengths=ints(9, 9, 0), output_final_state=True)
    assert torch.equal(y, want) and torch.equal(state, last)
    slots = torch.tensor([2**32, -2**63, 2**31 + 1], device="cuda")
    line = randn(4, 3, 32)
    before = line.clone()
    assert not short_conv_step(x[:, 0], line, w, slots=slots).any() and torch.equal(line, before)
    h = randn(4, 32, 8)
    before = h.clone()
    B = randn(3, 1, 8)
    assert not selective_scan_step(h, x[:, 0], x[:, 0], -torch.rand(32, 8, device="cuda"), B, B, slots=slots).any() and torch.equal(h, before)


# ----------------------------------------------------------------------------------------------------- empty batches
@gpu
@pytest.mark.parametrize("heads", [False, True])
def test_steps_of_no_sequences_in_other_types(heads):
    """Slots of 64 bits are converted, also where there are none."""
    from linquant_b200.kernels.layer import selective_scan_step

    state = randn(3, 4, 8, 16) if heads else randn(3, 32, 16)
    before = state.clone()
    u = torch.empty(0, 4, 8, device="cuda") if heads else torch.empty(0, 32, device="cuda")
    dt = torch.empty(0, 4, device="cuda") if heads else u
    A = -torch.rand(4, device="cuda") if heads else -torch.rand(32, 16, device="cuda")
    none, slots = torch.empty(0, 1, 16, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda")
    y = selective_scan_step(state, u, dt, A, none, none, z=torch.empty_like(u), slots=slots)
    assert y.shape == u.shape and torch.equal(state, before)


@gpu
def test_a_gate_of_heads_in_another_order():
    """Channels of a token that are not contiguous are copied."""
    from linquant_b200.kernels.layer import selective_scan_step

    state, u, z = randn(2, 3, 4, 16), randn(2, 3, 4), randn(2, 4, 3).transpose(1, 2)
    dt, A, B = randn(2, 3), -torch.rand(3, device="cuda"), randn(2, 1, 16)
    s1, s2 = state.clone(), state.clone()
    assert torch.equal(selective_scan_step(s1, u, dt, A, B, B, z=z), selective_scan_step(s2, u, dt, A, B, B, z=z.contiguous())) and torch.equal(s1, s2)


# ---------------------------------------------------------------------------------------------- decay of fp32 inputs
@gpu
@pytest.mark.parametrize("form", ["channels", "heads of 4", "heads of 3"])
def test_decay_of_a_step_is_that_of_expf(form):
    """dt A is a multiple of 1/8, exact in fp32: what is left is the exponential (1 ulp, 2^-23 of it) and the product with the
    state (half of one)."""
    from linquant_b200.kernels.layer import selective_scan_step

    n, N = 64, 16
    A = -torch.randint(1, 600, (n, N) if form == "channels" else (n,), device="cuda") / 4.0
    lead = () if form == "channels" else (int(form[-1]),)
    state, u = torch.ones(1, n, *lead, N, device="cuda"), torch.zeros(1, n, *lead, device="cuda")
    B = randn(1, 1, N)
    selective_scan_step(state, u, torch.full((1, n), 0.5, device="cuda"), A, B, B, dt_softplus=False)
    want = torch.exp(0.5 * A.double()).view(n, *([1] * (state.dim() - 1 - A.dim())), *A.shape[1:])
    assert ((state[0].double() - want).abs() <= 3 * ULP * want).all()


# -------------------------------------------------------------------------------------------------------- single rows
@gpu
def test_scale_of_a_single_row():
    """A row of codes without leading axes has one scale."""
    from linquant_b200.kernels.layer import int8_linear_fwd, quantize_rows_fwd

    w, sw = int_codes(4, 32), torch.rand(4, device="cuda")
    codes, scale = quantize_rows_fwd(randn(32))
    want = int8_linear_fwd(codes.view(1, 32), w, sw, x_scale=scale.view(1), out_dtype=F32)[0]
    for s in (scale, scale.view(1)):
        assert torch.equal(int8_linear_fwd(codes, w, sw, x_scale=s, out_dtype=F32), want)
    for wrong in (torch.ones(5, device="cuda"), torch.ones(0, device="cuda")):
        with pytest.raises(AssertionError):
            int8_linear_fwd(codes, w, sw, x_scale=wrong)


# -------------------------------------------------------------------------------------------- many sequences or groups
@gpu
@pytest.mark.parametrize("b,T,d,G,N", [(70001, 2, 3, 1, 5), (1, 3, 70000, 70000, 4), (300, 2, 600, 300, 16)])
def test_scan_of_more_rows_than_a_grid_axis(b, T, d, G, N):
    """Sequences times groups beyond 65535, the extent of a grid's second and third axis."""
    from linquant_b200.kernels.layer import selective_scan_fwd

    u, dt, B, C = randn(b, T, d), torch.rand(b, T, d, device="cuda") + 0.1, randn(b, T, G, N), randn(b, T, G, N)
    A, h0 = -(torch.rand(d, N, device="cuda") + 0.5), randn(b, d, N)
    y, h = selective_scan_fwd(u, dt, A, B, C, dt_softplus=False, initial_state=h0, output_final_state=True)
    want, mag, end, hm = ref.scan(u, dt, A, B, C, None, None, None, False, (0, INF), h0, None)
    ref.check(y, want, mag, 32 * T * ULP)  # 32 roundings a token at most, as in the tests of the operators
    ref.check(h, end, hm, 32 * T * ULP)


# ------------------------------------------------------------------------------------------ idle entries of a prompt
@gpu
@pytest.mark.parametrize("kind", ["mamba2", "mamba"])
def test_idle_entries_of_a_prompt_batch(kind):
    """A slot outside the cache, which a token step passes over, leaves nothing in a prompt either."""
    from linquant_b200.models import Mamba2Layer, MambaLayer

    layer = Mamba2Layer(256, 8, slots=4) if kind == "mamba2" else MambaLayer(256, 512, slots=4)
    x = randn(4, 70, 256, dtype=layer.dtype)
    r = torch.zeros_like(x)
    if kind == "mamba2":
        layer.calibrate(x, r)
    layer.prefill(x[2:3], r[2:3], ints(1))
    want, line = layer.state[1].clone(), layer.conv_state[1].clone()
    for t in (layer.state, layer.conv_state):
        t.fill_(7)
    layer.prefill(x, r, ints(-1, 4, 1, -9))
    assert torch.equal(layer.state[1], want) and torch.equal(layer.conv_state[1], line)
    for t in (layer.state, layer.conv_state):
        assert (t[[0, 2, 3]] == 7).all()
