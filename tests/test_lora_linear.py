"""INT8 product with low-rank adapters of many requests at once, against 64 bits."""

import ctypes

import pytest
import torch

from linquant_b200 import _cabi
from tests import layer_reference as ref
from tests.test_layer_host import filled

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
ULP = 2.0**-24
gpu = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seed():
    torch.manual_seed(13)


def randn(*shape, dtype=F32):
    return torch.randn(*shape, device="cuda").to(dtype)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def low_error(dtype, K, R, M):
    """Of the adapters' sum, relative to its terms' magnitudes. x a: one rounding (the tensor core cuts off, 2^-23) for each 16 of K and
    piece (six at most), 16 where the parts meet; t b the same over R. 16-bit outputs of more than 16 tokens take t and b as 16 bits
    each, and the sum is left in the output's type before the shared one joins it: half a step of that type, of a sum that is no
    larger than its terms' magnitudes together."""
    exact = (6 * (K / 16 + R / 16 + 2) + 32) * 2 * ULP
    return exact if dtype == F32 else exact + 2.0**-15 + (ref.UNIT[dtype] if M > 16 else 0)


def want_of(x, codes, x_scale, w, w_scale, a, b, which, scaling, bias):
    """y, the magnitude of its shared sum and of the adapters' sum. x: what the adapters see."""
    base = (codes.double() @ w.double().t()) * x_scale.double().unsqueeze(1) * w_scale.double()
    mag = base.abs()
    if bias is not None:
        base, mag = base + bias.double(), mag + bias.double().abs()
    low = torch.zeros_like(mag)
    x = x.double()
    for l in range(a.shape[0]):
        rows = (which == l).nonzero()[:, 0]
        if rows.numel():
            s = scaling if not torch.is_tensor(scaling) else float(scaling[l])
            base[rows] += s * (x[rows] @ a[l].double().t()) @ b[l].double().t()
            low[rows] = abs(s) * (x[rows].abs() @ a[l].double().abs().t()) @ b[l].double().abs().t()
    return base, mag, low


def agree(y, want, K, R):
    base, mag, low = want
    e = low_error(y.dtype, K, R, y.shape[0])
    ref.check(y, base, mag * (4 * ULP / e) + low, e)


def weights(N, K, R, L, dtype):
    from linquant_b200.kernels.layer import quantize_rows_fwd

    return *quantize_rows_fwd(randn(N, K) / K**0.5), (randn(L, R, K) / K**0.5).to(dtype), (randn(L, N, R) / R**0.5).to(dtype)


@gpu
@pytest.mark.parametrize("M,K,N,R,L,types,runs,out", [
    (1, 1, 1, 8, 1, (BF16, BF16), 1, None), (1, 64, 24, 8, 2, ("codes", BF16), 1, F32), (3, 5120, 260, 16, 8, (BF16, BF16), 1, None),
    (8, 300, 33, 24, 3, (F16, F16), 3, None), (8, 1000, 64, 16, 5, (F32, F32), 1, None), (13, 256, 100, 64, 20, ("codes", F16), 1, F16),
    (16, 640, 70, 128, 2, ("codes", F32), 5, None), (17, 128, 96, 16, 4, (BF16, F16), 1, None), (64, 520, 200, 40, 64, (F16, BF16), 1, None),
    (65, 101, 77, 16, 3, (F32, BF16), 4, F16), (200, 2560, 320, 16, 9, ("codes", BF16), 7, None), (40, 8192, 520, 32, 6, ("codes", F16), 1, F16),   # parts of K
    (129, 5120, 130, 8, 2, (BF16, BF16), 50, F32), (1000, 72, 1000, 128, 7, ("codes", BF16), 90, None), (700, 300, 2000, 16, 40, (F32, F32), 1, None),
    (2500, 64, 300, 64, 3, ("codes", F16), 800, F32), (20000, 48, 20, 24, 5, (BF16, BF16), 777, None), (10000, 40, 24, 16, 5, (F32, F32), 777, None),
    (4000, 128, 7700, 16, 6, ("codes", BF16), 333, None),  # pairs of CTAs
    (3900, 32, 7936, 8, 3, ("codes", F32), 64, F32), (0, 16, 8, 8, 2, (BF16, BF16), 1, None), (5, 32, 16, 5, 3, (BF16, BF16), 1, None),  # a rank that is padded
])
def test_product_with_adapters(M, K, N, R, L, types, runs, out):
    from linquant_b200.kernels.layer import int8_linear_fwd, lora_linear_fwd, quantize_rows_fwd

    form, ta = types
    w, ws, a, b = weights(N, K, R, L, ta)
    x = randn(M, K)
    x[..., :: 97] *= 20
    which = torch.randint(-1, L + 1, (max(1, -(-M // runs)),), device="cuda").repeat_interleave(runs)[:M].int()  # -1 and L: none
    scaling, bias = torch.rand(L, device="cuda") + 0.2, randn(N) if N % 2 == 0 else None
    if form == "codes":
        codes, xs = quantize_rows_fwd(x)
        args, seen = dict(x_scale=xs), codes.double() * xs.double().unsqueeze(1)
        given = codes
    else:
        given = x.to(form)
        codes, xs = quantize_rows_fwd(given)
        args, seen = {}, given.double()
    y = lora_linear_fwd(given, w, ws, a, b, which, scaling=scaling, bias=bias, out_dtype=out, **args)
    assert y.dtype == (out or (BF16 if form == "codes" else form)) and y.is_contiguous()
    agree(y, want_of(seen, codes, xs, w, ws, a, b, which, scaling, bias), K, R)
    plain = int8_linear_fwd(given, w, ws, bias=bias, out_dtype=out, **args)
    rows = (which < 0) | (which >= L)
    assert torch.equal(y[rows], plain[rows])  # rows without an adapter have the bits of the shared product
    assert torch.equal(y, lora_linear_fwd(given, w, ws, a, b, which, scaling=scaling, bias=bias, out_dtype=out, **args))


@gpu
@pytest.mark.parametrize("M", [5, 40, 300])
def test_what_is_not_a_rows_own_does_not_reach_it(M):
    """NaN in other requests' rows and adapters."""
    from linquant_b200.kernels.layer import lora_linear_fwd

    K, N, L = 96, 80, 4
    w, ws, a, b = weights(N, K, 16, L, BF16)
    x, which = randn(M, K, dtype=BF16), torch.randint(-1, 3, (M,), device="cuda").int()
    which[0], which[1] = 3, 1
    y = lora_linear_fwd(x, w, ws, a, b, which)
    x[0], a[3], b[3] = float("nan"), float("nan"), float("inf")
    z = lora_linear_fwd(x, w, ws, a, b, which)
    assert torch.isnan(z[0]).all() and torch.equal(y[1:], z[1:])


@gpu
def test_forms_of_arguments():
    """Leading axes, one scaling for all, adapters of 64 bits, views, several ranks stacked."""
    from linquant_b200.kernels.layer import int8_linear_fwd, lora_linear_fwd, stack_adapters

    K, N = 64, 48
    w, ws, _, _ = weights(N, K, 8, 1, BF16)
    pairs = [(randn(r, K, dtype=BF16), randn(N, r, dtype=BF16)) for r in (3, 16, 9)]
    a, b = stack_adapters(pairs)
    assert a.shape == (3, 16, K) and b.shape == (3, N, 16)
    x, which = randn(2, 6, K, dtype=BF16), torch.tensor([[0, 1, 2, 2**40, -2**40, 1], [2, 2, 2, 0, 0, 0]], device="cuda")
    y = lora_linear_fwd(x, w, ws, a, b, which, scaling=0.5)
    flat = lora_linear_fwd(x.view(12, K), w, ws, a, b, which.clamp(-1, 3).int().view(12), scaling=torch.full((3,), 0.5))
    assert y.shape == (2, 6, N) and torch.equal(y.view(12, N), flat)
    views = lora_linear_fwd(x, w, ws, a.transpose(1, 2).contiguous().transpose(1, 2), b.transpose(1, 2).contiguous().transpose(1, 2), which, scaling=0.5)
    assert torch.equal(y, views)
    assert torch.equal(lora_linear_fwd(x, w, ws, a[:0], b[:0], which), int8_linear_fwd(x, w, ws))  # nobody has an adapter yet
    one = lora_linear_fwd(x[0, 1], w, ws, a, b, torch.tensor(1, device="cuda"), scaling=0.5)
    assert one.shape == (N,)


@gpu
def test_captured_with_adapters_that_change():
    """A decode step's graph: the adapters of its rows are read when it is replayed."""
    from linquant_b200.kernels.layer import lora_linear_fwd

    w, ws, a, b = weights(64, 128, 16, 5, F16)
    x, which, s = randn(9, 128, dtype=F16), torch.zeros(9, device="cuda", dtype=torch.int32), torch.cuda.Stream()
    lora_linear_fwd(x, w, ws, a, b, which)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        y = lora_linear_fwd(x, w, ws, a, b, which)
    for _ in range(3):
        which.copy_(torch.randint(-1, 5, (9,), device="cuda"))
        x.copy_(randn(9, 128, dtype=F16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, lora_linear_fwd(x, w, ws, a, b, which))


# ------------------------------------------------------------------------------------------------------- without a GPU
def test_layout_matches_the_compiled_struct():
    L = _cabi.lib()
    L.lq_struct_bytes.restype = ctypes.c_ulonglong
    L.lq_struct_bytes.argtypes = [ctypes.c_int]
    assert L.lq_struct_bytes(9) == ctypes.sizeof(_cabi.LoraProblem)


@pytest.mark.parametrize("over,more,want", [({"M": 0}, {}, 0), ({}, {"R": 12}, 4), ({}, {"R": 136}, 4), ({}, {"R": 0}, 2), ({}, {"L": -1}, 2), ({}, {"dtype": 4}, 4),
                                            ({}, {"a": None}, 1), ({}, {"adapters": None}, 1), ({}, {"b": 4104}, 3), ({}, {"t": 4104}, 3), ({"K": 0}, {}, 2),
                                            ({"x": 4097}, {}, 3)])
def test_entry(over, more, want):
    p = filled(_cabi.LinearProblem, **{**dict(M=4, N=8, K=32, x_stride=32, w_stride=32, out_dtype=1), **over})
    q = filled(_cabi.LoraProblem, **{**dict(L=2, R=16, dtype=1, scale=1.0), **more})
    fn = _cabi.lib().lq_lora_linear
    fn.argtypes = [ctypes.POINTER(_cabi.LinearProblem), ctypes.POINTER(_cabi.LoraProblem), ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p]
    assert fn(ctypes.byref(p), ctypes.byref(q), None, 0, 0, None) == want


def test_cpu_tensors_are_refused():
    from linquant_b200.kernels import layer

    with pytest.raises(_cabi.LinQuantError):
        layer.lora_linear_fwd(torch.zeros(2, 16), torch.zeros(4, 16, dtype=torch.int8), torch.ones(4), torch.zeros(1, 8, 16), torch.zeros(1, 4, 8),
                              torch.zeros(2, dtype=torch.int32))
    with pytest.raises(AssertionError):
        layer.stack_adapters([(torch.zeros(4, 16), torch.zeros(8, 3))])


@gpu
@pytest.mark.parametrize("what,error", [("a", AssertionError), ("b", AssertionError), ("adapters", AssertionError), ("float", NotImplementedError), ("mixed", NotImplementedError),
                                        ("rank", NotImplementedError), ("scaling", AssertionError), ("codes", AssertionError), ("out", NotImplementedError)])
def test_refusals(what, error):
    from linquant_b200.kernels.layer import lora_linear_fwd

    w, ws, a, b = weights(24, 32, 136 if what == "rank" else 8, 2, F16)
    x, which = randn(3, 32, dtype=F16), ints(0, 1, 0)
    with pytest.raises(error):
        lora_linear_fwd(x.char() if what == "codes" else x, w, ws, a[..., :16] if what == "a" else a, b[:1] if what == "b" else b.float() if what == "mixed" else b,
                        which[:2] if what == "adapters" else which.float() if what == "float" else which, scaling=randn(3) if what == "scaling" else None,
                        out_dtype=torch.float64 if what == "out" else None)


@gpu
@pytest.mark.parametrize("M", [3, 11, 40, 300, 5000])
@pytest.mark.parametrize("form", ["codes", BF16])
def test_kernels_that_overlap(M, form):
    """The product starts while t and the adapters' share are being made: calls one behind the other, each on rows that the kernel ahead
    of it has just written, have the bits of calls that wait for the device in between."""
    from linquant_b200.kernels.layer import lora_linear_fwd, quantize_rows_fwd

    K, N, L, R = 640, 1000, 5, 24
    w, ws, a, b = weights(N, K, R, L, BF16)
    which = torch.randint(-1, L, (M,), device="cuda").int()
    source = [randn(M, K, dtype=BF16) for _ in range(4)]

    def call(i, x):
        x.copy_(source[i % 4])
        if form == "codes":
            codes, xs = quantize_rows_fwd(x)
            return lora_linear_fwd(codes, w, ws, a, b, which, scaling=0.5, x_scale=xs, out_dtype=BF16)
        return lora_linear_fwd(x, w, ws, a, b, which, scaling=0.5)

    want, x = [], torch.empty(M, K, device="cuda", dtype=BF16)
    for i in range(4):
        want.append(call(i, x))
        torch.cuda.synchronize()
    for round in range(6):
        got = [call(i, x) for i in range(8)]
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[i % 4]) for i, y in enumerate(got)), round


@gpu
def test_outputs_behind_32_bits():
    """2.1 million tokens, 2.2e9 outputs: rows at both ends and around the 65536th tile of 32."""
    from linquant_b200.kernels.layer import lora_linear_fwd, quantize_rows_fwd

    M, K, N, R, L = 2_100_003, 16, 1032, 8, 3
    w, ws, a, b = weights(N, K, R, L, BF16)
    x = randn(M, K, dtype=BF16)
    which = (torch.arange(M, device="cuda") // 1000 % 4).int()  # the fourth: none
    y = lora_linear_fwd(x, w, ws, a, b, which, scaling=0.5)
    rows = torch.cat([torch.arange(n, n + 40, device="cuda") for n in (0, 65535 * 32 - 20, M - 40)])
    codes, xs = quantize_rows_fwd(x[rows])
    base, mag, low = want_of(x[rows], codes, xs, w, ws, a, b, which[rows], 0.5, None)
    e = low_error(BF16, K, R, M)
    ref.check(y[rows], base, mag * (4 * ULP / e) + low, e)
