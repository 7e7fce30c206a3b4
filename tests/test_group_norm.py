"""Group norm with an activation, of single tokens and over the tokens of sequences, against 64 bits."""

import ctypes

import pytest
import torch

from linquant_b200 import _cabi
from tests import layer_reference as ref
from tests.test_layer_host import filled

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
ULP = 2.0**-24
INF = float("inf")
gpu = pytest.mark.gpu

# A mean is off by the roundings of its sum, of the values' magnitude: up to 30000 / 256 values a thread and the tree over threads,
# 140, or over tokens the chain of eights (at most 1024 tokens a thread here: 128 joins of three) and of rows and tiles, 450.
# The variance by as many, half of it in its root; scale, activation and gate by 64 (the exponentials at |x| up to 20).
NORM = 768 * ULP


@pytest.fixture(autouse=True)
def seed():
    torch.manual_seed(9)


def randn(*shape, dtype=F32):
    return torch.randn(*shape, device="cuda").to(dtype)


def want_of(x, groups, weight, bias, silu, gate, eps, n=None):
    """y and its magnitude of x (N, S, D): statistics over S and each group's channels; n: the rows of S that count."""
    x = x.double().cpu()
    N, S, D = x.shape
    y, mag = torch.zeros_like(x), torch.zeros_like(x)
    w = torch.ones(D, dtype=torch.float64) if weight is None else weight.double().cpu()
    b = torch.zeros(D, dtype=torch.float64) if bias is None else bias.double().cpu()
    for i in range(N):
        k = S if n is None else min(max(int(n[i]), 0), S)
        if k == 0:
            continue
        v = x[i, :k].view(k, groups, D // groups)
        mean, size = v.mean((0, 2), keepdim=True), v.abs().mean((0, 2), keepdim=True)
        inv = 1 / torch.sqrt(((v - mean) ** 2).mean((0, 2), keepdim=True) + eps)
        y[i, :k] = ((v - mean) * inv).reshape(k, D) * w + b
        mag[i, :k] = (((v - mean).abs() + size + v.abs()) * inv).reshape(k, D) * w.abs() + b.abs()
    if silu:
        y, mag = ref.silu(y), 1.1 * mag + y.abs()  # the slope is 1.1 at most
    if gate is not None:
        z = ref.silu(gate.double().cpu())
        y, mag = y * z, mag * z.abs()
    return y, mag


@gpu
@pytest.mark.parametrize("rows,D,groups,dtype,silu,gate,pad,affine", [
    (1, 1, 1, F32, False, False, 0, True), (3, 8, 8, F16, True, False, 0, True), (5, 64, 4, BF16, False, True, 0, True),
    (7, 2048, 16, BF16, True, True, 16, True), (33, 2048, 16, F16, False, True, 3, True),   # a gate off every boundary
    (4, 1026, 18, BF16, True, False, 0, True), (4, 255, 5, F16, False, True, 1, True), (2, 5120, 80, F32, False, False, 0, False),
    (3, 1024, 2, BF16, False, False, 0, True), (3, 4096, 1, F16, True, True, 8, True), (2, 30000, 1, BF16, False, False, 0, True),
    (2, 29999, 1, F32, True, True, 0, True), (70000, 24, 3, BF16, False, False, 0, True), (0, 16, 2, F32, True, False, 0, True),
    (9, 520, 1, F16, False, False, 2, True), (6, 300, 1, F32, True, True, 4, False),
])
def test_tokens(rows, D, groups, dtype, silu, gate, pad, affine):
    from linquant_b200.kernels.layer import group_norm_fwd

    x = (randn(rows, D) * 2 + randn(D)).to(dtype)
    w, b = (randn(D), randn(D)) if affine else (None, None)
    z = randn(rows, D + pad, dtype=dtype)[:, pad:] if gate else None
    y = group_norm_fwd(x, groups, w, b, activation="silu" if silu else None, gate=z)
    assert y.dtype == dtype and y.is_contiguous()
    want, mag = want_of(x.unsqueeze(1), groups, w, b, silu, None if z is None else z.unsqueeze(1), 1e-5)
    ref.check(y, want[:, 0], mag[:, 0], NORM)
    if rows > 1:  # rows of a wider buffer, leading axes
        wide = torch.zeros(rows, D + 8, device="cuda", dtype=dtype)
        wide[:, :D] = x
        y2 = group_norm_fwd(wide[:, :D].unsqueeze(0), groups, w, b, activation="silu" if silu else None, gate=None if z is None else z.unsqueeze(0))
        assert torch.equal(y, y2[0])


@gpu
@pytest.mark.parametrize("B,T,D,groups,dtype,silu,gate,pad,lengths", [
    (1, 1, 1, 1, F32, False, False, 0, None), (2, 1, 64, 8, BF16, True, False, 0, None), (2, 17, 1026, 18, F16, True, False, 0, (17, 0)),
    (3, 100, 57, 3, BF16, False, True, 2, (1, 99, 100)), (2, 1499, 512, 32, BF16, True, False, 0, (1499, 700)),
    (1, 5000, 72, 1, F32, False, False, 0, None), (2, 65, 2048, 1, F16, True, True, 8, (64, 999)), (2, 40, 4098, 2, BF16, False, False, 0, (40, -5)),
    (1, 33, 5000, 1, F32, True, False, 0, None), (1, 20, 6000, 250, F16, False, True, 0, None), (5, 300, 7, 7, F32, False, False, 1, None),
    (400, 3, 16, 2, BF16, False, False, 0, None), (0, 5, 16, 2, F32, True, False, 0, None), (2, 0, 16, 2, F32, True, False, 0, None),
])
def test_over_tokens(B, T, D, groups, dtype, silu, gate, pad, lengths):
    from linquant_b200.kernels.layer import group_norm_fwd

    x = (randn(B, T, D + pad) * 2 + randn(D + pad)).to(dtype)[..., pad:]
    w, b, z = randn(D), randn(D), randn(B, T, D, dtype=dtype) if gate else None
    n = None if lengths is None else torch.tensor(lengths, device="cuda", dtype=torch.int32)
    want, mag = want_of(x, groups, w, b, silu, z, 1e-5, n)
    if n is not None:
        for i in range(B):
            x[i, max(int(n[i]), 0):] = float("nan")
            if z is not None:
                z[i, max(int(n[i]), 0):] = INF
    y = group_norm_fwd(x, groups, w, b, activation="silu" if silu else None, gate=z, over_tokens=True, lengths=n)
    assert y.dtype == dtype and y.is_contiguous()
    ref.check(y, want, mag, NORM)
    for i in range(B):
        if n is not None:
            assert not y[i, max(int(n[i]), 0):].any()
    assert torch.equal(y, group_norm_fwd(x, groups, w, b, activation="silu" if silu else None, gate=z, over_tokens=True, lengths=n))


@gpu
@pytest.mark.parametrize("over", [False, True])
def test_far_means_and_small_variances(over):
    """Values whose mean is far from zero, groups without variance, a group with an infinity: only that group's values are NaN."""
    from linquant_b200.kernels.layer import group_norm_fwd

    x = randn(4, 96, 256) + 1000.0
    x[1, :, :64] = 3.0
    y = group_norm_fwd(x, 4, eps=1e-3, over_tokens=over)
    want, mag = want_of(x if over else x.flatten(0, 1).unsqueeze(1), 4, None, None, False, None, 1e-3)
    ref.check(y, want.reshape(y.shape), mag.reshape(y.shape), NORM)
    assert not y[1, :, :64].any()
    x[2, 5, 100] = INF
    bad = torch.isnan(group_norm_fwd(x, 4, over_tokens=over))
    expect = torch.zeros_like(bad)
    if over:
        expect[2, :, 64:128] = True
    else:
        expect[2, 5, 64:128] = True
    assert torch.equal(bad, expect)


@gpu
def test_forms_of_arguments():
    from linquant_b200.kernels.layer import group_norm_fwd

    x, w = randn(3, 10, 64, dtype=BF16), randn(64)
    y = group_norm_fwd(x, 4, w.half().double(), over_tokens=True, lengths=torch.tensor([10, 2**40, 5], device="cuda"))
    xt = x.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(y, group_norm_fwd(xt, 4, w.half().float(), over_tokens=True, lengths=torch.tensor([10, 10, 5], device="cuda", dtype=torch.int32)))
    t = group_norm_fwd(x[0, 0], 4, w)
    assert t.shape == (64,) and torch.equal(t, group_norm_fwd(x, 4, w)[0, 0])


@gpu
def test_two_graphs_at_once():
    from linquant_b200.kernels.layer import group_norm_fwd

    sets, outs, graphs, streams = [randn(2, 500, 96, dtype=F16) for _ in range(2)], [], [], [torch.cuda.Stream() for _ in range(2)]
    for s, x in zip(streams, sets):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            group_norm_fwd(x, 3, over_tokens=True)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            outs.append(group_norm_fwd(x, 3, over_tokens=True))
    for _ in range(3):
        for x in sets:
            x.copy_(randn(*x.shape, dtype=F16) + 1)
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(sets, outs):
            assert torch.equal(y, group_norm_fwd(x, 3, over_tokens=True))


# ------------------------------------------------------------------------------------------------------- without a GPU
def test_layout_matches_the_compiled_struct():
    L = _cabi.lib()
    L.lq_struct_bytes.restype = ctypes.c_ulonglong
    L.lq_struct_bytes.argtypes = [ctypes.c_int]
    assert L.lq_struct_bytes(8) == ctypes.sizeof(_cabi.GroupNormProblem)


@pytest.mark.parametrize("over,want", [({"B": 0}, 0), ({"D": 0}, 2), ({"groups": 3}, 2), ({"groups": 0}, 2), ({"dtype": 3}, 4), ({"x": None}, 1), ({"T": 2}, 2),
                                       ({}, 2), ({"over_tokens": 1}, 7), ({"over_tokens": 1, "B": 70000}, 2)])
def test_entry(over, want):
    p = filled(_cabi.GroupNormProblem, **{**dict(B=2, T=1, D=16, groups=4, dtype=1, x_stride_b=16, x_stride_t=16), **over})
    if over and not over.get("over_tokens"):
        p.lengths = None
    fn = _cabi.lib().lq_group_norm
    fn.argtypes = [ctypes.POINTER(type(p)), ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    assert fn(ctypes.byref(p), None, 0, None) == want


def test_cpu_tensors_are_refused():
    from linquant_b200.kernels import layer

    with pytest.raises(_cabi.LinQuantError):
        layer.group_norm_fwd(torch.zeros(2, 16), 4)
    with pytest.raises(NotImplementedError):
        layer.group_norm_fwd(torch.zeros(2, 16), 4, activation="relu")


@gpu
@pytest.mark.parametrize("what,error", [("groups", AssertionError), ("weight", AssertionError), ("gate", AssertionError), ("gate_type", NotImplementedError),
                                        ("dims", AssertionError), ("lengths", AssertionError), ("lengths_n", AssertionError), ("dtype", NotImplementedError)])
def test_refusals(what, error):
    from linquant_b200.kernels.layer import group_norm_fwd

    x = randn(2, 5, 16)
    with pytest.raises(error):
        group_norm_fwd(x[0] if what == "dims" else x.double() if what == "dtype" else x, 3 if what == "groups" else 4,
                       weight=randn(15) if what == "weight" else None, gate={"gate": x[:, :4], "gate_type": x.half()}.get(what),
                       over_tokens=what in ("dims", "lengths_n"),
                       lengths=torch.tensor([1, 2, 3] if what == "lengths_n" else [1, 2], device="cuda") if what.startswith("lengths") else None)


@gpu
def test_rows_behind_32_bits():
    """2.2e9 values: the last rows have what they have by themselves."""
    from linquant_b200.kernels.layer import group_norm_fwd

    x = torch.empty(2_100_003, 1032, device="cuda", dtype=torch.bfloat16).normal_()
    y = group_norm_fwd(x, 2)
    tail = x[-77:].clone()
    assert torch.equal(y[-77:], group_norm_fwd(tail, 2)) and torch.equal(y[:77], group_norm_fwd(x[:77].clone(), 2))
    del y
    z = group_norm_fwd(x.unsqueeze(0), 2, over_tokens=True, lengths=torch.tensor([130], device="cuda", dtype=torch.int32))
    # tiles of another length add in another order: fp32 roundings of the mean and variance, then a step of bf16 that may fall to the other side
    alone = group_norm_fwd(x[:130].clone().unsqueeze(0), 2, over_tokens=True)[0].float()
    assert ((z[0, :130].float() - alone).abs() <= alone.abs() * 2.0**-7 + 2.0**-16).all()
    assert not z[0, -1000:].any()
