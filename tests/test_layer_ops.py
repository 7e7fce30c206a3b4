"""Layer operators (short convolution, selective scan, INT8 product, norms) against plain forms in 64 bits."""

import pytest
import torch

from tests import layer_reference as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
ULP = 2.0**-24
INF = float("inf")


@pytest.fixture(autouse=True)
def seed():
    torch.manual_seed(7)


def randn(*shape, dtype=F32):
    return torch.randn(*shape, device="cuda").to(dtype)


def wide(*shape, dtype, pad=0, offset=0):
    """The first columns (from ``offset``) of a wider buffer; pad = 0: dense."""
    if not pad and not offset:
        return randn(*shape, dtype=dtype)
    return randn(*shape[:-1], shape[-1] + pad + offset, dtype=dtype)[..., offset:offset + shape[-1]]


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------ short convolution
# W + 1 roundings of the sum; SiLU's exponential at |x| up to 20 (2 + 1.2 |x| ulps), its quotient and product: 64 in all
CONV = 64 * ULP


@pytest.mark.parametrize("B,T,D,W,dtype,pad,offset,act,initial,lengths", [
    (1, 1, 1, 2, F32, 0, 0, True, False, None),
    (1, 1, 8, 4, BF16, 0, 0, True, True, None),           # shorter than the taps
    (2, 2, 64, 4, F16, 0, 0, False, True, (2, 1)),
    (3, 33, 136, 4, BF16, 24, 0, True, False, (33, 0, 7)),  # an empty sequence
    (2, 65, 101, 3, F16, 5, 0, True, True, (64, 65)),     # nothing aligned
    (2, 40, 64, 2, BF16, 64, 3, True, True, (99, -4)),    # lengths outside 0..T; x off a 16-byte boundary
    (1, 301, 1000, 4, F32, 0, 0, True, True, None),
    (4, 257, 264, 3, BF16, 0, 0, False, False, (257, 256, 8, 1)),
    (2, 700, 4096, 4, BF16, 0, 0, True, True, (700, 333)),  # long runs
    (0, 5, 8, 4, F16, 0, 0, True, False, None),
    (2, 0, 8, 4, F16, 0, 0, True, True, None),
])
def test_short_conv(B, T, D, W, dtype, pad, offset, act, initial, lengths):
    from linquant_b200.kernels.layer import short_conv_fwd

    x, w = wide(B, T, D, dtype=dtype, pad=pad, offset=offset), randn(D, W) * 0.5
    bias = randn(D) if D % 3 else None
    st = randn(B, W - 1, D, dtype=dtype) if initial else None
    n = None if lengths is None else ints(*lengths)
    if n is not None:  # what lies behind a sequence takes no part
        for b in range(B):
            x[b, max(int(n[b]), 0):] = float("nan")
    y, fs = short_conv_fwd(x, w, bias, "silu" if act else None, initial_state=st, lengths=n, output_final_state=True)
    want, mag, state = ref.conv(torch.nan_to_num(x), w, bias, st, n, act)
    assert y.dtype == dtype and y.is_contiguous()
    ref.check(y, want, mag, CONV)
    assert torch.equal(fs.double().cpu(), state)
    assert short_conv_fwd(x, w, bias, "silu" if act else None, initial_state=st, lengths=n)[1] is None


def test_short_conv_in_pieces_and_token_by_token():
    """Segments that hand their state on, and single tokens through a cache, give the bits of the whole call."""
    from linquant_b200.kernels.layer import short_conv_fwd, short_conv_step

    B, T, D = 2, 77, 520
    x, w, bias = randn(B, T, D, dtype=BF16), randn(D, 4), randn(D)
    y, fs = short_conv_fwd(x, w, bias, output_final_state=True)
    st, parts = None, []
    for a, b in ((0, 1), (1, 3), (3, 40), (40, 77)):
        o, st = short_conv_fwd(x[:, a:b], w, bias, initial_state=st, output_final_state=True)
        parts.append(o)
    assert torch.equal(torch.cat(parts, 1), y) and torch.equal(st, fs)
    cache = randn(5, 3, D, dtype=BF16)
    cache[[4, 1]] = 0
    keep, slots = cache.clone(), ints(4, 1)
    steps = torch.stack([short_conv_step(x[:, t], cache, w, bias, slots=slots) for t in range(T)], 1)
    assert torch.equal(steps, y) and torch.equal(cache[[4, 1]], fs)
    assert torch.equal(cache[[0, 2, 3]], keep[[0, 2, 3]])


@pytest.mark.parametrize("D,W,dtype,pad", [(64, 4, BF16, 0), (101, 3, F16, 4), (8, 2, F32, 8)])
def test_short_conv_step(D, W, dtype, pad):
    from linquant_b200.kernels.layer import short_conv_step

    B, S = 5, 7
    x, w, bias = wide(B, D, dtype=dtype, pad=pad), randn(D, W), randn(D)
    cache = randn(S, W - 1, D, dtype=dtype)
    before, slots = cache.clone(), ints(6, -1, 0, S, 2)  # two idle entries
    y = short_conv_step(x, cache, w, bias, slots=slots)
    live = [0, 2, 4]
    rows = slots[live].long()
    want, mag, state = ref.conv(x[live].unsqueeze(1), w, bias, before[rows], None, True)
    ref.check(y[live], want[:, 0], mag[:, 0], CONV)
    assert torch.equal(cache[rows].double().cpu(), state)
    assert not y[[1, 3]].any() and torch.equal(cache[[1, 3, 4, 5]], before[[1, 3, 4, 5]])


# ---------------------------------------------------------------------------------------------------- selective scan
# Steps dt >= 0.01 with rates |A| >= 0.7 forget in 1 / (1 - exp(-0.007)) = 143 tokens at most. A token's decay is off by
# 2 ulps of its exponential and 1 + |dt A log2 e| roundings of the exponent (|dt A| <= 16 where the decay is not zero), its
# input by six: 32 roundings a token at most
SCAN = 32 * 143 * ULP


def scan_inputs(b, T, d, G, N, dtype, pad=0):
    u = wide(b, T, d, dtype=dtype, pad=pad)
    dt = (wide(b, T, d, dtype=dtype, pad=pad).float().clamp(-2, 2) * 0.5).to(dtype)
    if pad:
        dt = torch.cat([dt, dt[..., :pad]], -1)[..., :d]
    bias = torch.rand(d, device="cuda") * 3 - 3.4  # dt raw > -4.5: softplus > 0.011
    A = -(torch.rand(d, N, device="cuda") * 15.3 + 0.7)
    return u, dt, A, wide(b, T, G, N, dtype=dtype, pad=pad), wide(b, T, G, N, dtype=dtype, pad=pad), bias


@pytest.mark.parametrize("b,T,d,G,N,dtype,pad,gate,initial,lengths", [
    (1, 1, 1, 1, 1, F32, 0, True, False, None),
    (1, 5, 3, 3, 2, F32, 3, False, True, None),
    (2, 33, 64, 1, 16, BF16, 0, True, True, (33, 0)),     # an empty sequence
    (3, 70, 130, 2, 13, F16, 7, True, True, (1, 32, 70)),
    (2, 64, 40, 1, 4, BF16, 0, False, False, (64, 63)),
    (1, 100, 66, 2, 7, F32, 0, True, True, (500,)),
    (1, 40, 50, 1, 31, F16, 0, True, True, None),
    (2, 37, 20, 4, 64, BF16, 1, True, True, (37, 16)),
    (1, 50, 9, 1, 100, F32, 0, True, True, None),
    (1, 35, 10, 2, 200, F32, 0, True, True, (33,)),
    (1, 40, 7, 1, 256, BF16, 0, True, False, None),
    (1, 300, 2050, 1, 16, BF16, 0, True, True, None),
    (9, 65, 4800, 3, 16, F16, 0, True, True, tuple(range(9, 72, 7))),
    (0, 4, 8, 1, 16, F32, 0, True, True, None),
    (2, 0, 8, 1, 16, F32, 0, True, True, None),
])
def test_selective_scan(b, T, d, G, N, dtype, pad, gate, initial, lengths):
    from linquant_b200.kernels.layer import selective_scan_fwd

    u, dt, A, B, C, bias = scan_inputs(b, T, d, G, N, dtype, pad)
    D, z = randn(d), wide(b, T, d, dtype=dtype, pad=pad) if gate else None
    h0 = randn(b, d, N) if initial else None
    n = None if lengths is None else ints(*lengths)
    want, mag, h, hm = ref.scan(u, dt, A, B, C, D, z, bias, True, (0, INF), h0, n)
    if n is not None:
        for i in range(b):
            for t in (u, dt, B, C) + ((z,) if gate else ()):
                t[i, int(n[i]):] = float("nan")
    y, fs = selective_scan_fwd(u, dt, A, B, C, D=D, z=z, dt_bias=bias, initial_state=h0, lengths=n, output_final_state=True)
    assert y.dtype == dtype and y.is_contiguous() and fs.dtype == F32
    ref.check(y, want, mag, SCAN)
    ref.check(fs, h, hm, SCAN)


def test_selective_scan_options():
    """No softplus, a step limit, no D, z, bias; parameters in half precision and double are converted."""
    from linquant_b200.kernels.layer import selective_scan_fwd

    u, dt, A, B, C, _ = scan_inputs(2, 45, 24, 1, 16, F32)
    dt = dt.abs() + 0.02
    y, fs = selective_scan_fwd(u, dt, A.double(), B, C, dt_softplus=False, dt_limit=(0.05, 0.4))
    want, mag, _, _ = ref.scan(u, dt, A, B, C, None, None, None, False, (0.05, 0.4), None, None)
    assert fs is None
    ref.check(y, want, mag, SCAN)
    # channels that are not contiguous: a copy
    y2, _ = selective_scan_fwd(u.transpose(1, 2).contiguous().transpose(1, 2), dt, A, B, C, dt_softplus=False, dt_limit=(0.05, 0.4))
    assert torch.equal(y, y2)


def test_selective_scan_in_pieces_and_token_by_token():
    """Segments that hand their fp32 state on, and single tokens through a cache, agree with the whole call."""
    from linquant_b200.kernels.layer import selective_scan_fwd, selective_scan_step

    b, T, d, N = 2, 75, 136, 16
    u, dt, A, B, C, bias = scan_inputs(b, T, d, 2, N, F32)
    D, z = randn(d), randn(b, T, d)
    kw = dict(D=D, dt_bias=bias)
    y, fs = selective_scan_fwd(u, dt, A, B, C, z=z, output_final_state=True, **kw)
    st, parts = None, []
    for i, j in ((0, 1), (1, 33), (33, 75)):
        o, st = selective_scan_fwd(u[:, i:j], dt[:, i:j], A, B[:, i:j], C[:, i:j], z=z[:, i:j], initial_state=st, output_final_state=True, **kw)
        parts.append(o)
    mag = ref.scan(u, dt, A, B, C, D, z, bias, True, (0, INF), None, None)[1]
    ref.check(torch.cat(parts, 1), y, mag, 2 * SCAN)
    cache, slots = torch.zeros(4, d, N, device="cuda"), ints(3, 0)
    steps = torch.stack([selective_scan_step(cache, u[:, t], dt[:, t], A, B[:, t], C[:, t], z=z[:, t], slots=slots, **kw) for t in range(T)], 1)
    ref.check(steps, y, mag, 2 * SCAN)
    assert not cache[[1, 2]].any()


@pytest.mark.parametrize("d,N,G,dtype,sdtype,pad", [(64, 16, 1, BF16, F32, 0), (101, 13, 1, F16, F32, 3), (6, 256, 2, F32, F32, 0),
                                                    (130, 16, 2, BF16, BF16, 0), (24, 8, 3, F16, F16, 0), (7, 1, 1, BF16, F16, 1)])
def test_selective_scan_step(d, N, G, dtype, sdtype, pad):
    from linquant_b200.kernels.layer import selective_scan_step

    b, S = 5, 7
    u, dt, A, B, C, bias = (t[:, 0] if t.dim() > 2 else t for t in scan_inputs(b, 1, d, G, N, dtype, pad))
    D, z, state = randn(d), wide(b, d, dtype=dtype, pad=pad), randn(S, d, N, dtype=sdtype)
    before, slots = state.clone(), ints(6, -3, 0, S, 2)
    y = selective_scan_step(state, u, dt, A, B, C, D=D, z=z, dt_bias=bias, slots=slots)
    live = [0, 2, 4]
    rows = slots[live].long()
    want, mag, h, hm = ref.scan_step(before[rows], u[live], dt[live], A, B[live], C[live], D, z[live], bias, True, (0, INF))
    ref.check(y[live], want, mag, 300 * ULP)  # one token: N terms and the 32 roundings of a decay
    ref.check(state[rows], h, hm, 64 * ULP)
    assert not y[[1, 3]].any() and torch.equal(state[[1, 3, 4, 5]], before[[1, 3, 4, 5]])


@pytest.mark.parametrize("H,P,N,G,dtype,sdtype,skip", [(80, 64, 128, 1, BF16, F32, "H"), (6, 32, 64, 2, F16, F32, "HP"), (3, 5, 17, 1, F32, F32, "H"),
                                                       (4, 64, 128, 4, BF16, BF16, None), (2, 128, 256, 1, F32, F16, "HP"), (5, 1, 16, 5, BF16, F32, "H")])
def test_selective_scan_step_of_heads(H, P, N, G, dtype, sdtype, skip):
    from linquant_b200.kernels.layer import selective_scan_step

    b, S = 4, 6
    u = wide(b, H * P, dtype=dtype, pad=16).unflatten(1, (H, P))
    z = randn(b, H, P, dtype=dtype)
    dt, bias, A = randn(b, H, dtype=dtype), randn(H) - 2, -(torch.rand(H, device="cuda") * 15 + 0.5)
    B, C, state = randn(b, G, N, dtype=dtype), randn(b, G, N, dtype=dtype), randn(S, H, P, N, dtype=sdtype)
    D = None if skip is None else randn(H) if skip == "H" else randn(H, P)
    before, slots = state.clone(), ints(5, 1, 77, 0)
    y = selective_scan_step(state, u, dt, A, B, C, D=D, z=z, dt_bias=bias, slots=slots)
    live, rows = [0, 1, 3], [5, 1, 0]
    want, mag, h, hm = ref.scan_step(before[rows], u[live], dt[live], A, B[live], C[live], D, z[live], bias, True, (0, INF))
    ref.check(y[live], want, mag, 300 * ULP)
    ref.check(state[rows], h, hm, 64 * ULP)
    assert not y[2].any() and torch.equal(state[2:5], before[2:5])
    with_rows = before.clone()
    y2 = selective_scan_step(with_rows[:b].contiguous(), u, dt, A, B, C, D=D, z=z, dt_bias=bias)
    want, mag, _, _ = ref.scan_step(before[:b], u, dt, A, B, C, D, z, bias, True, (0, INF))
    ref.check(y2, want, mag, 300 * ULP)


def test_offsets_that_pass_32_bits():
    """Caches of more than 2^32 elements: the last slots are reached, the ones that a truncated offset would hit are not."""
    from linquant_b200.kernels.layer import selective_scan_step, short_conv_step

    d, N = 4096, 256
    S = 2**32 // (d * N) + 2
    state = torch.zeros(S, d, N, dtype=BF16, device="cuda")
    last = randn(d, N, dtype=BF16)
    state[S - 1] = last
    u, dt, A, B, C, bias = (t[:, 0] if t.dim() > 2 else t for t in scan_inputs(1, 1, d, 1, N, F32))
    y = selective_scan_step(state, u, dt, A, B, C, dt_bias=bias, slots=ints(S - 1))
    want, mag, h, hm = ref.scan_step(last.unsqueeze(0), u, dt, A, B, C, None, None, bias, True, (0, INF))
    ref.check(y, want, mag, 600 * ULP)
    ref.check(state[S - 1:], h, hm, 64 * ULP)
    assert not state[:2].any()
    conv = state.view(-1)[:(state.numel() // (3 * d)) * 3 * d].view(-1, 3, d)
    conv[-1] = randn(3, d, dtype=BF16)
    before, x, w = conv[-1:].clone(), randn(1, d, dtype=BF16), randn(d, 4)
    y = short_conv_step(x, conv, w, slots=ints(conv.shape[0] - 1))
    want, mag, st = ref.conv(x.unsqueeze(1), w, None, before, None, True)
    ref.check(y, want[:, 0], mag[:, 0], CONV)
    assert torch.equal(conv[-1:].double().cpu(), st) and not conv[:8].any()


# ------------------------------------------------------------------------------------------------------ INT8 product
def int_codes(n, k, low=-127):
    return torch.randint(low, 128, (n, k), device="cuda", dtype=torch.int8)


def padded(t):
    buf = torch.full((t.shape[0], (t.shape[1] + 15) // 16 * 16), 99, device="cuda", dtype=torch.int8)  # what lies behind a row is not used
    buf[:, :t.shape[1]] = t
    return buf[:, :t.shape[1]]


@pytest.mark.parametrize("M", [1, 3, 8, 9, 16, 17, 32, 33, 64, 65, 128, 129, 200, 257, 600])
@pytest.mark.parametrize("K,N", [(1, 1), (15, 17), (16, 16), (64, 40), (65, 130), (1000, 257), (2560, 513), (5120, 2560)])
def test_int8_linear_is_exact(M, K, N):
    """Unit scales and fp32 outputs: the INT32 sums themselves, where they fit 24 bits."""
    from linquant_b200.kernels.layer import int8_linear_fwd

    x, w = int_codes(M, K, -128), int_codes(N, K, -128)
    y = int8_linear_fwd(padded(x), padded(w), torch.ones(N, device="cuda"), x_scale=torch.ones(M, device="cuda"), out_dtype=F32)
    want = x.double() @ w.double().t()
    assert torch.equal(y.double(), want.float().double()) and y.is_contiguous()


@pytest.mark.parametrize("M", [2, 40, 300])
@pytest.mark.parametrize("sign", [1, -1])
def test_int8_linear_longest_sums(M, sign):
    from linquant_b200.kernels.layer import int8_linear_fwd

    K, N = 131071, 20
    x, w = torch.full((M, K), -128, device="cuda", dtype=torch.int8), torch.full((N, K), -128 if sign > 0 else 127, device="cuda", dtype=torch.int8)
    y = int8_linear_fwd(x, w, torch.ones(N, device="cuda"), x_scale=torch.ones(M, device="cuda"), out_dtype=F32)
    assert (y == float(torch.tensor(K * -128 * (-128 if sign > 0 else 127), dtype=torch.float64).float())).all()


@pytest.mark.parametrize("out", [F16, BF16, F32])
@pytest.mark.parametrize("M,K,N,bias", [(3, 200, 100, True), (50, 333, 77, True), (200, 512, 392, False), (1030, 192, 1001, True)])
def test_int8_linear_scales(M, K, N, bias, out):
    from linquant_b200.kernels.layer import int8_linear_fwd

    x, w = int_codes(M, K), int_codes(N, K)
    sx, sw = torch.rand(M, device="cuda") * 0.01, torch.rand(N, device="cuda") * 0.01
    sx[0] = 0
    b = randn(N) if bias else None
    y = int8_linear_fwd(x, w, sw, x_scale=sx, bias=b, out_dtype=out)  # rows off 16 bytes: copied
    want = (x.double() @ w.double().t()) * sx.double()[:, None] * sw.double()
    mag = want.abs() + (0 if b is None else b.double().abs())
    ref.check(y, want + (0 if b is None else b.double()), mag, 4 * ULP)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("lead,K,pad", [((1,), 5, 0), ((3,), 64, 0), ((2, 7), 1001, 3), ((129,), 2560, 16), ((4,), 16384, 0), ((0,), 32, 0)])
def test_quantize_rows(lead, K, pad, dtype):
    from linquant_b200.kernels.layer import int8_linear_fwd, quantize_rows_fwd

    x = wide(*lead, K, dtype=dtype, pad=pad)
    x[:1] = 0
    codes, scale = quantize_rows_fwd(x)
    assert codes.shape == x.shape and codes.dtype == torch.int8 and scale.shape == x.shape[:-1]
    if x.numel():
        ref.check_codes(codes, scale, x.double().cpu())
    w = padded(int_codes(24, K))
    one = torch.ones(24, device="cuda")
    y = int8_linear_fwd(x, w, one, out_dtype=F32)  # the same codes made in the call
    assert torch.equal(y, int8_linear_fwd(codes, w, one, x_scale=scale, out_dtype=F32))
    assert int8_linear_fwd(x, w, one).dtype == dtype


@pytest.mark.parametrize("M", [2, 140])
def test_rows_that_are_not_finite(M):
    """An infinity or a NaN makes its own row's outputs not finite, and no other row's."""
    from linquant_b200.kernels.layer import int8_linear_fwd

    x = randn(M, 96, dtype=BF16)
    x[0, 5], x[1, 7] = INF, float("nan")
    y = int8_linear_fwd(x, padded(int_codes(40, 96)), torch.ones(40, device="cuda"))
    assert not torch.isfinite(y[:2]).any() and torch.isfinite(y[2:]).all()


# ------------------------------------------------------------------------------------------------------------- norms
NORM = 64 * ULP  # a sum of squares over 256 threads and eight values each, its root, three products; SiLU as above


@pytest.mark.parametrize("lead,D,dtype,pad,form", [
    ((1,), 1, F32, 0, "plain"), ((5,), 7, BF16, 0, "post"), ((3, 4), 64, F16, 0, "residual"), ((33,), 2560, BF16, 8, "post"),
    ((9,), 2561, F16, 0, "post"), ((6,), 5120, F32, 0, "f32"), ((2,), 16384, BF16, 0, "vector"), ((2,), 16383, F16, 1, "f32"),
    ((130,), 264, BF16, 0, "f32"), ((4,), 1100, F32, 4, "vector"), ((3,), 9000, BF16, 0, "residual"), ((0,), 64, F16, 0, "residual")])
def test_rms_norm(lead, D, dtype, pad, form):
    from linquant_b200.kernels.layer import rms_norm_fwd

    x, w = wide(*lead, D, dtype=dtype, pad=pad), randn(D)
    res = None if form == "plain" else wide(*lead, D, dtype=F32 if form == "f32" else dtype, pad=pad)
    post = randn(D) if form == "post" else None
    scale = randn(D) if form == "vector" else 0.4
    eps = 1e-5
    kw = dict(residual=res, residual_scale=scale, post_weight=post, eps=eps)
    v = x.double().cpu()
    mag = v.abs()
    if res is not None:
        v = ref.norm(v, eps) * post.double().cpu() if post is not None else v
        v = v * (scale.double().cpu() if form == "vector" else scale)
        mag, v = v.abs() + res.double().cpu().abs(), v + res.double().cpu()
    want = ref.norm(v, eps) * w.double().cpu()
    ymag = mag / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * w.double().cpu().abs()
    out = rms_norm_fwd(x, w, **kw)
    y, r = (out, None) if res is None else out
    ref.check(y, want, ymag, NORM)
    if res is not None:
        assert r.dtype == res.dtype
        ref.check(r, v, mag, NORM)
        none, r2 = rms_norm_fwd(x, None, **kw)
        assert none is None and torch.equal(r, r2)
    out = rms_norm_fwd(x, w, quantize=True, **kw)
    codes, s = out if res is None else out[0]
    if v.numel():
        tight, _ = ref.codes(want)  # a code may be off by the norm's own error, in steps of its scale
        assert ((codes.double().cpu() - tight).abs() <= 0.5 + (ymag / s.double().cpu()[..., None] + 127) * NORM).all()
        assert res is None or torch.equal(out[1], r)
    for o in (F16, BF16, F32):
        out = rms_norm_fwd(x, w, out_dtype=o, **kw)
        y = out if res is None else out[0]
        assert y.dtype == o
        ref.check(y, want, ymag, NORM)


@pytest.mark.parametrize("rows,D,group,dtype,pad", [(3, 8, 1, F32, 0), (5, 640, 64, BF16, 0), (7, 130, 13, F16, 3), (64, 5120, None, BF16, 5456),
                                                    (4, 2048, 128, F32, 0), (2, 16384, 8192, F16, 0), (6, 96, 32, BF16, 8), (2, 4098, 2049, F32, 1)])
@pytest.mark.parametrize("first", [True, False])
def test_gated_rms_norm(rows, D, group, dtype, pad, first):
    from linquant_b200.kernels.layer import gated_rms_norm_fwd

    x, z, w = randn(rows, D, dtype=dtype), wide(rows, D, dtype=dtype, pad=pad), randn(D)
    v, g = x.double().cpu(), ref.silu(z.double().cpu())
    n = D if group is None else group
    v = v * g if first else v
    want = (ref.norm(v.view(rows, -1, n), 1e-6) * w.double().cpu().view(-1, n)).view(rows, D)
    want = want if first else want * g
    ref.check(gated_rms_norm_fwd(x, z, w, group_size=group, gate_first=first, eps=1e-6), want, want.abs(), NORM)
    codes, s = gated_rms_norm_fwd(x, z, w, group_size=group, gate_first=first, eps=1e-6, quantize=True)
    tight, _ = ref.codes(want)
    assert (codes.double().cpu() - tight).abs().max() <= 0.5 + 2 * 127 * NORM


def test_rows_of_zeros():
    from linquant_b200.kernels.layer import gated_rms_norm_fwd, rms_norm_fwd

    x, w = torch.zeros(3, 200, device="cuda", dtype=BF16), randn(200)
    assert not rms_norm_fwd(x, w).any() and not gated_rms_norm_fwd(x, x, w).any()
    codes, scale = rms_norm_fwd(x, w, quantize=True)
    assert not codes.any() and not scale.any()


# -------------------------------------------------------------------------------------------------- streams, refusals
def test_on_another_stream():
    """Calls go to the current stream: results of a chain on a side stream are those of the default one."""
    from linquant_b200.kernels import layer

    x, w, sw = randn(256, 1024, dtype=BF16), padded(int_codes(512, 1024)), torch.rand(512, device="cuda")
    norm = randn(1024)

    def chain():
        codes, scale = layer.rms_norm_fwd(x, norm, quantize=True)
        y = layer.int8_linear_fwd(codes, w, sw, x_scale=scale, out_dtype=BF16)
        return layer.short_conv_fwd(y.unsqueeze(0), randn_w)[0]

    randn_w = randn(512, 4)
    want = chain()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)  # what is queued behind it must not run ahead on the default stream
        got = chain()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = chain()
    graph.replay()
    assert torch.equal(captured, want)


def test_refusals():
    from linquant_b200 import _cabi
    from linquant_b200.kernels import layer

    x, w = randn(2, 9, 32, dtype=BF16), randn(32, 4)
    bad_shape = [
        lambda: layer.short_conv_fwd(x, randn(31, 4)),
        lambda: layer.short_conv_fwd(x, w, initial_state=randn(2, 4, 32, dtype=BF16)),
        lambda: layer.short_conv_fwd(x, w, lengths=ints(1, 2, 3)),
        lambda: layer.short_conv_fwd(x[0], w),
        lambda: layer.short_conv_step(x[:, 0], randn(2, 2, 32, dtype=BF16), w),
        lambda: layer.short_conv_step(x[:, 0], randn(1, 3, 32, dtype=BF16), w),                    # fewer slots than sequences
        lambda: layer.short_conv_step(x[:, 0], randn(2, 32, 3, dtype=BF16).transpose(1, 2), w),    # in place: no copy
        lambda: layer.selective_scan_fwd(x, x, randn(32, 8), randn(2, 9, 1, 8, dtype=BF16), randn(2, 9, 1, 7, dtype=BF16)),
        lambda: layer.selective_scan_fwd(x, x[..., :31], randn(32, 8), *[randn(2, 9, 1, 8, dtype=BF16)] * 2),
        lambda: layer.selective_scan_fwd(x, x, randn(32, 8), *[randn(2, 9, 3, 8, dtype=BF16)] * 2),  # 32 channels in 3 groups
        lambda: layer.selective_scan_step(randn(2, 32, 8), x[:, 0], x[:, 0], randn(32), *[randn(2, 1, 8, dtype=BF16)] * 2),
        lambda: layer.int8_linear_fwd(x, int_codes(5, 31), randn(5)),
        lambda: layer.int8_linear_fwd(x, int_codes(5, 32), randn(4)),
        lambda: layer.int8_linear_fwd(x, int_codes(5, 32), randn(5), x_scale=randn(2, 9)),
        lambda: layer.int8_linear_fwd(int_codes(4, 32), int_codes(5, 32), randn(5)),
        lambda: layer.int8_linear_fwd(int_codes(1, 131072), int_codes(5, 131072), randn(5), x_scale=randn(1)),
        lambda: layer.rms_norm_fwd(x, randn(33)),
        lambda: layer.rms_norm_fwd(x, randn(32), residual=x[:1]),
        lambda: layer.gated_rms_norm_fwd(x, x, randn(32), group_size=5),
    ]
    for i, call in enumerate(bad_shape):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"call {i} was taken")
    unsupported = [
        lambda: layer.short_conv_fwd(x, randn(32, 5)),
        lambda: layer.short_conv_fwd(x, randn(32, 1)),
        lambda: layer.short_conv_fwd(x.double(), w),
        lambda: layer.short_conv_fwd(x, w, activation="gelu"),
        lambda: layer.short_conv_fwd(x, w, lengths=torch.ones(2, device="cuda")),
        lambda: layer.short_conv_fwd(x, w, initial_state=randn(2, 3, 32)),
        lambda: layer.short_conv_step(x[:, 0], randn(2, 3, 32), w),
        lambda: layer.selective_scan_fwd(x, x.float(), randn(32, 8), *[randn(2, 9, 1, 8, dtype=BF16)] * 2),
        lambda: layer.selective_scan_fwd(x, x, randn(32, 257), *[randn(2, 9, 1, 257, dtype=BF16)] * 2),
        lambda: layer.selective_scan_step(randn(2, 32, 8).double(), x[:, 0], x[:, 0], randn(32, 8), *[randn(2, 1, 8, dtype=BF16)] * 2),
        lambda: layer.int8_linear_fwd(x, randn(5, 32), randn(5)),
        lambda: layer.int8_linear_fwd(x, int_codes(5, 32), randn(5), out_dtype=torch.float64),
        lambda: layer.rms_norm_fwd(x.double(), randn(32)),
        lambda: layer.rms_norm_fwd(x, randn(32), residual=x.half()),
        lambda: layer.rms_norm_fwd(randn(2, 16385), randn(16385)),
        lambda: layer.gated_rms_norm_fwd(x, x.half(), randn(32)),
    ]
    for i, call in enumerate(unsupported):
        with pytest.raises(NotImplementedError):
            call()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(_cabi.LinQuantError):
        layer.rms_norm_fwd(x, None)  # nothing to compute
    with pytest.raises(_cabi.LinQuantError):
        layer.rms_norm_fwd(x, w[:, 0], post_weight=w[:, 0])  # a norm of the block's output goes to a residual
    with pytest.raises(_cabi.LinQuantError):
        layer.gated_rms_norm_fwd(x, x.cpu(), randn(32))


@pytest.mark.parametrize("out", [F16, BF16, F32])
@pytest.mark.parametrize("M,K,N", [(8210, 100, 3500), (20011, 272, 1290)])
def test_int8_linear_many_tiles(M, K, N, out):
    """Pairs of CTAs on one tile, the last rows and columns ragged (M past a pair's 256 tokens by less and by more than 128)."""
    from linquant_b200.kernels.layer import int8_linear_fwd

    x, w = int_codes(M, K, -128), int_codes(N, K, -128)
    xs, ws, b = (torch.rand(n, device="cuda") for n in (M, N, N))
    y = int8_linear_fwd(padded(x), padded(w), ws, x_scale=xs, bias=b, out_dtype=out)
    want = (x.double() @ w.double().t()) * xs.double()[:, None] * ws.double() + b.double()
    # three roundings to fp32 of a product and its sum with the bias, one to the output
    size = ((x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()).abs() + b.double()
    bound = 4 * 2.0**-24 * size + (0 if out == F32 else torch.finfo(out).eps / 2 * want.abs() + (2.0**-25 if out == F16 else 0))
    fits = want.abs() < torch.finfo(out).max
    assert ((y.double() - want).abs() <= bound * (1 + 2.0**-20))[fits].all()
    most = torch.finfo(out).max
    assert (torch.where(want > 0, y, -y).double() >= most)[~fits].all()  # behind the type's range: its largest value or infinity


@pytest.mark.parametrize("out", [F16, BF16, F32])
@pytest.mark.parametrize("M,K,N", [(17, 4096, 130), (40, 4111, 1001), (129, 8200, 64), (255, 16384, 2047), (30, 131071, 5)])
def test_int8_linear_long_rows(M, K, N, out):
    """Few tiles: parts of K that meet in a cluster. The sums are whole numbers, the same in any order."""
    from linquant_b200.kernels.layer import int8_linear_fwd

    x, w = int_codes(M, K, -128), int_codes(N, K, -128)
    one_m, one_n = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
    want = x.double() @ w.double().t()
    y = int8_linear_fwd(padded(x), padded(w), one_n * 2.0**-12, x_scale=one_m * 2.0**-3, out_dtype=out)
    # the sum rounds to fp32, scales that are powers of two round nothing, then one rounding to the output
    assert torch.equal(y, (want.float() * 2.0**-15).to(out))
    assert torch.equal(y, int8_linear_fwd(padded(x), padded(w), one_n * 2.0**-12, x_scale=one_m * 2.0**-3, out_dtype=out))


@pytest.mark.parametrize("heads", [False, True])
def test_steps_of_no_sequences(heads):
    from linquant_b200.kernels.layer import selective_scan_step, short_conv_step

    state = randn(3, 4, 8, 16) if heads else randn(3, 32, 16)
    before = state.clone()
    u = torch.empty(0, 4, 8, device="cuda", dtype=BF16) if heads else torch.empty(0, 32, device="cuda", dtype=BF16)
    dt = torch.empty(0, 4, device="cuda", dtype=BF16) if heads else u
    A = -torch.rand(4, device="cuda") if heads else -torch.rand(32, 16, device="cuda")
    none = torch.empty(0, 1, 16, device="cuda", dtype=BF16)
    assert selective_scan_step(state, u, dt, A, none, none).shape == u.shape and torch.equal(state, before)
    x, line = torch.empty(0, 8, device="cuda", dtype=BF16), torch.zeros(2, 3, 8, device="cuda", dtype=BF16)
    assert short_conv_step(x, line, torch.ones(8, 4, device="cuda")).shape == x.shape
    torch.cuda.synchronize()
