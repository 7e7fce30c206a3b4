"""Layer operators at sizes at which a CTA or a thread takes more than one piece of the work: long runs of the convolution, rings of
tiles that are filled again, rows, tiles and channels that a CTA walks over. Sizes follow from the SM count where a dispatch rule
counts SMs. Bounds as in the tests of the operators; the references run in 64 bits on the GPU."""

import pytest
import torch

from tests import layer_reference as ref
from tests.test_layer_ops import CONV, NORM, SCAN, ULP, int_codes, ints, padded, randn, scan_inputs, wide

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
INF = float("inf")


@pytest.fixture(autouse=True)
def seed():
    torch.manual_seed(13)


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def up(a, b):
    return -(-a // b)


def check(got, want, mag, f32):
    """``ref.check`` on the GPU."""
    dt = got.dtype
    got = got.double()
    bound = ref.UNIT[dt] * (want.abs() + f32 * mag) + f32 * mag + ref.TINY[dt]
    assert got.shape == want.shape and not torch.isnan(got).any()
    over = (got - want).abs() - bound
    assert float(over.max()) <= 0, f"{float(over.max()):.3e} over the bound"


# ------------------------------------------------------------------------------------------------ short convolution
def conv_run(B, T, D, vec):  # the dispatch rule: tokens a thread walks
    lanes, fill = B * (D // vec), sms() * 512
    return 128 if lanes * (T // 128) >= 3 * fill else 32 if lanes * (T // 32) >= fill else 8


@pytest.mark.parametrize("run,dtype,D,W,initial", [(32, BF16, 1024, 4, True), (32, F16, 1027, 3, True), (32, F32, 512, 2, False),
                                                   (128, BF16, 4096, 4, True), (128, F16, 2049, 4, False), (128, F32, 4096, 3, True)])
def test_short_conv_runs(run, dtype, D, W, initial):
    """Runs of 32 and 128 tokens (rings of 16 slots that are filled again; channels one by one where D is odd), uneven lengths."""
    from linquant_b200.kernels.layer import short_conv_fwd

    B, vec = 3, 16 // torch.empty(0, dtype=dtype).element_size()
    vec = vec if D % vec == 0 else 1
    T = next(t for t in range(32, 1 << 20, 32) if conv_run(B, t, D, vec) == run) + 13
    assert conv_run(B, T, D, vec) == run
    x, w, bias = randn(B, T, D, dtype=dtype), randn(D, W) * 0.5, randn(D)
    before = randn(B, W - 1, D, dtype=dtype) if initial else None
    n = ints(T, T - run - 5, T // 2 + 3)
    for b in range(1, B):
        x[b, int(n[b]):] = float("nan")
    y, last = short_conv_fwd(x, w, bias, initial_state=before, lengths=n, output_final_state=True)
    for b in range(B):
        m = int(n[b])
        line = torch.cat([torch.zeros(W - 1, D, device="cuda") if before is None else before[b].float(), x[b, :m].float()])
        s, mag = bias.double().expand(m, D).clone(), bias.double().abs().expand(m, D).clone()
        for i in range(W):
            term = line[i:i + m].double() * w[:, i].double()
            s += term
            mag += term.abs()
        check(y[b, :m], ref.silu(s), 1.1 * mag, CONV)
        assert not y[b, m:].any() and torch.equal(last[b].float(), line[m:])


# ---------------------------------------------------------------------------------------------------- selective scan
def scan_reference(u, dt, A, B, C, D, z, bias, h0, n):
    """``ref.scan`` with softplus, on the GPU."""
    rep = u.shape[2] // B.shape[2]
    step = ref.softplus(dt.double() + bias.double())
    Bd, Cd = B.double().repeat_interleave(rep, 2), C.double().repeat_interleave(rep, 2)
    h, A = h0.double(), A.double()
    hm = h.abs()
    y, mag = torch.zeros_like(u, dtype=torch.float64), torch.zeros_like(u, dtype=torch.float64)
    for t in range(u.shape[1]):
        on = (n > t)[:, None, None]
        a = torch.exp(step[:, t, :, None] * A)
        x = (step[:, t] * u[:, t].double())[..., None] * Bd[:, t]
        h, hm = torch.where(on, a * h + x, h), torch.where(on, a * hm + x.abs(), hm)
        y[:, t], mag[:, t] = torch.where(on[..., 0], (Cd[:, t] * h).sum(-1), 0.0), torch.where(on[..., 0], (Cd[:, t].abs() * hm).sum(-1), 0.0)
    on = torch.arange(u.shape[1], device="cuda")[None, :, None] < n[:, None, None]
    skip = torch.where(on, D.double() * u.double(), 0.0)
    gate = torch.where(on, ref.silu(z.double()), 0.0) if z is not None else torch.ones_like(y)
    return (y + skip) * gate, (mag + skip.abs()) * gate.abs(), h, hm


def scan_is_wide(b, G, Dg, N):  # the dispatch rule up to 16 states: 64 channels a CTA, not 16
    c16, c64 = (65, 103) if N <= 4 else (42, 94) if N <= 8 else (44, 128)
    return up(b * G * up(Dg, 16), sms()) * c16 >= up(b * G * up(Dg, 64), sms()) * c64


# channels enough for 64 of them a CTA ("wide"), or not; rows on 16 bytes come as TMA tiles, others in pieces
@pytest.mark.parametrize("T,G,N,dtype,channels,pad", [
    (700, 1, 16, BF16, "few", 0), (517, 2, 16, F32, "few", 0), (333, 1, 16, BF16, "wide", 0), (300, 1, 16, F32, "wide", 0),
    (450, 1, 13, F16, "few", 3), (290, 1, 13, BF16, "wide", 1),
    (650, 1, 8, BF16, "few", 0), (300, 2, 8, F16, "wide", 0), (300, 1, 8, F32, "wide", 0), (300, 1, 7, F32, "wide", 1),
    (600, 1, 4, F32, "few", 0), (300, 1, 4, F32, "wide", 0), (290, 1, 3, BF16, "wide", 0),
    (300, 1, 32, BF16, "few", 0), (260, 2, 32, F32, "few", 0), (300, 2, 64, BF16, "few", 0), (200, 1, 64, F32, "few", 0),
    (200, 1, 128, BF16, "few", 0), (150, 2, 128, F32, "few", 0), (200, 1, 256, BF16, "few", 0), (150, 1, 256, F32, "few", 0),
    (200, 1, 100, F16, "few", 2), (150, 1, 200, BF16, "few", 1)])
def test_selective_scan_tiles(T, G, N, dtype, channels, pad):
    """More tiles than the ring holds, in every shape of a CTA."""
    from linquant_b200.kernels.layer import selective_scan_fwd

    b = 2
    d = (up(sms() * 60, b * 64 * G) * 64 if channels == "wide" else 48) * G
    assert N > 16 or scan_is_wide(b, G, d // G, N) == (channels == "wide")
    u, dt, A, B, C, bias = scan_inputs(b, T, d, G, N, dtype, pad)
    D, z, h0, n = randn(d), wide(b, T, d, dtype=dtype, pad=pad), randn(b, d, N), ints(T, T - 39)
    want, mag, h, hm = scan_reference(u, dt, A, B, C, D, z, bias, h0, n)
    for t in (u, dt, B, C, z):
        t[1, T - 39:] = float("nan")
    y, end = selective_scan_fwd(u, dt, A, B, C, D=D, z=z, dt_bias=bias, initial_state=h0, lengths=n, output_final_state=True)
    check(y, torch.nan_to_num(want), torch.nan_to_num(mag), SCAN)
    check(end, h, hm, SCAN)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_selective_scan_of_tokens_ahead_of_sequences(dtype):
    """Inputs laid out token by token, the sequences of a token next to one another; expanded ones."""
    from linquant_b200.kernels.layer import selective_scan_fwd

    b, T, d, G, N = 3, 400, 96, 2, 16
    u, dt, z = (randn(T, b, d, dtype=dtype).transpose(0, 1) for _ in range(3))
    B, C = randn(T, b, G * N + 32, dtype=dtype)[..., :G * N].unflatten(-1, (G, N)).transpose(0, 1), randn(T, G, b, N, dtype=dtype).permute(2, 0, 1, 3)
    one = randn(1, T, G, N, dtype=dtype).expand(b, T, G, N)
    A = -torch.rand(d, N, device="cuda") - 0.1
    for c in (C, one):
        y, h = selective_scan_fwd(u, dt, A, B, c, z=z, output_final_state=True)
        y2, h2 = selective_scan_fwd(*(t.contiguous() for t in (u, dt, A, B, c)), z=z.contiguous(), output_final_state=True)
        assert torch.equal(y, y2) and torch.equal(h, h2)


@pytest.mark.parametrize("H,P,N,G,dtype,sdtype", [(80, 64, 128, 1, BF16, F32), (96, 16, 128, 2, F16, F32), (74, 32, 64, 1, F32, BF16), (120, 24, 16, 3, BF16, F32)])
def test_selective_scan_step_of_many_heads(H, P, N, G, dtype, sdtype):
    """Teams that walk over more than four channels of a head: where threads enough are left for the GPU."""
    from linquant_b200.kernels.layer import selective_scan_step

    per = 16 // torch.empty(0, dtype=sdtype).element_size()
    lanes = 1 << (up(N, per) - 1).bit_length()
    b = up(sms() * 1024, H * lanes)  # P channels by one team
    u, z, dt, bias = randn(b, H, P, dtype=dtype), randn(b, H, P, dtype=dtype), randn(b, H, dtype=dtype), randn(H) - 2
    A, D = -(torch.rand(H, device="cuda") * 15 + 0.5), randn(H)
    B, C, state = randn(b, G, N, dtype=dtype), randn(b, G, N, dtype=dtype), randn(b + 1, H, P, N, dtype=sdtype)
    slots = torch.randperm(b + 1, device="cuda")[:b].to(torch.int32)
    at, before = slots.long(), state.double()
    y = selective_scan_step(state, u, dt, A, B, C, D=D, z=z, dt_bias=bias, slots=slots)
    step = ref.softplus(dt.double() + bias.double())[..., None]
    rep = H // G
    Bd, Cd = (t.double().repeat_interleave(rep, 1)[:, :, None] for t in (B, C))
    old = before[at]
    a, x = torch.exp(step * A.double()[:, None])[..., None], (step * u.double())[..., None] * Bd
    h, hm, skip, gate = a * old + x, a * old.abs() + x.abs(), D.double()[:, None] * u.double(), ref.silu(z.double())
    check(y, ((h * Cd).sum(-1) + skip) * gate, ((hm * Cd.abs()).sum(-1) + skip.abs()) * gate.abs(), 300 * ULP)
    check(state[at], h, hm, 64 * ULP)
    idle = [i for i in range(b + 1) if i not in set(slots.tolist())]
    assert torch.equal(state[idle].double(), before[idle])


# ------------------------------------------------------------------------------------------------------------- norms
# Rows for several rounds of every CTA: of 128 threads or more an SM holds at most 16 CTAs
def rows_of(D):
    per_cta = max(1, 128 // max(1, up(D, 8)))
    return sms() * 16 * per_cta * 2 + 5


@pytest.mark.parametrize("D,dtype,form", [(64, BF16, "plain"), (250, F16, "residual"), (2560, BF16, "post"), (2561, F16, "post"), (2561, BF16, "plain"),
                                          (2560, BF16, "f32"), (2561, F16, "f32"), (5123, BF16, "residual"), (1536, F32, "residual")])
def test_rms_norm_of_many_rows(D, dtype, form):
    from linquant_b200.kernels.layer import rms_norm_fwd

    rows, eps = rows_of(D), 1e-5
    x, w = randn(rows, D, dtype=dtype), randn(D)
    res = None if form == "plain" else randn(rows, D, dtype=F32 if form == "f32" else dtype)
    post = randn(D) if form == "post" else None
    kw = dict(residual=res, residual_scale=0.4, post_weight=post, eps=eps)
    v = x.double()
    mag = v.abs()
    if res is not None:
        v = 0.4 * (ref.norm(v, eps) * post.double() if post is not None else v)
        mag, v = v.abs() + res.double().abs(), v + res.double()
    want = ref.norm(v, eps) * w.double()
    ymag = mag / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * w.double().abs()
    out = rms_norm_fwd(x, w, **kw)
    y = out if res is None else out[0]
    check(y, want, ymag, NORM)
    if res is not None:
        check(out[1], v, mag, NORM)
    out = rms_norm_fwd(x, w, quantize=True, **kw)
    codes, s = out if res is None else out[0]
    amax = want.abs().amax(-1, keepdim=True)
    assert ((codes.double() - want * 127 / amax).abs() <= 0.5 + (ymag / s.double()[:, None] + 127) * NORM).all()


@pytest.mark.parametrize("D,group,dtype,pitch,first", [(5120, None, BF16, 10576, True), (5120, 640, F16, 0, True), (1280, 64, BF16, 0, False),
                                                       (2561, None, F16, 0, False), (2561, None, BF16, 5122, True), (960, 96, F32, 0, True)])
def test_gated_rms_norm_of_many_rows(D, group, dtype, pitch, first):
    from linquant_b200.kernels.layer import gated_rms_norm_fwd

    rows, n = rows_of(group or D), group or D
    x, z, w = randn(rows, D, dtype=dtype), wide(rows, D, dtype=dtype, pad=pitch - D if pitch else 0), randn(D)
    v, g = x.double(), ref.silu(z.double())
    v = v * g if first else v
    want = (ref.norm(v.view(rows, -1, n), 1e-6) * w.double().view(-1, n)).view(rows, D)
    want = want if first else want * g
    check(gated_rms_norm_fwd(x, z, w, group_size=group, gate_first=first, eps=1e-6), want, want.abs(), NORM)
    codes, _ = gated_rms_norm_fwd(x, z, w, group_size=group, gate_first=first, eps=1e-6, quantize=True)
    amax = want.abs().amax(-1, keepdim=True)
    assert (codes.double() - want * 127 / amax).abs().max() <= 0.5 + 2 * 127 * NORM


@pytest.mark.parametrize("D,dtype", [(64, BF16), (2560, F16), (2561, BF16), (1001, F32)])
def test_codes_of_many_rows(D, dtype):
    from linquant_b200.kernels.layer import quantize_rows_fwd

    x = randn(rows_of(D), D, dtype=dtype)
    x[7] = 0
    codes, scale = quantize_rows_fwd(x)
    amax = x.double().abs().amax(-1)
    assert ((scale.double() - amax / 127).abs() <= 16 * ULP * amax / 127).all()
    step = torch.where(amax > 0, amax / 127, 1.0)[:, None]
    assert ((codes.double() - x.double() / step).abs() <= 0.5 + 127 * 16 * ULP).all()


# ------------------------------------------------------------------------------------------------------ INT8 product
def widest(M, N):  # the dispatch rule of tiles: the columns of one
    best = least = None
    for bn in (256, 128, 64):
        cost = up(up(M, 128) * up(N, bn), sms()) * (bn + 64)
        if least is None or cost < least:
            best, least = bn, cost
    return best


@pytest.mark.parametrize("out", [F16, BF16, F32])
@pytest.mark.parametrize("bn,K", [(256, 192), (128, 1000), (64, 400)])
def test_int8_linear_several_tiles_a_cta(bn, K, out):
    """One CTA a tile, each walking over several: both accumulators and the ring of stages are taken again."""
    from linquant_b200.kernels.layer import int8_linear_fwd

    M, N = next((m, n) for m in range(1000, 6000, 130) for n in range(1001, 12000, 210)
                if widest(m, n) == bn and up(m, 128) * up(n, bn) > 2 * sms() and up(m, 128) * up(n, 256) < 6 * sms())
    x, w = int_codes(M, K, -128), int_codes(N, K, -128)
    one_m, one_n = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
    want = x.double() @ w.double().t()
    # sums of up to 24 bits are exact, scales that are powers of two round nothing, then one rounding to the output
    y = int8_linear_fwd(padded(x), padded(w), one_n * 2.0**-12, x_scale=one_m * 2.0**-3, out_dtype=out)
    assert torch.equal(y, (want.float() * 2.0**-15).to(out))


@pytest.mark.parametrize("K", [48, 1000, 2560, 2561, 5120, 5200])
@pytest.mark.parametrize("M", [1, 3, 8, 13, 16])
def test_int8_linear_few_tokens_many_tiles(M, K):
    """CTAs that walk over tiles of 16 output channels, the codes made in the call and ahead of it."""
    from linquant_b200.kernels.layer import int8_linear_fwd, quantize_rows_fwd

    N = 16 * sms() * 5 + 3  # an SM holds two CTAs at most
    x, w, sw, bias = randn(M, K, dtype=BF16), padded(int_codes(N, K, -128)), torch.rand(N, device="cuda"), randn(N)
    codes, sx = quantize_rows_fwd(x)
    want = (codes.double() @ w.double().t()) * sx.double()[:, None] * sw.double()
    y = int8_linear_fwd(codes, w, sw, x_scale=sx, bias=bias, out_dtype=F32)
    check(y, want + bias.double(), want.abs() + bias.double().abs(), 4 * ULP)
    assert torch.equal(int8_linear_fwd(x, w, sw, bias=bias, out_dtype=F32), y)


@pytest.mark.parametrize("M", [4, 40, 300])
def test_int8_linear_rows_that_share_bytes(M):
    """One row of codes for every token, and rows that overlap, are read in place."""
    from linquant_b200.kernels.layer import int8_linear_fwd

    w, one, scale = int_codes(40, 64), torch.ones(40, device="cuda"), torch.ones(M, device="cuda")
    flat = int_codes(1, 16 * M + 64)[0]
    for x in (flat[:64].expand(M, 64), flat.as_strided((M, 64), (16, 1))):
        assert torch.equal(int8_linear_fwd(x, w, one, x_scale=scale, out_dtype=F32).double(), x.double() @ w.double().t())
