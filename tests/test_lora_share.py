"""Adapters whose share is larger than the outputs that it joins: what the type of y does not hold, and what cancels, for few tokens and many."""

import ctypes

import pytest
import torch

from linquant_b200 import _cabi
from tests import layer_reference as ref
from tests.test_layer_host import filled
from tests.test_lora_linear import BF16, F16, F32, ULP, want_of

gpu = pytest.mark.gpu


def exact_error(dtype, K, R):
    """Of the adapters' sum, relative to its terms' magnitudes: the tensor core's sums (one rounding, 2^-23, for each 16 of K and of R and each
    of six pieces, 16 where parts meet), and for 16-bit outputs the 16 bits that t and b are taken with. No rounding of the sum to y's type."""
    exact = (6 * (K / 16 + R / 16 + 2) + 32) * 2 * ULP
    return exact if dtype == F32 else exact + 2.0**-15


def opposed(M, K, N, R, size, rest, dtype):
    """Codes and weights of rank one, whose product has magnitudes of ``size``, and an adapter that takes it away again but for ``rest``:
    its first rank is the product's negative, the others random."""
    u = torch.randint(0, 2, (K,), device="cuda") * 2 - 1
    turn = torch.randint(0, 2, (M,), device="cuda") * 2 - 1
    sign = torch.randint(0, 2, (N,), device="cuda") * 2 - 1
    codes = torch.randint(30, 100, (M, K), device="cuda") * u * turn.unsqueeze(1)
    w = (64 * sign.unsqueeze(1) * u).to(torch.int8)
    xs, ws = torch.full((M,), 2.0**-6, device="cuda"), torch.full((N,), size / (K * 64 * 64 * 2.0**-6), device="cuda")
    a, b = torch.randn(1, R, K, device="cuda") / K**0.5, torch.randn(1, N, R, device="cuda") * rest / R**0.5
    a[0, 0] = u
    b[0, :, 0] = -sign * 64 * ws[0]
    return codes.to(torch.int8), xs, w, ws, a.to(dtype), b.to(dtype)


@gpu
@pytest.mark.parametrize("M", [7, 16, 17, 130, 3000])
@pytest.mark.parametrize("K,N,R", [(64, 96, 8), (300, 77, 24), (2048, 64, 16)])
@pytest.mark.parametrize("dtype,size", [(F16, 3e4), (F16, 2e5), (BF16, 1e6), (F32, 1e6)])
def test_a_share_that_cancels(M, K, N, R, dtype, size):
    from linquant_b200.kernels.layer import lora_linear_fwd

    torch.manual_seed(3)
    codes, xs, w, ws, a, b = opposed(M, K, N, R, size, 30.0, F32 if dtype == F32 else dtype)
    if dtype == F16:
        assert b.abs().max() < 6e4
    which = torch.zeros(M, device="cuda", dtype=torch.int32)
    seen = codes.double() * xs.double().unsqueeze(1)
    pad = torch.zeros(N, (K + 15) // 16 * 16, device="cuda", dtype=torch.int8)
    pad[:, :K] = w
    y = lora_linear_fwd(codes, pad[:, :K], ws, a, b, which, x_scale=xs, out_dtype=dtype)
    base, mag, low = want_of(seen, codes, xs, w, ws, a, b, which, 1.0, None)
    assert float(base.abs().max()) < 6e4 and float(low.max()) > size / 3  # the sum fits, its parts are large
    e = exact_error(dtype, K, R)
    ref.check(y, base, mag * (4 * ULP / e) + low, e)


@gpu
def test_rows_of_small_and_large_batches_agree():
    """A row on both sides of 16 tokens: the same sum, but for the roundings in front of it."""
    from linquant_b200.kernels.layer import lora_linear_fwd

    torch.manual_seed(4)
    codes, xs, w, ws, a, b = opposed(40, 256, 64, 16, 2e5, 30.0, F16)
    which = torch.zeros(40, device="cuda", dtype=torch.int32)
    many = lora_linear_fwd(codes, w, ws, a, b, which, x_scale=xs, out_dtype=F16)
    few = torch.cat([lora_linear_fwd(codes[i:i + 10], w, ws, a, b, which[i:i + 10], x_scale=xs[i:i + 10], out_dtype=F16) for i in range(0, 40, 10)])
    seen = codes.double() * xs.double().unsqueeze(1)
    base, mag, low = want_of(seen, codes, xs, w, ws, a, b, which, 1.0, None)
    e = exact_error(F16, 256, 16)
    bound = 2 * (ref.UNIT[F16] * base.abs() + (e * low + 4 * ULP * mag) * (1 + ref.UNIT[F16]))
    assert bool(torch.isfinite(many).all()) and bool(((many.double() - few.double()).abs() <= bound).all())


@gpu
def test_many_tokens_in_slabs():
    """More outputs than the share is held for at once: every slab's rows and both sides of its ends."""
    from linquant_b200.kernels.layer import lora_linear_fwd, quantize_rows_fwd

    torch.manual_seed(5)
    M, K, N, R, L = 150_001, 32, 4100, 8, 3  # 2.5 GB of fp32 shares
    w, ws = quantize_rows_fwd(torch.randn(N, K, device="cuda") / K**0.5)
    a, b = (torch.randn(L, R, K, device="cuda") / K**0.5).half(), (torch.randn(L, N, R, device="cuda") / R**0.5).half()
    x = torch.randn(M, K, device="cuda").half()
    which = (torch.arange(M, device="cuda") // 700 % 4).int()
    y = lora_linear_fwd(x, w, ws, a, b, which, scaling=0.5)
    codes, xs = quantize_rows_fwd(x)
    e = exact_error(F16, K, R)
    for i in range(0, M, 30_000):
        rows = slice(i, i + 30_000)
        base, mag, low = want_of(x[rows], codes[rows], xs[rows], w, ws, a, b, which[rows], 0.5, None)
        ref.check(y[rows], base, mag * (4 * ULP / e) + low, e)


# ------------------------------------------------------------------------------------------------------- without a GPU
def share_bytes(M, N, out):
    fn = _cabi.lib().lq_lora_share_bytes
    fn.argtypes, fn.restype = [ctypes.c_int] * 3, ctypes.c_size_t
    return fn(M, N, out)


def test_scratch_of_the_share():
    assert share_bytes(16, 4096, 1) == 0 and share_bytes(40, 4096, 2) == 0 and share_bytes(17, 0, 1) == 0  # few tokens; fp32 outputs; nothing
    assert share_bytes(17, 1000, 1) == 32 * 1000 * 4 and share_bytes(16384, 10576, 0) == 16384 * 10576 * 4  # one slab: whole blocks of 32 tokens
    for M, N in ((17, 1), (33, 77), (16384, 10576), (150_001, 4100), (2_100_003, 1032), (2**31 - 9000, 7), (2**31 - 9000, 2**20)):
        n = share_bytes(M, N, 1)
        pitch = (N + 3) // 4 * 4
        assert n >= min(M * N * 4, 2**28) and n <= max(2**30, 1024 * pitch * 4) + 64 * pitch * 4, (M, N, n)


@pytest.mark.parametrize("share,want", [(None, 1), (4104, 3)])
def test_a_share_without_its_scratch(share, want):
    p = filled(_cabi.LinearProblem, M=40, N=8, K=32, x_stride=32, w_stride=32, out_dtype=1)
    q = filled(_cabi.LoraProblem, L=2, R=16, dtype=1, scale=1.0, share=share)
    fn = _cabi.lib().lq_lora_linear
    fn.argtypes = [ctypes.POINTER(_cabi.LinearProblem), ctypes.POINTER(_cabi.LoraProblem), ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p]
    assert fn(ctypes.byref(p), ctypes.byref(q), None, 0, 0, None) == want
