"""Calls of one kernel with different amounts of shared memory, from two threads at once: none may be refused."""

import ctypes as C
import threading

import pytest
import torch

from linquant_b200 import _cabi

pytestmark = pytest.mark.gpu

CALLS = 5000  # where each call's own size is opted in to, 0.4 to 18 % of the larger ones are refused


def run(calls):
    """Each call in a thread of its own, CALLS times on a stream of its own; the statuses that were not 0."""
    bad, start = [], threading.Barrier(len(calls))

    def work(call):
        stream = torch.cuda.Stream()
        start.wait()
        bad.extend(s for s in (call(C.c_void_p(stream.cuda_stream)) for _ in range(CALLS)) if s != 0)

    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return bad


def entry(name, *types):
    fn = getattr(_cabi.lib(), name)
    fn.argtypes = [*types, C.c_void_p]
    return fn


def product(K, M=8, N=16):
    """INT8 product from values: a CTA holds the codes of its tokens."""
    v, y = torch.randn(M, K, device="cuda").bfloat16(), torch.empty(M, N, device="cuda", dtype=torch.bfloat16)
    w, x = (torch.ones(n, K, device="cuda", dtype=torch.int8) for n in (N, M))
    ws, xs = torch.ones(N, device="cuda"), torch.empty(M, device="cuda")
    p = _cabi.LinearProblem(M=M, N=N, K=K, out_dtype=1, x_stride=K, w_stride=K, x=x.data_ptr(), w=w.data_ptr(), x_scale=xs.data_ptr(),
                            w_scale=ws.data_ptr(), y=y.data_ptr())
    fn = entry("lq_int8_linear_values", C.POINTER(_cabi.LinearProblem), C.c_void_p, C.c_int, C.c_longlong)
    return lambda stream, keep=(v, y, w, x, ws, xs): fn(C.byref(p), v.data_ptr(), 1, K, stream)


def norm(D, post, rows=3):
    """Residual and norm of rows off 16 bytes: a CTA holds the parameters."""
    x, res, y, out = (torch.randn(rows, D, device="cuda").bfloat16() for _ in range(4))
    w = torch.ones(D, device="cuda")
    p = _cabi.NormProblem(rows=rows, D=D, group=D, dtype=1, out_dtype=1, eps=1e-5, residual_scale=1.0, x_stride=D, residual_stride=D, x=x.data_ptr(),
                          residual=res.data_ptr(), weight=w.data_ptr(), post_weight=w.data_ptr() if post else None, y=y.data_ptr(), residual_out=out.data_ptr())
    fn = entry("lq_rms_norm", C.POINTER(_cabi.NormProblem))
    return lambda stream, keep=(x, res, y, out, w): fn(C.byref(p), stream)


@pytest.mark.parametrize("calls", [lambda: (product(64), product(14000)), lambda: (norm(5201, False), norm(15001, True))], ids=["product", "norm"])
def test_layer_operators(calls):
    assert run(calls()) == []


def chunk_state(chunk, L=256, H=2, N=64):
    """Chunk states of Mamba-2 by way of the transposed codes of B: a chunk's rows lie in shared memory."""
    from linquant_b200.kernels.mamba2 import _ssd

    nc = L // chunk
    x, q = torch.randn(1, L, H, 64, device="cuda").half(), torch.ones(1, L, 1, N, device="cuda", dtype=torch.int8)
    dt, dA, one = torch.rand(1, H, nc, chunk, device="cuda"), torch.zeros(1, H, nc, chunk, device="cuda"), torch.ones(H, 64, device="cuda")
    call = _ssd.Call(x.device).dims(B=1, L=L, H=H, P=64, G=1, N=N, chunk=chunk)
    call.x(x)
    for name, t in (("q_B", q), ("q_BT", torch.empty_like(q)), ("dt", dt), ("dA", dA), ("alpha_hp", one), ("state_scale", one), ("bscale_g", one),
                    ("states", torch.empty(1, nc, H, 64, N, device="cuda", dtype=torch.int8))):
        call.put(name, t)
    fn = entry("lq_ssd_chunk_state_value", C.POINTER(_ssd.SsdProblem))
    return lambda stream: fn(C.byref(call.p), stream)


def test_chunk_states():
    assert run((chunk_state(128), chunk_state(256))) == []
