"""The layer operators' C entries and wrappers, as far as no GPU is needed: layouts, refusals before any launch."""

import ctypes

import pytest
import torch

from linquant_b200 import _cabi


def call(entry, p):
    fn = getattr(_cabi.lib(), entry)
    fn.argtypes = [ctypes.POINTER(type(p)), ctypes.c_void_p]
    return fn(ctypes.byref(p), None)


def filled(cls, **kw):
    p = cls()
    for name, t in cls._fields_:
        if t is ctypes.c_void_p:
            setattr(p, name, 4096)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def test_layouts_match_the_compiled_structs():
    L = _cabi.lib()
    L.lq_struct_bytes.restype = ctypes.c_ulonglong
    L.lq_struct_bytes.argtypes = [ctypes.c_int]
    for i, cls in enumerate((_cabi.ConvProblem, _cabi.ScanProblem, _cabi.LinearProblem, _cabi.NormProblem), 3):
        assert L.lq_struct_bytes(i) == ctypes.sizeof(cls), cls.__name__


@pytest.mark.parametrize("over,want", [({}, 0), ({"W": 5}, 4), ({"D": 0}, 2), ({"T": -1}, 2), ({"dtype": 7}, 4), ({"weight": None}, 1), ({"x": None, "T": 3}, 1)])
def test_conv_entry(over, want):
    p = filled(_cabi.ConvProblem, B=0, T=3, D=8, W=4, dtype=1, **{})
    if over.get("x", 0) is None:
        p.B = 1
    for k, v in over.items():
        setattr(p, k, v)
    assert call("lq_short_conv_fwd", p) == want


@pytest.mark.parametrize("over,want", [({}, 0), ({"N": 257}, 4), ({"N": 0}, 2), ({"G": 3}, 2), ({"H": 2, "P": 4}, 4), ({"A": None}, 1)])
def test_scan_entry(over, want):
    p = filled(_cabi.ScanProblem, B=0, T=3, D=8, N=16, G=1, dtype=1)
    for k, v in over.items():
        setattr(p, k, v)
    assert call("lq_selective_scan_fwd", p) == want


@pytest.mark.parametrize("over,want", [({}, 0), ({"H": 3, "P": 3}, 2), ({"H": 4, "P": 2, "G": 8}, 2), ({"state_dtype": 9}, 4), ({"state": None}, 1),
                                       ({"T": 2}, 2), ({"slots": None, "n_slots": -1}, 2)])
def test_scan_step_entry(over, want):
    p = filled(_cabi.ScanProblem, B=0, T=1, D=8, N=16, G=1, dtype=1, state_dtype=2)
    for k, v in over.items():
        setattr(p, k, v)
    assert call("lq_selective_scan_step", p) == want


@pytest.mark.parametrize("over,want", [({"M": 0}, 0), ({"K": 131072}, 2), ({"N": 0}, 2), ({"x": None}, 1), ({"x": 4097}, 3), ({"w_stride": 40}, 3),
                                       ({"out_dtype": 5}, 4)])
def test_linear_entry(over, want):
    p = filled(_cabi.LinearProblem, M=4, N=8, K=32, x_stride=32, w_stride=32, out_dtype=1)
    for k, v in over.items():
        setattr(p, k, v)
    assert call("lq_int8_linear", p) == want


@pytest.mark.parametrize("over,want", [({"rows": 0}, 0), ({"group": 5}, 2), ({"group": 4}, 4), ({"residual": None}, 1), ({"weight": None}, 1),
                                       ({"scale": None}, 1), ({"codes_stride": 8}, 3), ({"x": None}, 1)])
def test_norm_entry(over, want):
    p = filled(_cabi.NormProblem, rows=2, D=8, group=8, dtype=1, out_dtype=1, x_stride=8, residual_stride=8, codes_stride=16)
    for k, v in over.items():
        setattr(p, k, v)
    assert call("lq_rms_norm", p) == want


def test_cpu_tensors_are_refused():
    from linquant_b200.kernels import layer

    x = torch.zeros(2, 3, 16)
    w = torch.zeros(16, 4)
    for fn in (lambda: layer.short_conv_fwd(x, w), lambda: layer.short_conv_step(x[:, 0], torch.zeros(2, 3, 16), w),
               lambda: layer.selective_scan_fwd(x, x, torch.zeros(16, 4), x.unsqueeze(2), x.unsqueeze(2)),
               lambda: layer.selective_scan_step(torch.zeros(2, 16, 4), x[:, 0], x[:, 0], torch.zeros(16, 4), x[:, :1], x[:, :1]),
               lambda: layer.quantize_rows_fwd(x), lambda: layer.int8_linear_fwd(x, torch.zeros(4, 16, dtype=torch.int8), torch.ones(4)),
               lambda: layer.rms_norm_fwd(x, w[:, 0]), lambda: layer.gated_rms_norm_fwd(x, x, w[:, 0])):
        with pytest.raises(_cabi.LinQuantError):
            fn()
