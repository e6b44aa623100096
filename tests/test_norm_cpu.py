"""layer_norm and rms_norm without a GPU: the argument checks of the functions and of the C entry points."""

from __future__ import annotations

import ctypes

import pytest
import torch

import adambridge_b200 as ab
from adambridge_b200 import native


def test_struct_size_and_declared_arguments(kernels):
    assert kernels._lib.abx_norm_size() == ctypes.sizeof(native.Norm) == 64
    for name in ("abx_norm_forward", "abx_norm_backward", "abx_norm_backward_workspace_bytes"):
        assert getattr(kernels._lib, name).argtypes, name
    assert kernels._lib.abx_norm_backward_workspace_bytes.restype is ctypes.c_size_t


@pytest.mark.parametrize("fn", [ab.layer_norm, ab.rms_norm])
def test_cpu_tensors_and_shapes_are_refused(fn):
    with pytest.raises(ValueError, match="CUDA tensors only"):
        fn(torch.zeros(2, 4))
    for x in (torch.zeros(()), torch.zeros(3, 0)):
        with pytest.raises(ValueError, match="at least one value"):
            fn(x)


def norm(**change):
    n = native.Norm(x=0x10000, w=0x20000, b=0x30000, rows=4, cols=64, x_stride=64, dtype=native.DT_BF16,
                    w_dtype=native.DT_F32, rms=0, eps=1e-5)
    for k, v in change.items():
        setattr(n, k, v)
    return n


@pytest.mark.parametrize("change, code", [
    (dict(rows=-1), -1), (dict(cols=0), -1), (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(rms=1), -1),
    (dict(dtype=native.DT_FP8), -3), (dict(w_dtype=native.DT_F24), -13), (dict(x=None), -2), (dict(x=0x10001), -21),
    (dict(w=0x20002), -21), (dict(b=0x30002), -21)])
def test_c_refusals_come_before_any_launch(kernels, change, code):
    lib, launched = kernels._lib, kernels.launch_count()
    n = norm(**change)
    assert lib.abx_norm_forward(None, ctypes.byref(n), 0x40000, None, None) == code
    assert lib.abx_norm_backward(None, ctypes.byref(n), 0x50000, 64, 0x60000, 0x70000, 0x80000, 0x90000, None, 0xa0000,
                                 1 << 30) == code
    assert kernels.launch_count() == launched


@pytest.mark.parametrize("change, code", [
    (dict(dy=None), -2), (dict(mean=None), -2), (dict(rstd=None), -2), (dict(dy=0x50001), -21), (dict(dx=0x80001), -21),
    (dict(dw=0x90002), -21), (dict(db=0xb0001), -21), (dict(ws=0xa0004), -21), (dict(dx=None, dw=None, db=None), 0)])
def test_c_refusals_of_the_backward_pass(kernels, change, code):
    v = dict(dy=0x50000, mean=0x60000, rstd=0x70000, dx=0x80000, dw=0x90000, db=0xb0000, ws=0xa0000)
    v.update(change)
    n = norm()
    assert kernels._lib.abx_norm_backward(None, ctypes.byref(n), v["dy"], 64, v["mean"], v["rstd"], v["dx"], v["dw"],
                                          v["db"], v["ws"], 1 << 30) == code
    rms = norm(rms=1, b=None)
    assert kernels._lib.abx_norm_backward(None, ctypes.byref(rms), 0x50000, 64, None, 0x70000, None, None, 0xb0000,
                                          0xa0000, 1 << 30) == -1


def test_forward_refusals_and_no_rows(kernels):
    lib = kernels._lib
    n = norm()
    assert lib.abx_norm_forward(None, ctypes.byref(n), None, None, None) == -2
    assert lib.abx_norm_forward(None, ctypes.byref(n), 0x40001, None, None) == -21
    assert lib.abx_norm_forward(None, None, 0x40000, None, None) == -1
    empty = norm(rows=0, x=None)
    assert lib.abx_norm_forward(None, ctypes.byref(empty), 0x40000, None, None) == 0
