"""GraphAdamW without a GPU: argument checks of the class and of the C entry points, struct layouts, and the bindings."""

from __future__ import annotations

import ctypes

import pytest
import torch

import adambridge_b200 as ab
from adambridge_b200 import native


def test_struct_sizes(kernels):
    assert kernels._lib.abx_graph_tensor_size() == 8 * native.GRAPH_TENSOR_WORDS == 80
    assert kernels._lib.abx_graph_step_size() == ctypes.sizeof(native.GraphStep) == 88


def test_pointer_arguments_are_declared(kernels):
    """Without argtypes ctypes passes a Python integer as a 32-bit int and cuts a device address."""
    for name in ("abx_graph_adamw", "abx_i8_decode", "abx_i8_encode"):
        assert getattr(kernels._lib, name).argtypes, name


@pytest.mark.parametrize("kwargs, message", [
    (dict(precision="fp8"), "precision"), (dict(lr=-1.0), "learning rate"), (dict(betas=(1.0, 0.9)), "betas"),
    (dict(betas=(0.9, -0.1)), "betas"), (dict(eps=-1e-8), "epsilon"), (dict(weight_decay=-0.1), "weight_decay"),
    (dict(max_ctas=-1), "max_ctas"), (dict(lr=float("nan")), "learning rate")])
def test_constructor_refusals(kwargs, message):
    with pytest.raises(ValueError, match=message):
        ab.GraphAdamW([torch.nn.Parameter(torch.zeros(4))], **kwargs)


def test_lr_tensor_refusals():
    for lr in (torch.zeros(2), torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(TypeError, match="lr must be"):
            ab.GraphAdamW([torch.nn.Parameter(torch.zeros(4))], lr=lr)


def test_group_refusals_leave_no_group():
    opt = ab.GraphAdamW([torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(ValueError, match="at least one parameter"):
        opt.add_param_group({"params": []})
    twice = torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError, match="twice"), pytest.warns(UserWarning):   # torch only warns
        opt.add_param_group({"params": [twice, twice]})
    with pytest.raises(ValueError, match="betas"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(4))], "betas": (2.0, 0.9)})
    assert len(opt.param_groups) == 1


def test_cpu_parameters_are_refused():
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.zeros(4)
    with pytest.raises(ValueError, match="CUDA parameters only"):
        ab.GraphAdamW([p]).step()


def test_norm_type_and_no_gradients():
    opt = ab.GraphAdamW([torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(ValueError, match="L2"):
        opt.clip_grad_norm_(1.0, norm_type=1.0)
    assert float(opt.clip_grad_norm_(1.0)) == 0.0


def _tensor(**change):
    row = dict(w=0x1000, g=0x2000, master=0x3000, m=0x4000, v=0x5000, m_scale=0x6000, v_scale=0x7000, step=0x8000, n=256,
               index=0, dtype=native.DT_BF16)
    row.update(change)
    return torch.tensor([[row[k] for k in ("w", "g", "master", "m", "v", "m_scale", "v_scale", "step", "n")]
                         + [row["index"] | row["dtype"] << 32]], dtype=torch.int64)


def _shared(**change):
    s = native.GraphStep(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, moments=native.DT_I8, stochastic=1)
    for k, v in change.items():
        setattr(s, k, v)
    return s


def _call(kernels, tensor, shared, n=1, ticket=0x9000, max_ctas=0):
    return kernels._lib.abx_graph_adamw(None, tensor.data_ptr(), n, ctypes.byref(shared), ticket, max_ctas)


@pytest.mark.parametrize("tensor, shared, code", [
    (dict(n=-1), {}, -1), (dict(index=0x80000000), {}, -1), (dict(dtype=native.DT_FP8), {}, -3),
    (dict(w=0), {}, -2), (dict(g=0), {}, -2), (dict(m=0), {}, -2), (dict(v=0), {}, -2), (dict(step=0), {}, -2),
    (dict(master=0), {}, -2), (dict(m_scale=0), {}, -7), (dict(v_scale=0), {}, -7),
    (dict(w=0x1001), {}, -21), (dict(g=0x2001), {}, -21), (dict(m=0x4008), {}, -21), (dict(v=0x5004), {}, -21),
    (dict(master=0x3004), {}, -21), (dict(step=0x8004), {}, -21), (dict(m_scale=0x6002), {}, -21),
    (dict(dtype=native.DT_F32, w=0x1002), {}, -21),
    ({}, dict(moments=native.DT_FP8), -4), ({}, dict(beta1=1.0), -1), ({}, dict(beta2=float("nan")), -1),
    ({}, dict(lr_ptr=0xa004, lr_f64=1), -21), ({}, dict(g_scale=0xa002), -21), ({}, dict(skip=0xa001), -21),
    ({}, dict(norm=0xa003), -21)])
def test_c_refusals_come_before_any_launch(kernels, tensor, shared, code):
    launched = kernels.launch_count()
    assert _call(kernels, _tensor(**tensor), _shared(**shared)) == code
    assert kernels.launch_count() == launched


def test_c_refusals_of_the_call(kernels):
    assert _call(kernels, _tensor(), _shared(), n=-1) == -1
    assert _call(kernels, _tensor(), _shared(), ticket=None) == -1
    assert _call(kernels, _tensor(), _shared(), ticket=0x9002) == -21
    assert _call(kernels, _tensor(), _shared(), max_ctas=-1) == -1
    assert _call(kernels, _tensor(), _shared(), n=0) == 0
    assert _call(kernels, _tensor(n=0), _shared()) == 0          # an empty tensor is left out


def test_i8_refusals(kernels):
    decode, encode = kernels._lib.abx_i8_decode, kernels._lib.abx_i8_encode
    assert decode(None, 0x1000, 0x2000, 0x3000, -1, 0) == -1 == encode(None, 0x3000, 0x1000, 0x2000, 4, 2)
    assert decode(None, None, 0x2000, 0x3000, 4, 0) == -2 == encode(None, None, 0x1000, 0x2000, 4, 1)
    assert decode(None, 0x1000, None, 0x3000, 4, 0) == -7
    assert decode(None, 0x1004, 0x2000, 0x3000, 4, 0) == -21 == encode(None, 0x3002, 0x1000, 0x2000, 4, 1)
    assert decode(None, None, None, None, 0, 0) == 0
