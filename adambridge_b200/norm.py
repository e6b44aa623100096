"""Layer norm and RMS norm over the last axis, with their backward passes, on libabx's kernels.

A norm is bound by memory: forward reads ``x`` once and writes ``y`` once, backward reads ``x`` and the gradient once
and writes ``dx`` once, with the rows' statistics (fp32) kept in between.  The gradients of the weight and the bias --
what an optimizer of this package updates -- are summed over the rows in fp32 in a fixed order, so the same input gives
the same bits, and rounded once.  Nothing synchronizes with the host; a training step that uses them can be captured
into a CUDA graph together with :class:`~adambridge_b200.graph_adamw.GraphAdamW`.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import native

__all__ = ["layer_norm", "rms_norm"]

_TYPES = (torch.float32, torch.bfloat16)


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """(tensor, rows, elements between rows): ``t`` itself where its rows lie evenly spaced, else a contiguous copy."""
    cols = t.shape[-1]
    if not t.is_contiguous():
        try:
            rows = t.view(-1, cols)
            if cols > 1 and rows.stride(1) != 1:
                raise RuntimeError
            return t, rows.shape[0], rows.stride(0) if rows.shape[0] > 1 else cols
        except RuntimeError:
            t = t.contiguous()
    return t, t.numel() // cols, cols


def _check(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, eps: float) -> None:
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"a norm needs at least one value along the last axis, got the shape {tuple(x.shape)}")
    if not x.is_cuda:
        raise ValueError("adambridge_b200's norms run on CUDA tensors only")
    if x.dtype not in _TYPES:
        raise TypeError(f"x must be float32 or bfloat16, got {x.dtype}")
    if not eps >= 0.0:
        raise ValueError(f"invalid epsilon: {eps}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.shape != x.shape[-1:]:
            raise ValueError(f"{name} has the shape {tuple(t.shape)}, the last axis {x.shape[-1]} values")
        if t.dtype not in _TYPES:
            raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must have one dtype, got {weight.dtype} and {bias.dtype}")


def _describe(x, rows, stride, weight, bias, eps, rms) -> native.Norm:
    either = weight if weight is not None else bias
    return native.Norm(x.data_ptr(), None if weight is None else weight.data_ptr(),
                       None if bias is None else bias.data_ptr(), rows, x.shape[-1], stride,
                       native.dtype_code_of(x.dtype), native.dtype_code_of(either.dtype if either is not None else x.dtype),
                       rms, eps)


def _forward(x, weight, bias, eps, rms, keep):
    """(y, x as the kernels read it, statistics or None): the statistics are rstd, then the mean, one fp32 per row."""
    xr, rows, stride = _rows(x)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    with torch.cuda.device(x.device):
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        stats = torch.empty((1 if rms else 2, rows), dtype=torch.float32, device=x.device) if keep else None
        native.load().norm_forward(None, _describe(xr, rows, stride, weight, bias, eps, rms), y, stats)
    return y, xr, stats


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, rms):
        y, xr, stats = _forward(x, weight, bias, eps, rms, True)
        ctx.save_for_backward(xr, weight, bias, stats)
        ctx.eps, ctx.rms = eps, rms
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        xr, rows, stride = _rows(x)
        dyr, _, dy_stride = _rows(dy)
        with torch.cuda.device(x.device):
            w = None if weight is None else weight.contiguous()
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if want_x else None
            dw = torch.empty_like(weight, memory_format=torch.contiguous_format) if want_w else None
            db = torch.empty_like(bias, memory_format=torch.contiguous_format) if want_b else None
            native.load().norm_backward(None, _describe(xr, rows, stride, w, None if bias is None else bias.contiguous(),
                                                        ctx.eps, ctx.rms), dyr, dy_stride, stats, dx, dw, db)
        return dx, dw, db, None, None


def _norm(x, weight, bias, eps, rms):
    eps = float(eps)
    _check(x, weight, bias, eps)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _Norm.apply(x, weight, bias, eps, rms)
    return _forward(x, weight, bias, eps, rms, False)[0]


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis of a CUDA tensor, ``var`` the mean square
    deviation.

    ``x`` is float32 or bfloat16, of any shape and strides (rows that are not evenly spaced, or not contiguous, are
    copied first); ``weight`` and ``bias``, each optional, are float32 or bfloat16 vectors of one dtype, which need not be
    ``x``'s.  All arithmetic is fp32; ``y`` and the gradients are rounded once to ``x``'s and the weight's dtype.  Runs on
    the current stream of ``x``'s device.  Gradients are those of first order."""
    return _norm(x, weight, bias, eps, False)


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """``x / sqrt(mean(x * x) + eps) * weight`` over the last axis of a CUDA tensor; otherwise as :func:`layer_norm`."""
    return _norm(x, weight, None, eps, True)
