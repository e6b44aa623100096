"""Layer norm and RMS norm over the last axis, with their backward passes, on libabx's kernels.

A norm is bound by memory: forward reads ``x`` once and writes ``y`` once, backward reads ``x`` and the gradient once
and writes ``dx`` once, with the rows' statistics (fp32) kept in between.  The gradients of the weight and the bias --
what an optimizer of this package updates -- are summed over the rows in fp32 in a fixed order, so the same input gives
the same bits, and rounded once.  Nothing synchronizes with the host; a training step that uses them can be captured
into a CUDA graph together with :class:`~adambridge_b200.graph_adamw.GraphAdamW`.
"""

from __future__ import annotations

import torch

from . import native

__all__ = ["layer_norm", "rms_norm"]


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis of a CUDA tensor, ``var`` the mean square
    deviation.

    ``x`` is float32 or bfloat16, of any shape and strides (rows that are not evenly spaced, or not contiguous, are
    copied first); ``weight`` and ``bias``, each optional, are float32 or bfloat16 vectors of one dtype, which need not be
    ``x``'s.  All arithmetic is fp32, so a row whose sum, or whose sum of squared deviations, passes the range of fp32 gives
    what elementary fp32 operations give (NaN, or a deviation of infinity); ``y`` and the gradients are rounded once to ``x``'s and the weight's dtype.  Runs on
    the current stream of ``x``'s device.  Gradients are those of first order and reverse mode: differentiating
    them raises, and so do forward-mode tangents and traces (``torch.jit.trace``, ``make_fx``, fake tensors)."""
    return native.torch_ops().norm(x, weight, bias, eps, False)


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """``x / sqrt(mean(x * x) + eps) * weight`` over the last axis of a CUDA tensor; otherwise as :func:`layer_norm`."""
    return native.torch_ops().norm(x, weight, None, eps, True)
