"""Operators of a residual policy torso over the t8b_layer_norm_* / t8b_linear_* / t8b_gated_* entry
points: layer norm, the linear map with bias, activation and residual, and the gated projection,
each with its gradients.

Arguments are CUDA tensors whose last axis is contiguous; leading axes count as rows and need one
stride between them (a column range of a wider buffer is fine). Matrix operands are bf16 or f16,
both of one type; a bias is fp32 or of that type; norms take fp32 too. Outputs are new tensors. Work
is queued on `stream` (a torch.cuda.Stream of the tensors' device; torch's current stream by
default), where inputs must be ready, and outputs and workspaces belong to that stream as torch's
own do. A call of the wrong types or shapes raises ValueError before anything is queued. Nothing is
recorded for automatic differentiation: the gradients are the *_backward functions.

The checks and allocations are the module _operators (bindings/operators.cpp, built by build.py).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import T8B_OK, T8bError
from . import _operators

ACTIVATIONS = ("none", "relu", "gelu", "silu", "tanh")

_operators.bind(T8bError, torch.OutOfMemoryError, *(C.cast(getattr(_lib.lib(), "t8b_" + name), C.c_void_p).value for name in (
    "last_error", "layer_norm_forward", "layer_norm_workspace", "layer_norm_backward", "linear_workspace",
    "linear_forward", "linear_backward", "gated_workspace", "gated_forward", "gated_backward")))


def _on(stream, x):
    """The context in which a call on `stream` is queued; its kernels run where x is."""
    if isinstance(x, torch.Tensor) and x.device != stream.device:
        raise ValueError(f"the stream is on {stream.device}, x on {x.device}")
    return torch.cuda.stream(stream)


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, out_dtype=None, save: bool = False, stream=None):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last axis, in `out_dtype` (x's by
    default); with `save` also each row's fp32 mean and 1 / sqrt(variance + eps)."""
    if stream is not None:
        with _on(stream, x):
            return _operators.layer_norm(x, weight, bias, eps, out_dtype, save)
    return _operators.layer_norm(x, weight, bias, eps, out_dtype, save)


def layer_norm_backward(dy, x, weight, bias, mean, rstd, residual_gradient=None, stream=None):
    """(dx, dweight, dbias) of layer_norm from dy and what its `save` gave. `residual_gradient` (of
    x's type and shape) is added to dx. dweight and dbias are None where weight and bias are."""
    if stream is not None:
        with _on(stream, x):
            return _operators.layer_norm_backward(dy, x, weight, bias, mean, rstd, residual_gradient)
    return _operators.layer_norm_backward(dy, x, weight, bias, mean, rstd, residual_gradient)


def linear(x, weight, bias=None, activation: str = "none", residual=None, out_dtype=None, save: bool = False,
           stream=None):
    """activation(x weight^T + bias) + residual in `out_dtype` (x's type by default, or fp32; the
    residual has it too); with `save` also pre = x weight^T + bias in x's type, for the gradient.
    activation: "none", "relu", "gelu" (z Phi(z)), "silu" or "tanh"."""
    if stream is not None:
        with _on(stream, x):
            return _operators.linear(x, weight, bias, activation, residual, out_dtype, save)
    return _operators.linear(x, weight, bias, activation, residual, out_dtype, save)


def linear_backward(dy, x, weight, bias=None, pre=None, activation: str = "none", input_gradient: bool = True,
                    stream=None):
    """(dx, dweight, dbias) of linear from its output's gradient (which is the residual's gradient
    too) and `pre`, which an activation needs. dx is None without `input_gradient` (a first layer
    has no use for it), dbias without a bias."""
    if stream is not None:
        with _on(stream, x):
            return _operators.linear_backward(dy, x, weight, bias, pre, activation, input_gradient)
    return _operators.linear_backward(dy, x, weight, bias, pre, activation, input_gradient)


def gated(x, weight, bias=None, activation: str = "silu", save: bool = False, stream=None):
    """activation(gate) * up with [gate | up] = x weight^T + bias in one kernel: weight [2 out][in]
    and bias [2 out] hold the gate's rows first. With `save` also [gate | up], for the gradient."""
    if stream is not None:
        with _on(stream, x):
            return _operators.gated(x, weight, bias, activation, save)
    return _operators.gated(x, weight, bias, activation, save)


def gated_backward(dh, x, weight, bias=None, pre=None, activation: str = "silu", input_gradient: bool = True,
                   stream=None):
    """(dx, dweight, dbias) of gated from its output's gradient and `pre`."""
    if stream is not None:
        with _on(stream, x):
            return _operators.gated_backward(dh, x, weight, bias, pre, activation, input_gradient)
    return _operators.gated_backward(dh, x, weight, bias, pre, activation, input_gradient)


def status(stream=None, device=None):
    """Waits for `stream` (by default torch's current one of `device`, or of the current device) and
    raises T8bError if a wait inside an operator's kernel ran out of its limit on that device since the
    last call: that call's outputs are not valid. Each device keeps its own record."""
    with torch.cuda.device(stream.device if stream is not None else device):
        raw = (stream if stream is not None else torch.cuda.current_stream()).cuda_stream
        result = _lib.lib().t8b_operators_status(raw)
    if result != T8B_OK:
        raise T8bError(result, _lib.lib().t8b_last_error().decode())
