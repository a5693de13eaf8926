"""Operators of a residual policy torso over the t8b_layer_norm_* / t8b_linear_* / t8b_gated_* entry
points: layer norm, the linear map with bias, activation and residual, and the gated projection,
each with its gradients.

Arguments are CUDA tensors whose last axis is contiguous; leading axes count as rows and need one
stride between them (a column range of a wider buffer is fine). Matrix operands are bf16 or f16,
both of one type; a bias is fp32 or of that type; norms take fp32 too. Outputs are new tensors. Work is queued
on `stream` (a torch.cuda.Stream; torch's current stream by default), where inputs must be ready,
and outputs and workspaces belong to that stream as torch's own do. A call of the wrong types or
shapes raises ValueError before anything is queued.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import T8B_OK, T8bError

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3, "tanh": 4}

_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch.cuda.current_device
_entries: dict = {}


def _entry(name):
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.lib(), name)
    return fn


def _check(status):
    if status != T8B_OK:
        message = _lib.lib().t8b_last_error().decode()
        if status == _lib.T8B_EINVAL:
            raise ValueError(message)
        raise T8bError(status, message)


class _On:
    """The tensors' device and the stream of a call, current while it allocates and queues."""

    __slots__ = ("index", "stream", "entered")

    def __init__(self, tensor, stream):
        self.index = tensor.get_device()
        if self.index < 0:
            raise ValueError("expected CUDA tensors")
        self.stream = stream

    def __enter__(self):
        self.entered = ()
        if _current_device() != self.index:
            self.entered += (torch.cuda.device(self.index),)
        if self.stream is not None:
            self.entered += (torch.cuda.stream(self.stream),)
        for each in self.entered:
            each.__enter__()
        return _raw_stream(self.index)

    def __exit__(self, *exc):
        for each in reversed(self.entered):
            each.__exit__(*exc)


def _rows(t, name, columns, device, dtype=None):
    """(pointer, rows, row stride) of a tensor of rows of `columns` elements."""
    if t.get_device() != device:
        raise ValueError(f"{name} is on another device")
    if dtype is not None and t.dtype is not dtype:
        raise ValueError(f"{name} is {t.dtype}, expected {dtype}")
    shape = t.shape
    if not shape or shape[-1] != columns:
        raise ValueError(f"{name} has shape {tuple(shape)}, expected rows of {columns}")
    if t.stride(-1) != 1 and columns > 1:
        raise ValueError(f"{name}: the last axis must be contiguous")
    if len(shape) == 2:
        rows = shape[0]
        # a stride that addresses nothing (one row) may be anything
        return t.data_ptr(), rows, t.stride(0) if rows > 1 else columns
    if len(shape) == 1:
        return t.data_ptr(), 1, columns
    rows, step = 1, None
    for size, stride in zip(reversed(shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if step is None:
            step = stride
        elif stride != step * rows:
            raise ValueError(f"{name}: its leading axes have no common row stride")
        rows *= size
    return t.data_ptr(), rows, step if rows > 1 else columns


def _vector(t, name, count, device, dtypes):
    if t is None:
        return 0
    if t.get_device() != device:
        raise ValueError(f"{name} is on another device")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} is {t.dtype}, expected one of {dtypes}")
    if t.shape != (count,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of {count}")
    return t.data_ptr()


def _activation(name):
    try:
        return ACTIVATIONS[name]
    except KeyError:
        raise ValueError(f"activation {name!r}: one of {', '.join(ACTIVATIONS)}") from None


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, out_dtype=None, save: bool = False, stream=None):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last axis, in `out_dtype` (x's by
    default); with `save` also each row's fp32 mean and 1 / sqrt(variance + eps)."""
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if x.dtype not in _TYPES or out_dtype not in _TYPES:
        raise ValueError("layer norm takes and gives fp32, bf16 or f16")
    on = _On(x, stream)
    n = x.shape[-1] if x.dim() else 0
    px, rows, stride = _rows(x, "x", n, on.index)
    first = weight if weight is not None else bias
    kind = (first.dtype,) if first is not None else (torch.float32,)
    if kind[0] not in _TYPES:
        raise ValueError("layer norm parameters are fp32, bf16 or f16")
    pw, pb = _vector(weight, "weight", n, on.index, kind), _vector(bias, "bias", n, on.index, kind)
    with on as raw:
        y = x.new_empty(x.shape, dtype=out_dtype)
        mean = rstd = None
        if save:
            mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
            rstd = x.new_empty(x.shape[:-1], dtype=torch.float32)
        _check(_entry("t8b_layer_norm_forward")(
            px, _TYPES[x.dtype], stride, pw, pb, _TYPES[kind[0]], eps, rows, n, y.data_ptr(), _TYPES[out_dtype], n,
            mean.data_ptr() if save else 0, rstd.data_ptr() if save else 0, raw))
    return (y, mean, rstd) if save else y


def layer_norm_backward(dy, x, weight, bias, mean, rstd, residual_gradient=None, stream=None):
    """(dx, dweight, dbias) of layer_norm from dy and what its `save` gave. `residual_gradient` (of
    x's type and shape) is added to dx. dweight and dbias are None where weight and bias are."""
    if x.dtype not in _TYPES or dy.dtype not in _TYPES:
        raise ValueError("layer norm takes fp32, bf16 or f16")
    on = _On(x, stream)
    device, n = on.index, x.shape[-1] if x.dim() else 0
    px, rows, x_stride = _rows(x, "x", n, device)
    if dy.shape != x.shape:
        raise ValueError(f"dy has shape {tuple(dy.shape)}, x {tuple(x.shape)}")
    pdy, _, dy_stride = _rows(dy, "dy", n, device)
    pr, r_stride = 0, n
    if residual_gradient is not None:
        if residual_gradient.shape != x.shape:
            raise ValueError(f"residual_gradient has shape {tuple(residual_gradient.shape)}, x {tuple(x.shape)}")
        pr, _, r_stride = _rows(residual_gradient, "residual_gradient", n, device, x.dtype)
    first = weight if weight is not None else bias
    kind = (first.dtype,) if first is not None else (torch.float32,)
    if kind[0] not in _TYPES:
        raise ValueError("layer norm parameters are fp32, bf16 or f16")
    pw = _vector(weight, "weight", n, device, kind)
    _vector(bias, "bias", n, device, kind)
    if mean.numel() != rows or rstd.numel() != rows:
        raise ValueError("mean and rstd must have one value a row")
    statistics = [_vector(v.reshape(-1) if v.dim() != 1 else v, name, rows, device, (torch.float32,))
                  for v, name in ((mean, "mean"), (rstd, "rstd"))]
    with on as raw:
        dx = x.new_empty(x.shape, dtype=x.dtype)
        dweight = torch.empty_like(weight) if weight is not None else None
        dbias = torch.empty_like(bias) if bias is not None else None
        size = _entry("t8b_layer_norm_workspace")(rows, n) if first is not None else 0
        workspace = x.new_empty(size, dtype=torch.uint8) if size else None
        _check(_entry("t8b_layer_norm_backward")(
            pdy, _TYPES[dy.dtype], dy_stride, px, _TYPES[x.dtype], x_stride, pw, _TYPES[kind[0]], *statistics, pr,
            r_stride, rows, n, dx.data_ptr(), n, dweight.data_ptr() if dweight is not None else 0,
            dbias.data_ptr() if dbias is not None else 0, workspace.data_ptr() if size else 0, size, raw))
    return dx, dweight, dbias


def _operands(x, weight, parts, stream):
    """Checks shared by the linear map (parts = 1) and the gated projection (2)."""
    kind = x.dtype
    if kind is not torch.bfloat16 and kind is not torch.float16:
        raise ValueError(f"x is {kind}: matrix operands are bf16 or f16")
    if weight.dim() != 2 or weight.shape[0] % parts:
        raise ValueError(f"weight has shape {tuple(weight.shape)}, expected [{'2 out' if parts == 2 else 'out'}][in]")
    on = _On(x, stream)
    columns, n = weight.shape
    px, rows, x_stride = _rows(x, "x", n, on.index)
    pw, _, w_stride = _rows(weight, "weight", n, on.index, kind)
    return on, kind, columns, n, px, rows, x_stride, pw, w_stride


def _forward_workspace(name, px, x_stride, pw, w_stride, rows, n, out, x):
    """Room for packed copies where the rows of x or weight start off 16-byte boundaries."""
    if not ((px | pw) & 15 or (x_stride | w_stride) & 7) or rows == 0:
        return None, 0, 0
    size = _entry(name)(rows, n, out, 0)
    workspace = x.new_empty(size, dtype=torch.uint8)
    return workspace, workspace.data_ptr(), size


def linear(x, weight, bias=None, activation: str = "none", residual=None, out_dtype=None, save: bool = False,
           stream=None):
    """activation(x weight^T + bias) + residual in `out_dtype` (x's type by default, or fp32; the
    residual has it too); with `save` also pre = x weight^T + bias in x's type, for the gradient.
    activation: "none", "relu", "gelu" (z Phi(z)), "silu" or "tanh"."""
    on, kind, out, n, px, rows, x_stride, pw, w_stride = _operands(x, weight, 1, stream)
    act = _activation(activation)
    out_dtype = kind if out_dtype is None else out_dtype
    if out_dtype is not kind and out_dtype is not torch.float32:
        raise ValueError(f"out_dtype {out_dtype}: fp32 or x's type")
    pb = _vector(bias, "bias", out, on.index, (torch.float32, kind))
    shape = (*x.shape[:-1], out)
    pr, r_stride = 0, out
    if residual is not None:
        if residual.shape != shape:
            raise ValueError(f"residual has shape {tuple(residual.shape)}, expected {shape}")
        pr, _, r_stride = _rows(residual, "residual", out, on.index, out_dtype)
    with on as raw:
        y = x.new_empty(shape, dtype=out_dtype)
        pre = x.new_empty(shape, dtype=kind) if save else None
        workspace, pws, size = _forward_workspace("t8b_linear_workspace", px, x_stride, pw, w_stride, rows, n, out, x)
        _check(_entry("t8b_linear_forward")(
            _TYPES[kind], px, x_stride, pw, w_stride, pb, _TYPES[bias.dtype] if bias is not None else 0, act, pr,
            r_stride, rows, n, out, y.data_ptr(), _TYPES[out_dtype], out, pre.data_ptr() if save else 0, out, pws,
            size, raw))
    return (y, pre) if save else y


def gated(x, weight, bias=None, activation: str = "silu", save: bool = False, stream=None):
    """activation(gate) * up with [gate | up] = x weight^T + bias in one kernel: weight [2 out][in]
    and bias [2 out] hold the gate's rows first. With `save` also [gate | up], for the gradient."""
    on, kind, columns, n, px, rows, x_stride, pw, w_stride = _operands(x, weight, 2, stream)
    act, out = _activation(activation), columns // 2
    pb = _vector(bias, "bias", columns, on.index, (torch.float32, kind))
    with on as raw:
        h = x.new_empty((*x.shape[:-1], out), dtype=kind)
        pre = x.new_empty((*x.shape[:-1], columns), dtype=kind) if save else None
        workspace, pws, size = _forward_workspace("t8b_gated_workspace", px, x_stride, pw, w_stride, rows, n, out, x)
        _check(_entry("t8b_gated_forward")(
            _TYPES[kind], px, x_stride, pw, w_stride, pb, _TYPES[bias.dtype] if bias is not None else 0, act, rows, n,
            out, h.data_ptr(), out, pre.data_ptr() if save else 0, columns, pws, size, raw))
    return (h, pre) if save else h


def _backward(entry, query, parts, dy, x, weight, bias, pre, activation, input_gradient, stream):
    on, kind, columns, n, px, rows, x_stride, pw, w_stride = _operands(x, weight, parts, stream)
    act, out = _activation(activation), columns // parts
    if dy.shape != (*x.shape[:-1], out):
        raise ValueError(f"the output's gradient has shape {tuple(dy.shape)}, expected {(*x.shape[:-1], out)}")
    pdy, _, dy_stride = _rows(dy, "the output's gradient", out, on.index, kind)
    pp, p_stride = 0, columns
    if parts == 2 or act:
        if pre is None:
            raise ValueError("pre (what the forward pass's `save` gave) is needed")
        if pre.shape != (*x.shape[:-1], columns):
            raise ValueError(f"pre has shape {tuple(pre.shape)}, expected {(*x.shape[:-1], columns)}")
        pp, _, p_stride = _rows(pre, "pre", columns, on.index, kind)
    _vector(bias, "bias", columns, on.index, (torch.float32, kind))
    with on as raw:
        dx = x.new_empty(x.shape, dtype=kind) if input_gradient else None
        dweight = x.new_empty((columns, n), dtype=kind)
        dbias = torch.empty_like(bias) if bias is not None else None
        size = _entry(query)(rows, n, out, 1)
        workspace = x.new_empty(size, dtype=torch.uint8) if size else None
        _check(_entry(entry)(
            _TYPES[kind], pdy, dy_stride, px, x_stride, pw, w_stride, pp, p_stride,
            _TYPES[bias.dtype] if bias is not None else 0, act, rows, n, out, dx.data_ptr() if input_gradient else 0,
            n, dweight.data_ptr(), n, dbias.data_ptr() if dbias is not None else 0,
            workspace.data_ptr() if size else 0, size, raw))
    return dx, dweight, dbias


def linear_backward(dy, x, weight, bias=None, pre=None, activation: str = "none", input_gradient: bool = True,
                    stream=None):
    """(dx, dweight, dbias) of linear from its output's gradient (which is the residual's gradient
    too) and `pre`, which an activation needs. dx is None without `input_gradient` (a first layer
    has no use for it), dbias without a bias."""
    return _backward("t8b_linear_backward", "t8b_linear_workspace", 1, dy, x, weight, bias, pre, activation,
                     input_gradient, stream)


def gated_backward(dh, x, weight, bias=None, pre=None, activation: str = "silu", input_gradient: bool = True,
                   stream=None):
    """(dx, dweight, dbias) of gated from its output's gradient and `pre`."""
    return _backward("t8b_gated_backward", "t8b_gated_workspace", 2, dh, x, weight, bias, pre, activation,
                     input_gradient, stream)


def status(stream=None):
    """Waits for `stream` (torch's current one) and raises T8bError if a wait inside an operator's
    kernel ran out of its limit since the last call: that call's outputs are not valid."""
    raw = stream.cuda_stream if stream is not None else torch.cuda.current_stream().cuda_stream
    _check(_entry("t8b_operators_status")(raw))
