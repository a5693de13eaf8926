"""Operators of a residual policy torso over the t8b_layer_norm_* / t8b_linear_* / t8b_gated_* entry
points (layer norm, the linear map with bias, activation and residual, and the gated projection) and
of a policy with memory over t8b_causal_conv_* / t8b_selective_scan_* / t8b_policy_loss (the short causal
convolution, the selective scan, the clipped policy loss), each with its gradients.

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
    "linear_forward", "linear_backward", "gated_workspace", "gated_forward", "gated_backward", "causal_conv_forward",
    "causal_conv_workspace", "causal_conv_backward", "causal_conv_step", "selective_scan_saved",
    "selective_scan_workspace", "selective_scan_forward", "selective_scan_backward", "selective_scan_step",
    "policy_loss")))


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


# ---------------------------------------------------------------- a policy with memory
# Sequences are tensors [sequences][steps][channels] in any order of the first two axes (a rollout's
# [step][fight] data as data.transpose(0, 1)); outputs lie in x's order. `reset` [sequences][steps] (bool or
# uint8) marks the steps at which a new round begins: nothing before such a step, the initial state included,
# reaches it. `lengths` [sequences] (int32) ends sequences early: what lies past a sequence's length is not
# read, outputs and gradients there are 0, and its final state is the one after its last step.


def causal_conv(x, weight, bias=None, activation: str = "none", state=None, reset=None, lengths=None,
                final: bool = False, stream=None):
    """activation(bias + sum over j of weight[:, width - 1 - j] x[t - j]), one filter of 2 to 4 taps a channel
    (weight [channels][width]; weight and bias fp32 or of x's type). `state` [sequences][width - 1][channels]
    of x's type holds the inputs before the first step, oldest first (zeros by default); with `final` also
    the last inputs, which are the next call's state."""
    if stream is not None:
        with _on(stream, x):
            return _operators.causal_conv(x, weight, bias, activation, state, reset, lengths, final)
    return _operators.causal_conv(x, weight, bias, activation, state, reset, lengths, final)


def causal_conv_backward(dy, x, weight, bias=None, activation: str = "none", state=None, reset=None, lengths=None,
                         dfinal=None, stream=None):
    """(dx, dweight, dbias, dstate) of causal_conv from its output's gradient and, where it is given, the
    final state's. dbias and dstate are None where bias and state are."""
    if stream is not None:
        with _on(stream, x):
            return _operators.causal_conv_backward(dy, x, weight, bias, activation, state, reset, lengths, dfinal)
    return _operators.causal_conv_backward(dy, x, weight, bias, activation, state, reset, lengths, dfinal)


def causal_conv_step(x, weight, bias, state, activation: str = "none", reset=None, stream=None):
    """One step of causal_conv for every sequence: x [sequences][channels], reset [sequences]. `state` is moved
    on in place."""
    if stream is not None:
        with _on(stream, x):
            return _operators.causal_conv_step(x, weight, bias, state, activation, reset)
    return _operators.causal_conv_step(x, weight, bias, state, activation, reset)


def selective_scan(u, delta, a, b, c, d=None, z=None, delta_bias=None, softplus: bool = True, state=None, reset=None,
                   lengths=None, final: bool = False, save: bool = False, stream=None):
    """The selective state space scan: with size = softplus(delta + delta_bias) (or without the softplus),
    h = exp(size a) h + size u b and y = (sum over states of c h + d u) silu(z).

    u, delta and z [sequences][steps][channels], b and c [sequences][steps][states] or [sequences][steps]
    [groups][states] (a group serves channels / groups channels in a row), all of one type; a [channels]
    [states] (up to 64), d and delta_bias [channels], and `state` [sequences][channels][states] (zeros by
    default) fp32. Returns y, then with `final` the state after the last step, then with `save` what the
    backward pass needs."""
    if stream is not None:
        with _on(stream, u):
            return _operators.selective_scan(u, delta, a, b, c, d, z, delta_bias, softplus, state, reset, lengths, final,
                                             save)
    return _operators.selective_scan(u, delta, a, b, c, d, z, delta_bias, softplus, state, reset, lengths, final, save)


def selective_scan_backward(dy, u, delta, a, b, c, saved, d=None, z=None, delta_bias=None, softplus: bool = True,
                            state=None, reset=None, lengths=None, dfinal=None, stream=None):
    """(du, ddelta, da, db, dc, dd, dz, ddelta_bias, dstate) of selective_scan from its output's gradient, what
    its `save` gave and, where it is given, the final state's gradient; the other arguments as they were. dd,
    dz, ddelta_bias and dstate are None where d, z, delta_bias and state are."""
    if stream is not None:
        with _on(stream, u):
            return _operators.selective_scan_backward(dy, u, delta, a, b, c, saved, d, z, delta_bias, softplus, state,
                                                      reset, lengths, dfinal)
    return _operators.selective_scan_backward(dy, u, delta, a, b, c, saved, d, z, delta_bias, softplus, state, reset,
                                              lengths, dfinal)


def selective_scan_step(u, delta, a, b, c, state, d=None, z=None, delta_bias=None, softplus: bool = True, reset=None,
                        stream=None):
    """One step of selective_scan for every sequence: u, delta and z [sequences][channels], b and c
    [sequences][states] or [sequences][groups][states], reset [sequences]. `state` is moved on in place."""
    if stream is not None:
        with _on(stream, u):
            return _operators.selective_scan_step(u, delta, a, b, c, state, d, z, delta_bias, softplus, reset)
    return _operators.selective_scan_step(u, delta, a, b, c, state, d, z, delta_bias, softplus, reset)


def policy_loss(logits, actions, old_log_probabilities, advantages, mask=None, reference=None, weights=None,
                clip: float = 0.2, clip_high=None, kl: float = 0.0, entropy: float = 0.0, gradient: bool = True,
                stream=None):
    """(loss, log_probabilities, entropies, divergences), fp32 values of each row, of the clipped policy loss
    -min(r advantage, min(max(r, 1 - clip), 1 + clip_high) advantage) + kl divergence - entropy H with r =
    exp(log_probability - old), and with `gradient` also dlogits, the gradient of the sum over rows of
    weight loss (weights fp32; by default 1 / rows each, the mean).

    logits [...][n] of any type; actions (int64), old_log_probabilities and advantages (fp32) one a row. mask:
    which logits are legal, bool or uint8 [...][n], or int32 [...][ceil(n / 32)] with one bit each as the
    simulator packs them. reference: a frozen policy's logits (of the logits' type and shape: the
    divergence is the exact one over the legal actions) or its log-probabilities of the actions (fp32, one
    a row: exp(e) - e - 1 with e = reference - log_probability). A row whose action is not a legal one (-1, say:
    padding) gives 0 everywhere. clip_high is `clip` by default. The rows of dlogits start on 16 bytes: it is a
    column range of a wider buffer where n does not do that by itself."""
    if stream is not None:
        with _on(stream, logits):
            return _operators.policy_loss(logits, actions, old_log_probabilities, advantages, mask, reference, weights,
                                          clip, clip_high, kl, entropy, gradient)
    return _operators.policy_loss(logits, actions, old_log_probabilities, advantages, mask, reference, weights, clip,
                                  clip_high, kl, entropy, gradient)


def status(stream=None, device=None):
    """Waits for `stream` (by default torch's current one of `device`, or of the current device) and
    raises T8bError if a wait inside an operator's kernel ran out of its limit on that device since the
    last call: that call's outputs are not valid. Each device keeps its own record."""
    with torch.cuda.device(stream.device if stream is not None else device):
        raw = (stream if stream is not None else torch.cuda.current_stream()).cuda_stream
        result = _lib.lib().t8b_operators_status(raw)
    if result != T8B_OK:
        raise T8bError(result, _lib.lib().t8b_last_error().decode())
