"""act(x W^T + b) + r over the pixels of a feature image (gs3d_linear_fwd,
gs3d_linear_bwd) and its first-order autograd."""

import ctypes
from typing import Any

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from ..runtime import abi, native
from ._common import (DTYPES, activation_code, check_checkpoint, check_input, check_like, launch, recorded, rows_of,
                      scratch)
from .activations import QuantizedActivations, empty_quantized


def _forward(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, activation: int,
             quantized: QuantizedActivations | None) -> tuple[Tensor, Tensor, int, Tensor, Tensor | None]:
    """(result, x as rows, their stride, weight, bias), the latter as the
    kernels read them; where `quantized` is given x's 8-bit form goes there."""
    outer, inner = weight.shape
    y = torch.empty(x.shape[:-1] + (outer,), dtype=x.dtype, device=x.device)
    rows, x_stride = rows_of(x)
    weight = weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    a = abi.LinearArgs()
    a.rows, a.inner, a.outer = x.numel() // inner, inner, outer
    a.dtype, a.activation = DTYPES[x.dtype], activation
    a.x, a.x_stride = native.ptr(rows), x_stride
    a.weight, a.bias, a.y = native.ptr(weight), native.ptr(bias), native.ptr(y)
    if residual is not None:
        residual, a.residual_stride = rows_of(residual)
        a.residual = native.ptr(residual)
    if quantized is not None:
        a.codes, a.scales = native.ptr(quantized.codes), native.ptr(quantized.scales)
    if a.rows:
        nbytes = native.query("gs3d_linear_fwd_scratch_bytes", a.rows, inner, outer, a.dtype)
        work = scratch(nbytes, x.device) if nbytes else None
        launch("gs3d_linear_fwd", ctypes.byref(a), x.device, native.ptr(work), nbytes)
    return y, rows, x_stride, weight, bias


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, activation: int,
                checkpoint: str | None) -> Tensor:
        # The input is needed for the weight's gradient and for the slope of an
        # activation; without either it is not kept.
        save = any(ctx.needs_input_grad[:3])
        keep = save and (activation != abi.ACT_NONE or ctx.needs_input_grad[1])
        quantized = empty_quantized(x) if keep and checkpoint is not None else None
        y, rows, x_stride, weight, bias = _forward(x, weight, bias, residual, activation, quantized)
        if save:
            kept: tuple[Tensor | None, ...] = (rows if keep else None, None, None)
            if quantized is not None:
                kept = (None, quantized.codes, quantized.scales)
            ctx.save_for_backward(*kept, weight, bias)
            ctx.shape, ctx.x_stride, ctx.activation = x.shape, x_stride, activation
        ctx.set_materialize_grads(False)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, gradient: Tensor | None) -> tuple[Tensor | None, ...]:
        if gradient is None:
            return (None,) * 6
        needs_x, needs_weight, needs_bias, needs_residual = ctx.needs_input_grad[:4]
        grads: list[Tensor | None] = [None, None, None, gradient if needs_residual else None]
        if needs_x or needs_weight or needs_bias:
            x, codes, scales, weight, bias = ctx.saved_tensors
            outer, inner = weight.shape
            upstream, stride = rows_of(gradient)
            new = lambda shape: torch.empty(shape, dtype=weight.dtype, device=weight.device)
            grads[0] = new(ctx.shape) if needs_x else None
            grads[1] = new((outer, inner)) if needs_weight else None
            grads[2] = new((outer,)) if needs_bias else None
            a = abi.LinearBwdArgs()
            a.rows, a.inner, a.outer = gradient.numel() // outer, inner, outer
            a.dtype, a.activation = DTYPES[weight.dtype], ctx.activation
            a.x, a.x_stride = native.ptr(x), ctx.x_stride
            a.codes, a.scales = native.ptr(codes), native.ptr(scales)
            a.weight, a.bias = native.ptr(weight), native.ptr(bias)
            a.upstream, a.upstream_stride = native.ptr(upstream), stride
            a.grad_x, a.grad_weight, a.grad_bias = (native.ptr(g) for g in grads[:3])
            nbytes = native.query("gs3d_linear_bwd_call_scratch_bytes", ctypes.byref(a))
            work = scratch(nbytes, weight.device) if nbytes else None
            launch("gs3d_linear_bwd", ctypes.byref(a), weight.device, native.ptr(work), nbytes)
        return (*grads, None, None)


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, *, activation: str = "none",
           residual: Tensor | None = None, checkpoint: str | None = None) -> Tensor:
    """activation(x weight^T + bias) + residual for every pixel.

    x is (..., K), weight (N, K), bias (N,) and residual (..., N), all of one
    dtype (float32, bfloat16 or float16) on one device; the result is (..., N).
    Products are summed in 32 bits and rounded once.  ``activation`` is "none",
    "relu", "silu" or "gelu" (the exact one, z Phi(z)).  Differentiable in
    every tensor; the backward pass computes the activation's argument again
    rather than keep it, and takes the gradient at it to twice the dtype's
    precision.  With checkpoint="int8" the input is kept in 8 bits
    (``quantize_activations``) and the gradients are those at the kept value.
    """
    check_input("x", x, 1)
    inner = x.shape[-1]
    if not (isinstance(weight, Tensor) and weight.ndim == 2 and 1 <= weight.shape[0] <= abi.MAX_CHANNELS):
        raise ValueError(f"weight must be (N, K) with 1 <= N <= {abi.MAX_CHANNELS}")
    outer = weight.shape[0]
    check_like("weight", weight, x, (outer, inner))
    check_like("bias", bias, x, (outer,))
    check_like("residual", residual, x, tuple(x.shape[:-1]) + (outer,))
    code = activation_code(activation)
    check_checkpoint(checkpoint)
    if not recorded(x, weight, bias, residual):
        return _forward(x, weight, bias, residual, code, None)[0]
    return _Linear.apply(x, weight, bias, residual, code, checkpoint)
