"""Group normalisation of channel-last images with an activation
(gs3d_group_norm_fwd, gs3d_group_norm_bwd) and its first-order autograd."""

import ctypes
import math
from numbers import Integral, Real
from typing import Any

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from ..runtime import abi, native
from ._common import (DTYPES, activation_code, check_checkpoint, check_input, check_like, launch, recorded, rows_of,
                      scratch)
from .activations import QuantizedActivations, empty_quantized


def _scratch(shape, groups: int, dtype: int, device: torch.device) -> Tensor:
    images, pixels = math.prod(shape[:-3]), shape[-3] * shape[-2]
    return scratch(native.query("gs3d_group_norm_scratch_bytes", images, pixels, shape[-1], groups, dtype), device)


def _forward(x: Tensor, weight: Tensor | None, bias: Tensor | None, groups: int, eps: float, activation: int,
             quantized: QuantizedActivations | None) -> tuple[Tensor, Tensor, int, Tensor | None, Tensor | None, Tensor]:
    """(result, x as rows, their stride, weight, bias, statistics), the inputs
    as the kernels read them; where `quantized` is given x's 8-bit form goes
    there."""
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    images, channels = math.prod(x.shape[:-3]), x.shape[-1]
    rows, x_stride = rows_of(x)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    statistics = torch.empty((images, groups, 2), dtype=torch.float32, device=x.device)
    a = abi.GroupNormArgs()
    a.images, a.pixels, a.channels, a.groups = images, x.shape[-3] * x.shape[-2], channels, groups
    a.dtype, a.activation, a.eps = DTYPES[x.dtype], activation, eps
    a.x, a.x_stride = native.ptr(rows), x_stride
    a.weight, a.bias, a.y, a.statistics = (native.ptr(t) for t in (weight, bias, y, statistics))
    if quantized is not None:
        a.codes, a.scales = native.ptr(quantized.codes), native.ptr(quantized.scales)
    if x.numel():
        work = _scratch(x.shape, groups, a.dtype, x.device)
        launch("gs3d_group_norm_fwd", ctypes.byref(a), x.device, native.ptr(work), work.numel())
    return y, rows, x_stride, weight, bias, statistics


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x: Tensor, weight: Tensor | None, bias: Tensor | None, groups: int, eps: float,
                activation: int, checkpoint: str | None) -> Tensor:
        quantized = empty_quantized(x) if checkpoint is not None else None
        y, rows, x_stride, weight, bias, statistics = _forward(x, weight, bias, groups, eps, activation, quantized)
        kept: tuple[Tensor | None, ...] = (rows, None, None)
        if quantized is not None:
            kept = (None, quantized.codes, quantized.scales)
        ctx.save_for_backward(*kept, weight, bias, statistics)
        ctx.shape, ctx.x_stride, ctx.groups, ctx.activation = x.shape, x_stride, groups, activation
        ctx.set_materialize_grads(False)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, gradient: Tensor | None) -> tuple[Tensor | None, ...]:
        if gradient is None:
            return (None,) * 7
        x, codes, scales, weight, bias, statistics = ctx.saved_tensors
        channels = ctx.shape[-1]
        upstream, stride = rows_of(gradient)
        grads = [torch.empty(shape, dtype=gradient.dtype, device=gradient.device) if needed else None
                 for shape, needed in zip((ctx.shape, (channels,), (channels,)), ctx.needs_input_grad)]
        a = abi.GroupNormBwdArgs()
        a.images, a.pixels = math.prod(ctx.shape[:-3]), ctx.shape[-3] * ctx.shape[-2]
        a.channels, a.groups = channels, ctx.groups
        a.dtype, a.activation = DTYPES[gradient.dtype], ctx.activation
        a.x, a.x_stride = native.ptr(x), ctx.x_stride
        a.codes, a.scales = native.ptr(codes), native.ptr(scales)
        a.weight, a.bias, a.statistics = native.ptr(weight), native.ptr(bias), native.ptr(statistics)
        a.upstream, a.upstream_stride = native.ptr(upstream), stride
        a.grad_x, a.grad_weight, a.grad_bias = (native.ptr(g) for g in grads)
        work = _scratch(ctx.shape, ctx.groups, a.dtype, gradient.device)
        launch("gs3d_group_norm_bwd", ctypes.byref(a), gradient.device, native.ptr(work), work.numel())
        return (*grads, None, None, None, None)


def group_norm(x: Tensor, groups: int, weight: Tensor | None = None, bias: Tensor | None = None, *,
               eps: float = 1e-5, activation: str = "none", checkpoint: str | None = None) -> Tensor:
    """activation((x - mean) / sqrt(var + eps) * weight + bias) of channel-last
    images.

    x is (..., H, W, C), every leading index an image of its own; mean and
    (biased) variance are taken per image and group of C / groups neighbouring
    channels over all its pixels.  weight and bias are (C,); all of one dtype
    (float32, bfloat16 or float16).  Statistics are held in 32 bits.
    Activations as in ``linear``.  Differentiable in every tensor; with
    checkpoint="int8" the input is kept in 8 bits for the backward pass, which
    takes x where it occurs (not in the statistics, which are kept whole) as
    the kept value.
    """
    check_input("x", x, 3)
    channels = x.shape[-1]
    if isinstance(groups, bool) or not isinstance(groups, Integral) or groups < 1 or channels % groups:
        raise ValueError(f"groups must be a positive divisor of the {channels} channels, got {groups!r}")
    if math.prod(x.shape[:-3]) > abi.MAX_IMAGES:
        raise ValueError(f"x has more than {abi.MAX_IMAGES} images")
    check_like("weight", weight, x, (channels,))
    check_like("bias", bias, x, (channels,))
    if isinstance(eps, bool) or not isinstance(eps, Real) or not 0.0 < ctypes.c_float(eps).value < math.inf:
        raise ValueError(f"eps must be positive and finite in 32 bits, got {eps!r}")
    code = activation_code(activation)
    check_checkpoint(checkpoint)
    if not recorded(x, weight, bias):
        return _forward(x, weight, bias, int(groups), float(eps), code, None)[0]
    return _GroupNorm.apply(x, weight, bias, int(groups), float(eps), code, checkpoint)
