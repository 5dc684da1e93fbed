"""Activations in 8 bits (gs3d_quantize_activations): int8 codes and one
power-of-two scale per 32 neighbouring channels of a pixel, 1.03 bytes a
value."""

from dataclasses import dataclass

import torch
from torch import Tensor

from ..runtime import native
from ._common import DTYPES, check_input, check_untraced, launch, rows_of

BLOCK = 32


@dataclass(slots=True)
class QuantizedActivations:
    """codes (..., C) int8 and scales (..., ceil(C / 32)) uint8: the value of a
    code is code * 2**(scale - 127) of its block.  Scale 255 marks a block that
    held a value that was not finite; it reads back as NaN."""

    codes: Tensor
    scales: Tensor
    dtype: torch.dtype

    @native.no_grad
    def dequantize(self) -> Tensor:
        """The values that were kept, in the dtype that was quantised."""
        check_untraced("dequantize")
        codes, scales = self.codes, self.scales
        if not (isinstance(codes, Tensor) and codes.is_cuda and codes.dtype == torch.int8 and codes.ndim):
            raise ValueError("codes must be a CUDA int8 tensor of at least one dimension")
        if not (isinstance(scales, Tensor) and scales.device == codes.device and scales.dtype == torch.uint8):
            raise ValueError(f"scales must be uint8 on {codes.device}")
        channels = codes.shape[-1]
        if channels < 1 or tuple(scales.shape) != _scales_shape(codes.shape):
            raise ValueError(f"codes {tuple(codes.shape)} need a channel and scales {_scales_shape(codes.shape)}, got "
                             f"{tuple(scales.shape)}")
        if self.dtype not in DTYPES:
            raise ValueError(f"dtype must be one of {tuple(DTYPES)}, got {self.dtype}")
        out = torch.empty(codes.shape, dtype=self.dtype, device=codes.device)
        if out.numel():
            codes, scales = codes.contiguous(), scales.contiguous()
            launch("gs3d_dequantize_activations", native.ptr(codes), out.device, native.ptr(scales),
                   out.numel() // channels, channels, DTYPES[self.dtype], native.ptr(out))
        return out


def _scales_shape(shape) -> tuple[int, ...]:
    return (*shape[:-1], (shape[-1] + BLOCK - 1) // BLOCK)


def empty_quantized(x: Tensor) -> QuantizedActivations:
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scales = torch.empty(_scales_shape(x.shape), dtype=torch.uint8, device=x.device)
    return QuantizedActivations(codes, scales, x.dtype)


@native.no_grad
def quantize_activations(x: Tensor) -> QuantizedActivations:
    """x (..., C) in 8 bits.  Per 32 neighbouring channels the scale is the
    smallest 2**e with max |x| <= 127 * 2**e, e from -126 to 121 (float16: 9);
    codes are rounded to nearest, ties to even, and at most 127 in size, so the
    last percent of the type's range is cut off.  Not differentiable; ``linear`` and
    ``group_norm`` keep their inputs in this form with checkpoint="int8"."""
    check_untraced("quantize_activations")
    check_input("x", x, 1)
    x = x.detach()
    channels = x.shape[-1]
    out = empty_quantized(x)
    if x.numel():
        rows, stride = rows_of(x)
        launch("gs3d_quantize_activations", native.ptr(rows), x.device, stride, x.numel() // channels, channels,
               DTYPES[x.dtype], native.ptr(out.codes), native.ptr(out.scales))
    return out
