"""Activations in 8 bits (gs3d_quantize_activations): int8 codes and one
power-of-two scale per 32 neighbouring channels of a pixel, 1.03 bytes a
value."""

from dataclasses import dataclass

import torch
from torch import Tensor

from ..runtime import native
from ._common import DTYPES, check_input, launch, rows_of

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
        out = torch.empty(self.codes.shape, dtype=self.dtype, device=self.codes.device)
        channels = self.codes.shape[-1]
        if out.numel():
            launch("gs3d_dequantize_activations", native.ptr(self.codes), out.device, native.ptr(self.scales),
                   out.numel() // channels, channels, DTYPES[self.dtype], native.ptr(out))
        return out


def empty_quantized(x: Tensor) -> QuantizedActivations:
    channels = x.shape[-1]
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scales = torch.empty(x.shape[:-1] + ((channels + BLOCK - 1) // BLOCK,), dtype=torch.uint8, device=x.device)
    return QuantizedActivations(codes, scales, x.dtype)


@native.no_grad
def quantize_activations(x: Tensor) -> QuantizedActivations:
    """x (..., C) in 8 bits.  Per 32 neighbouring channels the scale is the
    smallest 2**e with max |x| <= 127 * 2**e, e from -126 to 121 (float16: 9);
    codes are rounded to nearest, ties to even, and at most 127 in size, so the
    last percent of the type's range is cut off.  Not differentiable; ``linear`` and
    ``group_norm`` keep their inputs in this form with checkpoint="int8"."""
    check_input("x", x, 1)
    x = x.detach()
    channels = x.shape[-1]
    out = empty_quantized(x)
    if x.numel():
        rows, stride = rows_of(x)
        launch("gs3d_quantize_activations", native.ptr(rows), x.device, stride, x.numel() // channels, channels,
               DTYPES[x.dtype], native.ptr(out.codes), native.ptr(out.scales))
    return out
