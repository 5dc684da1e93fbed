"""The decoder's checks and plans on the host."""

import ctypes

import pytest
import torch

from dsl_splat_amd import decoding
from dsl_splat_amd.runtime import abi, native

P = ctypes.c_void_p(256)


def test_eight_bits_off_the_device_are_refused():
    """Codes and scales that were moved to the host are not addresses for a kernel."""
    kept = decoding.QuantizedActivations(torch.zeros((4, 40), dtype=torch.int8), torch.zeros((4, 2), dtype=torch.uint8),
                                         torch.float32)
    with pytest.raises(ValueError, match="CUDA"):
        kept.dequantize()


def _bwd_bytes(rows, inner, outer, dtype, activation=abi.ACT_NONE, **gradients):
    a = abi.LinearBwdArgs()
    a.rows, a.inner, a.outer, a.dtype, a.activation = rows, inner, outer, dtype, activation
    for name in gradients:
        setattr(a, name, P)
    return native.query("gs3d_linear_bwd_call_scratch_bytes", ctypes.byref(a))


@pytest.mark.parametrize("dtype", (abi.DTYPE_F32, abi.DTYPE_BF16, abi.DTYPE_F16))
@pytest.mark.parametrize("inner,outer", [(128, 512), (64, 64), (300, 70), (512, 33)])
def test_scratch_of_a_backward_call_follows_what_it_asks_for(inner, outer, dtype):
    rows, every = 1_920_000, dict(grad_x=1, grad_weight=1, grad_bias=1)
    most = native.query("gs3d_linear_bwd_scratch_bytes", rows, inner, outer, dtype)
    assert _bwd_bytes(rows, inner, outer, dtype, abi.ACT_SILU, **every) == most
    # Without an activation: 512 splits' dW and db at most and W^T, padded to
    # whole chunks; nothing that grows with the rows.
    padded = 4 * (inner + 64) * (outer + 64)
    assert _bwd_bytes(rows, inner, outer, dtype, **every) <= 513 * padded
    assert _bwd_bytes(rows, inner, outer, dtype, grad_x=1) <= padded
    assert _bwd_bytes(rows, inner, outer, dtype, grad_bias=1) <= 512 * padded
    assert _bwd_bytes(0, inner, outer, dtype, abi.ACT_SILU, **every) == 0
    assert _bwd_bytes(-1, inner, outer, dtype, **every) == 0
