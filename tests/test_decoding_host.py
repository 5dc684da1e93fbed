"""The decoder's checks and plans on the host."""

import ctypes
import os
import subprocess
from collections import Counter

import pytest
import torch

import dsl_splat_amd
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


@pytest.fixture(scope="module")
def deal(tmp_path_factory):
    """csrc/xcd.hpp's deal_block, compiled for the host."""
    folder = tmp_path_factory.mktemp("xcd")
    source, library = str(folder / "deal.cpp"), str(folder / "deal.so")
    with open(source, "w") as f:
        f.write('#include "xcd.hpp"\nextern "C" void deal(unsigned b, unsigned g, unsigned t, unsigned* out)'
                '{ gs3d::Dealt d = gs3d::deal_block(b, g, t); out[0] = d.group; out[1] = d.tile; }\n')
    csrc = os.path.join(os.path.dirname(dsl_splat_amd.__file__), "csrc")
    subprocess.run(["g++", "-shared", "-fPIC", "-std=c++17", "-D__host__=", "-D__device__=", "-I", csrc, source, "-o",
                    library], check=True, timeout=120)
    function = ctypes.CDLL(library).deal
    out = (ctypes.c_uint * 2)()

    def call(block, groups, tiles):
        function(block, groups, tiles, out)
        return out[0], out[1]

    return call


@pytest.mark.parametrize("groups,tiles", [(1, 1), (1, 128), (2, 256), (7, 5), (8, 64), (9, 32), (15, 4), (42, 12),
                                          (85, 6), (170, 3), (64, 8), (1000, 1)])
def test_blocks_are_dealt_evenly(deal, groups, tiles):
    """Every block once, as many on each of the eight XCDs to within one, and
    eight groups at a time each on one."""
    dealt = [deal(b, groups, tiles) for b in range(groups * tiles)]
    assert sorted(dealt) == [(g, t) for g in range(groups) for t in range(tiles)]
    load = Counter(b % 8 for b in range(groups * tiles))
    assert max(load.values()) - min(load[x] for x in range(8)) <= 1
    for g in range(groups // 8 * 8):
        assert len({b % 8 for b, at in enumerate(dealt) if at[0] == g}) == 1
    assert deal(2**31 - 1, 2**27, 16) == (2**27 - 1, 15)
