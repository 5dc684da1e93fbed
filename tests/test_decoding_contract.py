"""The decoder's C entry points and Python checks that need no device."""

import ctypes

import pytest
import torch

from dsl_splat_amd import decoding
from dsl_splat_amd.runtime import abi, native

P = ctypes.c_void_p(256)


def _linear():
    a = abi.LinearArgs()
    a.rows, a.inner, a.outer = 10, 8, 6
    a.x, a.x_stride, a.weight, a.y = P, 8, P, P
    return a


def _linear_bwd():
    a = abi.LinearBwdArgs()
    a.rows, a.inner, a.outer = 10, 8, 6
    a.x, a.x_stride, a.weight, a.upstream, a.upstream_stride, a.grad_weight = P, 8, P, P, 6, P
    return a


def _norm():
    a = abi.GroupNormArgs()
    a.images, a.pixels, a.channels, a.groups, a.eps = 2, 10, 8, 4, 1e-5
    a.x, a.x_stride, a.y, a.statistics = P, 8, P, P
    return a


def _norm_bwd():
    a = abi.GroupNormBwdArgs()
    a.images, a.pixels, a.channels, a.groups = 2, 10, 8, 4
    a.x, a.x_stride, a.statistics, a.upstream, a.upstream_stride = P, 8, P, P, 8
    return a


@pytest.mark.parametrize("make,name,scratch,changes", [
    (_linear, "gs3d_linear_fwd", True, [
        ("rows", -1), ("rows", abi.MAX_ROWS + 1), ("inner", 0), ("outer", 0), ("inner", abi.MAX_CHANNELS + 1),
        ("dtype", 3), ("dtype", -1), ("activation", 4), ("activation", -1), ("x_stride", 7), ("x", None),
        ("weight", None), ("y", None)]),
    (_linear_bwd, "gs3d_linear_bwd", True, [
        ("rows", -1), ("inner", 0), ("outer", abi.MAX_CHANNELS + 1), ("dtype", 3), ("activation", 4), ("x_stride", 7),
        ("x", None), ("weight", None), ("upstream", None), ("upstream_stride", 5), ("codes", P), ("scales", P)]),
    (_norm, "gs3d_group_norm_fwd", True, [
        ("images", -1), ("images", abi.MAX_IMAGES + 1), ("pixels", -1), ("channels", 0), ("groups", 0), ("groups", 3),
        ("dtype", 3), ("activation", 4), ("eps", 0.0), ("eps", float("nan")), ("x_stride", 7), ("x", None),
        ("y", None), ("statistics", None)]),
    (_norm_bwd, "gs3d_group_norm_bwd", True, [
        ("images", -1), ("pixels", abi.MAX_ROWS + 1), ("channels", abi.MAX_CHANNELS + 4), ("groups", 3), ("dtype", 3),
        ("activation", 4), ("x_stride", 7), ("x", None), ("statistics", None), ("upstream", None),
        ("upstream_stride", 7), ("codes", P), ("scales", P)]),
])
def test_entry_points_check_their_arguments(make, name, scratch, changes):
    call = getattr(native.load(), name)
    more = (P, 1 << 40)
    for field, value in changes:
        a = make()
        setattr(a, field, value)
        assert call(ctypes.byref(a), *more, None) == abi.GS3D_ERR_ARGUMENT, (name, field, value)
    assert call(None, *more, None) == abi.GS3D_ERR_ARGUMENT
    if scratch:
        a = make()
        if name == "gs3d_linear_fwd":
            a.rows, a.inner, a.outer, a.x_stride, a.dtype = 100_000, 300, 16, 300, abi.DTYPE_BF16  # packed weights
        assert call(ctypes.byref(a), P, 1, None) == abi.GS3D_ERR_SCRATCH
        assert call(ctypes.byref(a), None, 1 << 40, None) == abi.GS3D_ERR_SCRATCH


def test_quantize_entry_points_check_their_arguments():
    lib = native.load()
    for args in ((P, 8, -1, 8, 0, P, P), (P, 8, 4, 0, 0, P, P), (P, 7, 4, 8, 0, P, P), (P, 8, 4, 8, 3, P, P),
                 (None, 8, 4, 8, 0, P, P), (P, 8, 4, 8, 0, None, P), (P, 8, 4, 8, 0, P, None)):
        assert lib.gs3d_quantize_activations(*args, None) == abi.GS3D_ERR_ARGUMENT
    assert lib.gs3d_quantize_activations(None, 8, 0, 8, 0, None, None, None) == abi.GS3D_OK
    for args in ((P, P, -1, 8, 0, P), (P, P, 4, 0, 0, P), (P, P, 4, 8, 3, P), (None, P, 4, 8, 0, P),
                 (P, None, 4, 8, 0, P), (P, P, 4, 8, 0, None)):
        assert lib.gs3d_dequantize_activations(*args, None) == abi.GS3D_ERR_ARGUMENT
    assert lib.gs3d_dequantize_activations(None, None, 0, 8, 0, None, None) == abi.GS3D_OK


def test_scratch_queries():
    for rows in (0, 1, 1000, 2_000_000):
        assert native.query("gs3d_linear_bwd_scratch_bytes", rows, 33, 97, abi.DTYPE_BF16) > 0
    assert native.query("gs3d_linear_bwd_scratch_bytes", 10, 0, 97, 0) == 0
    assert native.query("gs3d_group_norm_scratch_bytes", 2, 1000, 64, 8, abi.DTYPE_F32) > 0
    assert native.query("gs3d_group_norm_scratch_bytes", 2, 1000, 64, 7, abi.DTYPE_F32) == 0
    # Empty work is a no-op.
    a = _linear()
    a.rows, a.x, a.weight, a.y = 0, None, None, None
    assert native.load().gs3d_linear_fwd(ctypes.byref(a), None, 0, None) == abi.GS3D_OK
    n = _norm()
    n.pixels, n.x, n.y, n.statistics = 0, None, None, None
    assert native.load().gs3d_group_norm_fwd(ctypes.byref(n), None, 0, None) == abi.GS3D_OK


def test_operators_refuse_host_tensors():
    x = torch.zeros((4, 5, 8))
    for call in (lambda: decoding.linear(x, torch.zeros(6, 8)), lambda: decoding.group_norm(x, 2),
                 lambda: decoding.quantize_activations(x), lambda: decoding.linear([1.0], torch.zeros(1, 1))):
        with pytest.raises(ValueError, match="CUDA"):
            call()
