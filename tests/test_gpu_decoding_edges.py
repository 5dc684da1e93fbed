"""The decoder at the edges of its arguments."""

import ctypes
import math

import pytest
import torch

import decoding_reference as ref
from dsl_splat_amd import decoding
from dsl_splat_amd.runtime import abi, native

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _case(rows, inner, outer, dtype):
    g = torch.Generator().manual_seed(rows + inner + outer)
    normal = lambda *shape, scale=1.0: (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)
    return normal(rows, inner), normal(outer, inner, scale=inner ** -0.5), normal(outer, scale=0.3), normal(rows, outer)


def _same(name, got, want, bound):
    """Within the bound where the formula is finite, else the formula's value."""
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), name
    assert torch.equal(got[~fine].isnan(), want[~fine].isnan()), name
    assert ((got - want).abs()[fine] <= bound[fine]).all(), name


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer", [(300, 33, 97), (133, 40, 72), (130, 16, 5), (257, 64, 64),
                                              (200, 300, 140)])
@pytest.mark.parametrize("checkpoint", (None, "int8"))
def test_relu_of_infinite_arguments(checkpoint, rows, inner, outer, dtype):
    """relu's slope is 1 or 0 at an infinity, so gradients stay what the formula
    gives, whether or not the channels and rows fill the kernels' tiles."""
    print("linear", rows, inner, outer, dtype, checkpoint, flush=True)
    x, w, b, up = _case(rows, inner, outer, dtype)
    if checkpoint is None:  # (in 8 bits the block reads back as NaN)
        x[7, 3], x[rows - 1, 0] = math.inf, -math.inf
        clean = ref.linear_grads(torch.where(torch.isfinite(x), x, torch.zeros_like(x)), w, b, up, "relu")["x"][1]
        leaf = x.detach().requires_grad_(True)
        (dx,) = torch.autograd.grad(decoding.linear(leaf, w, b, activation="relu"), leaf, up)
        z = x.double() @ w.double().T + b.double()
        dz = up.double() * (z > 0)
        bound = clean.amax() + (outer + 2) * (ref.U + ref.UNIT[dtype]) * (dz.abs() @ w.double().abs())
        _same("dx", dx, dz @ w.double(), bound)
    # An infinite weight: z is infinite in every row but only of its channel.
    x = torch.where(torch.isfinite(x), x, torch.ones_like(x))
    w = w.clone()
    w[2, 1] = math.inf
    leaf = w.detach().requires_grad_(True)
    (dw,) = torch.autograd.grad(decoding.linear(x, leaf, b, activation="relu", checkpoint=checkpoint), leaf, up)
    seen = (ref.kept(x) if checkpoint else x).double()
    z = seen @ w.double().T + b.double()
    dz = up.double() * torch.where(z.isnan(), z, (z > 0).double())
    size = seen.abs() @ torch.where(torch.isfinite(w), w, 0 * b[:, None]).double().abs().T + b.double().abs()
    near = up.double().abs() * (z.abs() <= (inner + 2) * ref.U * size)
    bound = near.T @ seen.abs() + ((rows + 2) * ref.U + ref.UNIT[dtype]) * (dz.abs().T @ seen.abs()) + ref.TINY[dtype]
    _same("dw", dw, dz.T @ seen, bound)


def test_no_pixels_at_the_c_entry_of_the_product():
    """Sums over no rows are zero; nothing is read for them."""
    dw, db = torch.ones(6 * 8, device=DEV), torch.ones(6, device=DEV)
    a = abi.LinearBwdArgs()
    a.rows, a.inner, a.outer, a.grad_weight, a.grad_bias = 0, 8, 6, native.ptr(dw), native.ptr(db)
    work = torch.empty(1 << 20, dtype=torch.uint8, device=DEV)
    stream = native.stream(torch.device(DEV, 0))
    native.call("gs3d_linear_bwd", ctypes.byref(a), native.ptr(work), work.numel(), stream)
    torch.cuda.synchronize()
    assert not dw.any() and not db.any()


@pytest.mark.parametrize("images,pixels", [(0, 5), (3, 0)])
def test_no_pixels_at_the_c_entry_of_the_norm(images, pixels):
    dw, db = torch.ones(8, device=DEV), torch.ones(8, device=DEV)
    a = abi.GroupNormBwdArgs()
    a.images, a.pixels, a.channels, a.groups = images, pixels, 8, 4
    a.grad_weight, a.grad_bias = native.ptr(dw), native.ptr(db)
    native.call("gs3d_group_norm_bwd", ctypes.byref(a), None, 0, native.stream(torch.device(DEV, 0)))
    torch.cuda.synchronize()
    assert not dw.any() and not db.any()


def test_quantized_values_of_any_layout():
    g = torch.Generator().manual_seed(4)
    x = torch.randn((40, 64), generator=g).to(DEV)
    q = decoding.quantize_activations(x)
    part = decoding.QuantizedActivations(q.codes[::2], q.scales[::2], q.dtype)
    assert torch.equal(part.dequantize(), q.dequantize()[::2])
    bad = [(q.codes.int(), q.scales, q.dtype), (q.codes, q.scales.int(), q.dtype), (q.codes, q.scales[:-1], q.dtype),
           (q.codes, q.scales[:, :1], q.dtype), (q.codes.cpu(), q.scales, q.dtype), (q.codes, q.scales.cpu(), q.dtype),
           (q.codes, q.scales, torch.float64), (q.codes[:, :0], q.scales[:, :0], q.dtype)]
    for i, args in enumerate(bad):
        with pytest.raises(ValueError):
            decoding.QuantizedActivations(*args).dequantize()
            pytest.fail(f"case {i} was accepted")


def test_backward_of_a_plain_product_reserves_no_room_for_an_activation():
    """Without an activation dz is the upstream gradient itself: beside the
    gradients the backward pass takes the splits' sums (512 at most of dW) and
    the weights once more."""
    rows, inner, outer = 200_000, 64, 512
    x, w, b, up = _case(rows, inner, outer, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = decoding.linear(*leaves)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    grads = torch.autograd.grad(y, leaves, up)
    torch.cuda.synchronize()
    most = sum(g.numel() * 2 for g in grads) + 512 * (outer * inner + outer) * 4 + 2 * outer * inner + (1 << 22)
    assert torch.cuda.max_memory_allocated() - before <= most


class _Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.decoder = decoding.FeatureDecoder(16, 24, 10, groups=4, device=DEV)

    def forward(self, x):
        return self.decoder(x)


def test_traces_replay_the_operators():
    g = torch.Generator().manual_seed(3)
    x, other = (torch.randn((6, 7, 16), generator=g).to(DEV) for _ in range(2))
    net = _Net()
    for grad in (False, True):
        with torch.set_grad_enabled(grad):
            traced = torch.jit.trace(net, x, check_trace=False)
            # Memory that a replay may be given.
            junk = [torch.full((n,), math.nan, device=DEV) for n in (420, 1008, 4096)]
            del junk
            for value in (other, x):
                assert torch.equal(traced(value), net(value))
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(lambda t: decoding.quantize_activations(t).dequantize(), x, check_trace=False)


@pytest.mark.parametrize("eps", (1e-46, 1e39))
def test_eps_outside_32_bits_is_refused(eps):
    """The kernels hold eps in 32 bits, where these are 0 and infinite."""
    with pytest.raises(ValueError, match="eps"):
        decoding.group_norm(torch.zeros((2, 2, 8), device=DEV), 2, eps=eps)
