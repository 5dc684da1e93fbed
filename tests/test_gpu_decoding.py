"""The feature decoder's operators on the GPU against their formulas in 64 bits
(tests/decoding_reference.py, which also derives every bound)."""

import math

import numpy as np
import pytest
import torch

import decoding_reference as ref
from dsl_splat_amd import decoding, gs3d, synthetic
from dsl_splat_amd.runtime import abi

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _normal(g, *shape, scale=1.0, shift=0.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype).to(DEV)


def _linear_case(seed, rows, inner, outer, dtype, residual=True, lead=None):
    g = torch.Generator().manual_seed(seed)
    lead = (rows,) if lead is None else lead
    x = _normal(g, *lead, inner, dtype=dtype)
    w = _normal(g, outer, inner, scale=inner ** -0.5, dtype=dtype)
    b = _normal(g, outer, scale=0.3, dtype=dtype)
    r = _normal(g, *lead, outer, dtype=dtype) if residual else None
    up = _normal(g, *lead, outer, dtype=dtype)
    return x, w, b, r, up


def _check_linear(x, w, b, r, up, activation, checkpoint=None):
    leaves = [t if t is None else t.detach().requires_grad_(True) for t in (x, w, b, r)]
    y = decoding.linear(*leaves[:3], activation=activation, residual=leaves[3], checkpoint=checkpoint)
    assert y.shape == x.shape[:-1] + (w.shape[0],) and y.dtype == x.dtype and y.is_contiguous()
    want, bound = ref.linear(x.reshape(-1, x.shape[-1]), w, b, None if r is None else r.reshape(-1, w.shape[0]),
                             activation)
    ref.check("y", y, want, bound)
    named = [(n, t) for n, t in zip(("x", "weight", "bias", "residual"), leaves) if t is not None]
    got = torch.autograd.grad(y, [t for _, t in named], up)
    seen = ref.kept(x) if checkpoint else x
    grads = ref.linear_grads(seen, w, b, up, activation)
    for (name, leaf), value in zip(named, got):
        assert value.shape == leaf.shape and value.dtype == leaf.dtype
        if name == "residual":
            assert torch.equal(value, up)
        else:
            ref.check("grad " + name, value, *grads[name])


SIZES = [(1, 1, 1), (1, 32, 512), (2, 512, 3), (5, 3, 7), (63, 33, 97), (64, 64, 64), (129, 100, 130), (1023, 31, 33),
         (1025, 48, 20), (300, 257, 259), (2000, 512, 40), (2111, 40, 512), (70000, 32, 128), (4099, 8, 8), (700, 16, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer", SIZES)
def test_linear_sizes(rows, inner, outer, dtype):
    print("linear", rows, inner, outer, dtype, flush=True)
    kind = ("none", "silu", "gelu")[(rows + inner) % 3]
    _check_linear(*_linear_case(rows + inner, rows, inner, outer, dtype, residual=outer % 2 == 0), kind)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", ("none", "relu", "silu", "gelu"))
def test_linear_activations(activation, dtype):
    print("linear", activation, dtype, flush=True)
    x, w, b, r, up = _linear_case(3, 1500, 40, 72, dtype)
    x = x * 4  # arguments from deep in both tails
    _check_linear(x, w, b, r, up, activation)
    _check_linear(x, w, None, None, up, activation)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer", [(1, 5, 4), (64, 32, 32), (1003, 33, 97), (2500, 128, 128), (900, 300, 70),
                                              (33000, 64, 96)])
def test_linear_checkpoint(rows, inner, outer, dtype):
    print("linear int8", rows, inner, outer, dtype, flush=True)
    for kind in ("none", "silu"):
        _check_linear(*_linear_case(rows, rows, inner, outer, dtype), kind, checkpoint="int8")


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_strides_and_offsets(dtype):
    x, w, b, r, up = _linear_case(11, 0, 33, 50, dtype, lead=(3, 17, 29))
    g = torch.Generator().manual_seed(12)

    def inside(t, left, right, fill):
        """t as a slice of wider rows whose other values are `fill`."""
        wide = torch.full(t.shape[:-1] + (left + t.shape[-1] + right,), fill, dtype=dtype, device=DEV)
        wide[..., left:left + t.shape[-1]] = t
        return wide[..., left:left + t.shape[-1]]

    # Slices of wider images, off the 16-byte grid, beside values that would
    # show; a transposed weight; images out of order in memory; a residual and
    # an upstream gradient with strides of their own.
    _check_linear(inside(x, 1, 6, math.nan), w.T.contiguous().T, b, inside(r, 3, 2, math.nan), inside(up, 5, 1, math.nan),
                  "silu")
    _check_linear(x.permute(1, 0, 2, 3), w, b, r.permute(1, 0, 2, 3), up.permute(1, 0, 2, 3), "gelu")
    _check_linear(x[:, ::2], w, b, r[:, ::2], up[:, ::2], "silu", checkpoint="int8")
    one = _normal(g, 1, 1, 33, dtype=dtype)
    _check_linear(one.expand(4, 5, 33), w, b, None, up[0, 0, :1].expand(4, 5, 50), "none")
    # An upstream gradient without any memory of its own.
    leaf = x.detach().requires_grad_(True)
    decoding.linear(leaf, w, b).sum().backward()
    want, bound = ref.linear_grads(x, w, b, torch.ones_like(up), "none")["x"]
    ref.check("grad of a sum", leaf.grad, want, bound)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_values_that_are_not_finite_stay_in_their_pixel(dtype):
    x, w, b, r, up = _linear_case(21, 300, 33, 40, dtype)
    clean = decoding.linear(x, w, b, activation="silu")
    bad = x.clone()
    bad[7, 32], bad[150, 0], bad[299, 5] = math.nan, math.inf, -math.inf
    got = decoding.linear(bad, w, b, activation="silu")
    rows = torch.ones(300, dtype=torch.bool, device=DEV)
    rows[[7, 150, 299]] = False
    assert torch.equal(got[rows], clean[rows])
    assert got[7].isnan().all() and not torch.isfinite(got[150]).all() and not torch.isfinite(got[299]).all()
    # Through the backward pass: only their pixels' input gradients, every weight gradient of their channel.
    for checkpoint in (None, "int8"):
        leaf, weight = bad.detach().requires_grad_(True), w.detach().requires_grad_(True)
        dx, dw = torch.autograd.grad(decoding.linear(leaf, weight, b, activation="silu", checkpoint=checkpoint),
                                     [leaf, weight], up)
        assert torch.isfinite(dx[rows]).all() and dx[7].isnan().all()
        assert dw[:, 32].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_without_pixels(dtype):
    x, w, b, r, up = _linear_case(5, 0, 8, 6, dtype)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    y = decoding.linear(*leaves[:3], activation="silu", residual=leaves[3])
    assert y.shape == (0, 6)
    grads = torch.autograd.grad(y, leaves, up)
    assert grads[0].shape == (0, 8) and not grads[1].any() and not grads[2].any()
    assert decoding.quantize_activations(x).dequantize().shape == (0, 8)


def test_linear_computes_what_is_asked_for():
    x, w, b, r, up = _linear_case(31, 500, 24, 36, torch.float32)
    full = ref.linear_grads(x, w, b, up, "silu")
    for wanted in (("x",), ("weight",), ("bias",), ("x", "bias")):
        leaves = {n: t.detach().requires_grad_(n in wanted) for n, t in (("x", x), ("weight", w), ("bias", b))}
        y = decoding.linear(leaves["x"], leaves["weight"], leaves["bias"], activation="silu")
        got = torch.autograd.grad(y, [leaves[n] for n in wanted], up)
        for name, value in zip(wanted, got):
            ref.check(name, value, *full[name])
    with torch.no_grad():
        assert not decoding.linear(x.requires_grad_(True), w, b).requires_grad


def test_linear_rows_past_32_bits():
    """Rows whose elements lie beyond 2^31 and 2^32 elements of the first."""
    rows, stride = 70_000, 65_600
    storage = torch.empty(rows * stride, dtype=torch.bfloat16, device=DEV)
    x = storage.view(rows, stride)[:, :24]
    g = torch.Generator().manual_seed(1)
    x.copy_(_normal(g, rows, 24, dtype=torch.bfloat16))
    w = _normal(g, 16, 24, scale=0.2, dtype=torch.bfloat16)
    up = _normal(g, rows, 16, dtype=torch.bfloat16)
    assert rows * stride > 2 ** 32
    _check_linear(x, w, None, None, up, "silu")
    q = decoding.quantize_activations(x)
    assert torch.equal(q.dequantize().double(), ref.kept(x[:]).to(DEV))


def test_linear_gradients_against_differences():
    """Directional derivatives of <up, y> from central differences of the
    operator's own forward in 32 bits."""
    x, w, b, r, up = _linear_case(41, 400, 20, 28, torch.float32)
    g = torch.Generator().manual_seed(42)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    for kind in ("silu", "gelu"):
        grads = torch.autograd.grad(decoding.linear(*leaves, activation=kind, residual=r), leaves, up)
        for i, leaf in enumerate(leaves):
            d = _normal(g, *leaf.shape)
            h = 2.0 ** -6
            values = []
            for sign in (1, -1):
                args = [t.detach() for t in leaves]
                args[i] = args[i] + sign * h * d
                values.append((decoding.linear(*args, activation=kind, residual=r).double() * up.double()).sum())
            slope = ((values[0] - values[1]) / (2 * h)).item()
            exact = (grads[i].double() * d.double()).sum().item()
            # Third derivative at most 2 in size; the forward's own bound, twice, over 2h.
            args = [t.detach() for t in leaves]
            step = {0: (d, w, None), 1: (x, d, None), 2: (torch.zeros_like(x), w, d)}[i]
            along = (step[0].double() @ step[1].double().T + (0 if step[2] is None else step[2].double())).abs()
            cut = (up.double().abs() * 2 * along ** 3).sum().item() * h * h / 6
            noise = (up.double().abs() * ref.linear(args[0].abs() + h * d.abs().max(), args[1], args[2], r, kind)[1]).sum().item() / h
            own = (grads[i].double().abs() * d.double().abs()).sum().item() * 2.0 ** -20
            assert abs(slope - exact) <= cut + noise + own, (kind, i, slope, exact, cut, noise)


# --------------------------------------------------------------------------
# Group norm


def _norm_case(seed, images, height, width, channels, dtype, shift=0.0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = _normal(g, images, height, width, channels, scale=scale, shift=shift, dtype=dtype)
    w = _normal(g, channels, scale=0.3, shift=1.0, dtype=dtype)
    b = _normal(g, channels, scale=0.3, dtype=dtype)
    up = _normal(g, images, height, width, channels, dtype=dtype)
    return x, w, b, up


def _check_norm(x, groups, w, b, up, activation, checkpoint=None, eps=1e-5):
    flat = lambda t: t.reshape(-1, t.shape[-3] * t.shape[-2], t.shape[-1])
    leaves = [t if t is None else t.detach().requires_grad_(True) for t in (x, w, b)]
    y = decoding.group_norm(leaves[0], groups, leaves[1], leaves[2], eps=eps, activation=activation,
                            checkpoint=checkpoint)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    norm = ref.Norm(flat(x), groups, w, b, eps, activation)
    ref.check("y", y, *norm.forward())
    named = [(n, t) for n, t in zip(("x", "weight", "bias"), leaves) if t is not None]
    got = torch.autograd.grad(y, [t for _, t in named], up)
    grads = norm.grads(flat(ref.kept(x) if checkpoint else x), flat(up))
    for (name, leaf), value in zip(named, got):
        assert value.shape == leaf.shape and value.dtype == leaf.dtype
        ref.check("grad " + name, value, *grads[name])


NORMS = [(1, 1, 1, 1, 1), (1, 1, 1, 8, 2), (2, 1, 3, 5, 5), (3, 7, 5, 12, 4), (2, 16, 16, 48, 6), (1, 33, 31, 97, 1),
         (4, 20, 13, 64, 8), (1, 64, 50, 128, 32), (2, 11, 9, 255, 15), (1, 5, 4, 512, 512), (1, 40, 30, 36, 3),
         (1, 130, 120, 16, 16), (5, 2, 2, 2100, 7), (1, 9, 10, 4096, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("images,height,width,channels,groups", NORMS)
def test_norm_sizes(images, height, width, channels, groups, dtype):
    print("norm", images, height, width, channels, groups, dtype, flush=True)
    x, w, b, up = _norm_case(channels + height, images, height, width, channels, dtype)
    kind = ("silu", "none", "gelu")[(channels + groups) % 3]
    _check_norm(x, groups, w, b, up, kind)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", ("none", "relu", "silu", "gelu"))
def test_norm_activations(activation, dtype):
    x, w, b, up = _norm_case(1, 2, 23, 19, 40, dtype)
    _check_norm(x, 5, w, b, up, activation)
    _check_norm(x, 8, None, None, up, activation)
    _check_norm(x, 4, w, None, up, activation, eps=0.1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels,groups", [(32, 4), (33, 3), (70, 7), (128, 32)])
def test_norm_checkpoint(channels, groups, dtype):
    x, w, b, up = _norm_case(channels, 2, 21, 30, channels, dtype)
    for kind in ("none", "silu"):
        _check_norm(x, groups, w, b, up, kind, checkpoint="int8")


@pytest.mark.parametrize("shift", (100.0, 4000.0))
def test_norm_far_from_zero(shift):
    """A mean far larger than the spread: a difference of squares would lose
    every digit of the variance at 4000."""
    x, w, b, up = _norm_case(9, 2, 40, 50, 24, torch.float32, shift=shift)
    x[0, 0, 0] = 0.0  # and a first pixel unlike the others
    _check_norm(x, 6, w, b, up, "silu")


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_flat_images(dtype):
    """An empty view: every pixel alike, the variance zero."""
    x = torch.full((2, 12, 10, 16), 0.5, dtype=dtype, device=DEV)
    x[1] = 0
    _, w, b, up = _norm_case(2, 2, 12, 10, 16, dtype)
    _check_norm(x, 4, w, b, up, "silu")


def test_norm_strides_and_views():
    x, w, b, up = _norm_case(13, 6, 14, 9, 33, torch.bfloat16)
    wide = torch.full((2, 3, 14, 9, 40), math.nan, dtype=torch.bfloat16, device=DEV)
    wide[..., 2:35] = x.view(2, 3, 14, 9, 33)
    _check_norm(wide[..., 2:35], 3, w, b, up.view(2, 3, 14, 9, 33), "silu")
    _check_norm(x.permute(0, 2, 1, 3), 11, w, b, up.permute(0, 2, 1, 3), "gelu")
    _check_norm(x[:, 1:, 2:], 3, w, b, up[:, 1:, 2:], "silu", checkpoint="int8")
    _check_norm(x[0], 3, w, b, up[0, :1, :1].expand(14, 9, 33), "none")


def test_norm_values_that_are_not_finite_stay_in_their_group():
    x, w, b, up = _norm_case(14, 3, 10, 12, 24, torch.float32)
    clean = decoding.group_norm(x, 4, w, b, activation="silu")
    bad = x.clone()
    bad[1, 3, 4, 7] = math.nan
    got = decoding.group_norm(bad, 4, w, b, activation="silu")
    hit = torch.zeros(3, 10, 12, 24, dtype=torch.bool, device=DEV)
    hit[1, :, :, 6:12] = True
    assert torch.equal(got[~hit], clean[~hit]) and got[hit].isnan().all()


@pytest.mark.parametrize("shape", [(0, 4, 5, 8), (2, 0, 5, 8), (2, 4, 0, 8)])
def test_norm_without_pixels(shape):
    x = torch.empty(shape, device=DEV, requires_grad=True)
    w = torch.ones(8, device=DEV, requires_grad=True)
    y = decoding.group_norm(x, 2, w, activation="silu")
    assert y.shape == shape
    dx, dw = torch.autograd.grad(y, [x, w], torch.ones_like(y))
    assert dx.shape == shape and not dw.any()


# --------------------------------------------------------------------------
# Eight bits


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", [(1, 1), (3, 7), (65, 31), (64, 32), (129, 33), (1000, 64), (77, 97), (513, 300),
                                           (9, 4096)])
def test_quantized_values(rows, channels, dtype):
    g = torch.Generator().manual_seed(rows + channels)
    x = torch.randn((rows, channels), generator=g) * torch.exp2(torch.randint(-12, 8, (rows, 1), generator=g).float())
    x[0] = 0
    x[-1] = 127.0  # the edge of a scale
    x = x.to(dtype).to(DEV)
    q = decoding.quantize_activations(x)
    assert q.codes.shape == x.shape and q.scales.shape == (rows, -(-channels // 32))
    got = q.dequantize()
    assert got.dtype == dtype and torch.equal(got.double(), ref.kept(x))
    assert (q.codes.int().abs() <= 127).all()
    # Kept values keep themselves.
    again = decoding.quantize_activations(got)
    assert torch.equal(again.dequantize(), got)


def test_quantized_ties_and_extremes():
    x = torch.zeros((8, 32), device=DEV)
    x[0, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5])           # scale 1: ties to even
    x[1, :3] = torch.tensor([127.5, 1.0, 3.0])                 # scale 2
    x[2, :2] = torch.tensor([3.4028234e38, -1.0])              # the largest float
    x[3, :3] = torch.tensor([1e-40, -1e-45, 0.0])              # below every scale: zeros
    x[4, :2] = torch.tensor([2.0 ** -126, -(2.0 ** -120)])     # the smallest scale
    x[5, 3], x[6, 31], x[7, 0] = math.nan, math.inf, -math.inf
    q = decoding.quantize_activations(x)
    got = q.dequantize()
    assert q.codes[0, :4].tolist() == [127, 0, 2, -2] and q.scales[0, 0] == 127
    assert q.codes[1, :3].tolist() == [64, 0, 2] and q.scales[1, 0] == 128
    assert torch.equal(got[:5].double(), ref.kept(x[:5]))
    assert got[5:].isnan().all() and (q.scales[5:] == 255).all()
    half = torch.tensor([[65504.0, -65504.0, 3.0]], dtype=torch.float16, device=DEV)
    assert decoding.quantize_activations(half).dequantize()[0].tolist() == [65024.0, -65024.0, 0.0]


def test_checkpoints_take_less_memory():
    x = torch.randn((200_000, 64), device=DEV, dtype=torch.bfloat16)
    w = torch.randn((64, 64), device=DEV, dtype=torch.bfloat16, requires_grad=True)

    def held(checkpoint):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        h = decoding.group_norm((x + 0).view(400, 500, 64), 8, activation="silu", checkpoint=checkpoint)
        h = decoding.linear(x + 0, w, activation="silu", checkpoint=checkpoint)
        return torch.cuda.memory_allocated() - before, h

    whole, y0 = held(None)
    eight, y1 = held("int8")
    assert torch.equal(y0, y1)
    values = x.numel()
    assert whole - eight >= 2 * values - (values + values // 32) - 4096


# --------------------------------------------------------------------------
# Streams, graphs, repeated calls, refusals, the decoder


def test_side_stream():
    x, w, b, r, up = _linear_case(51, 3000, 48, 64, torch.float32)
    want = decoding.linear(x, w, b, activation="silu", residual=r)
    norm = decoding.group_norm(want.view(50, 60, 64), 8, activation="gelu")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = torch.zeros_like(x)
        torch.cuda._sleep(20_000_000)
        late.copy_(x)
        y = decoding.linear(late, w, b, activation="silu", residual=r)
        n = decoding.group_norm(y.view(50, 60, 64), 8, activation="gelu")
        q = decoding.quantize_activations(n).dequantize()
    side.synchronize()
    assert torch.equal(y, want) and torch.equal(n, norm)
    assert torch.equal(q, decoding.quantize_activations(norm).dequantize())


def test_repeated_calls_agree_to_the_bit():
    x, w, b, r, up = _linear_case(52, 40_000, 96, 72, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def once():
        y = decoding.linear(*leaves, activation="gelu", residual=r)
        n = decoding.group_norm(y.view(200, 200, 72), 9, activation="silu")
        return [y, n, *torch.autograd.grad(n, leaves, up.view(200, 200, 72))]

    first = once()
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(first, once()))


def test_graph_replays():
    x, w, b, r, up = _linear_case(53, 3600, 40, 48, torch.bfloat16)

    def step():
        with torch.no_grad():
            y = decoding.linear(x, w, b, activation="silu", residual=r)
            n = decoding.group_norm(y.view(60, 60, 48), 6, activation="gelu")
            return [y, n, decoding.quantize_activations(n).dequantize()]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    g = torch.Generator().manual_seed(54)
    for _ in range(4):
        x.copy_(_normal(g, *x.shape, dtype=x.dtype))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, step()))
        torch.cuda.synchronize()


def test_refusals():
    x, w, b, r, _ = _linear_case(61, 10, 8, 6, torch.float32)
    image = torch.zeros((4, 5, 8), device=DEV)
    bad = [
        lambda: decoding.linear(x, w.half(), b),
        lambda: decoding.linear(x, w.cpu(), b),
        lambda: decoding.linear(x, w[:, :7], b),
        lambda: decoding.linear(x, w[0], b),
        lambda: decoding.linear(x, w, b[:5]),
        lambda: decoding.linear(x, w, b.double()),
        lambda: decoding.linear(x, w, b, residual=r[:9]),
        lambda: decoding.linear(x, w, b, residual=r[:1]),
        lambda: decoding.linear(x, w, b, activation="tanh"),
        lambda: decoding.linear(x, w, b, activation=None),
        lambda: decoding.linear(x, w, b, checkpoint="int4"),
        lambda: decoding.linear(x.double(), w.double()),
        lambda: decoding.linear(x[:, :0], w[:, :0]),
        lambda: decoding.linear(x, w[:0]),
        lambda: decoding.linear(torch.zeros((2, 4097), device=DEV), torch.zeros((2, 4097), device=DEV)),
        lambda: decoding.group_norm(image[0], 2),
        lambda: decoding.group_norm(image, 3),
        lambda: decoding.group_norm(image, 0),
        lambda: decoding.group_norm(image, True),
        lambda: decoding.group_norm(image, 2.0),
        lambda: decoding.group_norm(image, 2, torch.ones(7, device=DEV)),
        lambda: decoding.group_norm(image, 2, torch.ones(8, device=DEV).half()),
        lambda: decoding.group_norm(image, 2, eps=0.0),
        lambda: decoding.group_norm(image, 2, eps=math.nan),
        lambda: decoding.group_norm(image, 2, activation="swish"),
        lambda: decoding.group_norm(image, 2, checkpoint="fp8"),
        lambda: decoding.group_norm(image.int(), 2),
        lambda: decoding.quantize_activations(x.int()),
        lambda: decoding.quantize_activations(x.cpu()),
        lambda: decoding.FeatureDecoder(8, 30, 4, groups=8),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {i} was accepted")
    y = decoding.linear(x.requires_grad_(True), w, b, activation="silu")
    (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def _plain_decoder(decoder, features):
    """FeatureDecoder's formula with torch, in 64 bits."""
    h = features.double()
    p = lambda t: t.detach().double()
    h = ref.activate(h @ p(decoder.weights[0]).T + p(decoder.biases[0]), decoder.activation)
    for i in range(len(decoder.scales)):
        v = h.reshape(-1, h.shape[-3] * h.shape[-2], decoder.groups, h.shape[-1] // decoder.groups)
        m = v.mean((1, 3), keepdim=True)
        a = ((v - m) / ((v - m).square().mean((1, 3), keepdim=True) + 1e-5).sqrt()).reshape(h.shape)
        a = ref.activate(a * p(decoder.scales[i]) + p(decoder.shifts[i]), decoder.activation)
        h = a @ p(decoder.weights[i + 1]).T + p(decoder.biases[i + 1]) + h
    return h @ p(decoder.weights[-1]).T + p(decoder.biases[-1])


@pytest.mark.parametrize("checkpoint", (None, "int8"))
def test_decoder_trains_on_rendered_features(checkpoint):
    torch.manual_seed(0)
    scene = synthetic.make_scene("feat32", n=3000, width=120, height=88, seed=3).to(DEV)
    features = scene.features.clone().requires_grad_(True)
    decoder = decoding.FeatureDecoder(32, 48, 20, blocks=2, groups=6, checkpoint=checkpoint, device=DEV)
    teacher = torch.randn((1, 88, 120, 20), device=DEV)
    params = [features, *decoder.parameters()]
    optimiser = torch.optim.Adam(params, lr=5e-3)
    losses = []
    for step in range(25):
        res = gs3d.rasterize(scene.means, scene.quats, scene.scales, scene.opacities, scene.viewmats, scene.Ks,
                             scene.width, scene.height, features=features)
        out = decoder(res.features)
        if step == 0:
            want = _plain_decoder(decoder, res.features.detach())
            # Five products of at most 48 terms and two norms in 32 bits.
            assert ((out.double() - want).norm() / want.norm()).item() < 1e-5
        loss = (out - teacher).square().mean()
        optimiser.zero_grad()
        loss.backward()
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in params)
        optimiser.step()
        losses.append(loss.item())
    assert features.grad.abs().sum() > 0
    assert losses[-1] < 0.98 * losses[0], losses


def test_decoder_gradients():
    """Against autograd through the plain formula in 64 bits."""
    torch.manual_seed(1)
    decoder = decoding.FeatureDecoder(16, 24, 10, blocks=1, groups=4, activation="gelu", device=DEV)
    x = torch.randn((2, 20, 30, 16), device=DEV, requires_grad=True)
    up = torch.randn((2, 20, 30, 10), device=DEV)
    got = torch.autograd.grad(decoder(x), [x, *decoder.parameters()], up)
    wide = [t.detach().double().requires_grad_(True) for t in (x, *decoder.parameters())]
    xs, w0, w1, w2, b0, b1, b2, s, t = wide
    h = ref.activate(xs @ w0.T + b0, "gelu")
    v = h.reshape(2, 600, 4, 6)
    m = v.mean((1, 3), keepdim=True)
    a = ((v - m) / ((v - m).square().mean((1, 3), keepdim=True) + 1e-5).sqrt()).reshape(h.shape) * s + t
    out = (ref.activate(a, "gelu") @ w1.T + b1 + h) @ w2.T + b2
    want = torch.autograd.grad(out, wide, up.double())
    for a, c in zip(got, want):
        # Sums of at most 1200 rows of 32-bit products: far inside 1e-4 of the gradient's size.
        assert ((a.double() - c).norm() / c.norm()).item() < 1e-4
