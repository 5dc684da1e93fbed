"""Training steps of the decoder's operators on streams of their own and in
captured graphs, and norms of long images and wide groups."""

import pytest
import torch

import decoding_reference as ref
from dsl_splat_amd import decoding

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _tensors(seed, dtype, inner=40, outer=48, rows=3600):
    g = torch.Generator().manual_seed(seed)
    normal = lambda *shape, scale=1.0: (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)
    x, w = normal(rows, inner), normal(outer, inner, scale=inner ** -0.5)
    b, up = normal(outer, scale=0.3), normal(rows, outer)
    return [t.requires_grad_(True) for t in (x, w, b)], up


def _step(leaves, up, checkpoint):
    """A product and a norm, forward and backward."""
    y = decoding.linear(*leaves, activation="silu", checkpoint=checkpoint)
    n = decoding.group_norm(y.view(60, 60, -1), 6, activation="gelu", checkpoint=checkpoint)
    return [y.detach(), n.detach(), *torch.autograd.grad(n, leaves, up.view(n.shape))]


# One pass, three products of which one packs its weights, and wide ones.
WIDTHS = [(40, 48), (300, 72), (260, 510)]


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("inner,outer", WIDTHS)
@pytest.mark.parametrize("checkpoint", (None, "int8"))
def test_backward_on_another_stream(checkpoint, inner, outer, dtype):
    leaves, up = _tensors(71, dtype, inner, outer)
    want = _step(leaves, up, checkpoint)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = [torch.zeros_like(t) for t in leaves]
        torch.cuda._sleep(20_000_000)
        for a, t in zip(late, leaves):
            a.copy_(t.detach())
        got = _step([t.requires_grad_(True) for t in late], up, checkpoint)
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("inner,outer", WIDTHS)
@pytest.mark.parametrize("checkpoint", (None, "int8"))
def test_captured_training_steps(checkpoint, inner, outer, dtype):
    leaves, up = _tensors(72, dtype, inner, outer)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(leaves, up, checkpoint)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(leaves, up, checkpoint)
    for seed in range(4):
        others, gradient = _tensors(80 + seed, dtype, inner, outer)
        with torch.no_grad():
            for a, t in zip(leaves, others):
                a.copy_(t)
            up.copy_(gradient)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, _step(leaves, up, checkpoint)))
        torch.cuda.synchronize()


class _Long(ref.Norm):
    # 127 pixels a thread at most, then 512 strips' sums a thread at most, and
    # trees over both.
    RUN = 1200


@pytest.mark.parametrize("images,height,width,channels,groups", [(4, 540, 960, 64, 8), (1, 300, 400, 512, 1),
                                                                 (1, 700, 900, 64, 1), (3, 200, 100, 96, 2)])
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_long_norms(images, height, width, channels, groups, dtype):
    print("norm", images, height, width, channels, groups, dtype, flush=True)
    g = torch.Generator(DEV).manual_seed(channels)
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEV)
    x, up = (normal(images, height, width, channels) + 0.5).to(dtype), normal(images, height, width, channels).to(dtype)
    w, b = (normal(channels) * 0.3 + 1).to(dtype), (normal(channels) * 0.3).to(dtype)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = decoding.group_norm(leaves[0], groups, *leaves[1:], activation="silu")
    got = torch.autograd.grad(y, leaves, up)
    flat = lambda t: t.detach().reshape(images, height * width, channels)
    norm = _Long(flat(x), groups, w.detach(), b.detach(), 1e-5, "silu")
    ref.check("y", y, *norm.forward())
    grads = norm.grads(flat(x), flat(up))
    for name, value in zip(("x", "weight", "bias"), got):
        ref.check("grad " + name, value, *grads[name])
        # and far nearer than the bounds in the sum of all
        want = grads[name][0]
        off = (value.double().reshape(want.shape) - want).norm() / want.norm()
        assert off <= 2 * ref.UNIT[dtype] + 2.0 ** -20, (name, off.item())
