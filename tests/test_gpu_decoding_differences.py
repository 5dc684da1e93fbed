"""The decoder's gradients against central differences along a direction near
the gradient's own, so that every bound is a small part of the slope."""

import pytest
import torch

import decoding_reference as ref
from dsl_splat_amd import decoding

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _normal(g, *shape, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=g) * scale + shift).to(DEV)


@pytest.mark.parametrize("kind", ("silu", "gelu"))
def test_product(kind):
    """Differences of the operator's own forward in 32 bits.  They are off by
    h^2 / 6 of the third derivative (at most 2 a term), and by the forward's
    bound, twice over 2 h."""
    g = torch.Generator().manual_seed(91)
    x, w, b = _normal(g, 400, 20), _normal(g, 28, 20, scale=20 ** -0.5), _normal(g, 28, scale=0.3)
    up = _normal(g, 400, 28)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(decoding.linear(*leaves, activation=kind), leaves, up)
    exact = ref.linear_grads(x.detach(), w.detach(), b.detach(), up, kind)
    x, w, b = (t.detach() for t in leaves)
    h = 2.0 ** -6
    for i, name in enumerate(("x", "weight", "bias")):
        d = exact[name][0].float()
        along = (lambda: d @ w.T, lambda: x @ d.T, lambda: d.expand(400, 28))[i]()  # what the argument moves by
        d, along = d / along.square().mean().sqrt(), along.double() / along.double().square().mean().sqrt()
        values, noise = [], 0.0
        for sign in (1, -1):
            args = [x, w, b]
            args[i] = args[i] + sign * h * d
            moved = args[i].double() - (x, w, b)[i].double()  # as rounded
            values.append((decoding.linear(*args, activation=kind).double() * up.double()).sum().item())
            noise += (up.double().abs() * ref.linear(*args, None, kind)[1]).sum().item() / (2 * h)
            noise += (exact[name][0].abs() * (moved - sign * h * d.double()).abs()).sum().item() / (2 * h) * 2
        slope = (values[0] - values[1]) / (2 * h)
        cut = (up.double().abs() * 2 * along.abs() ** 3).sum().item() * h * h / 6
        own = (exact[name][1] * d.double().abs()).sum().item()
        mine = (grads[i].double() * d.double()).sum().item()
        bound = cut + noise + own
        print(kind, name, slope, mine, bound, flush=True)
        assert bound <= 0.05 * abs(slope)
        assert abs(slope - mine) <= bound


@pytest.mark.parametrize("kind", ("none", "silu", "gelu"))
def test_norm(kind):
    """Differences of the formula's forward in 64 bits, off by some h^2 of the
    slope and by roundings near 1e-12 / h of it, h = 1e-4: 1e-6 for both."""
    g = torch.Generator().manual_seed(92)
    x, up = _normal(g, 2, 9, 11, 24), _normal(g, 2, 9, 11, 24)
    w, b = _normal(g, 24, scale=0.3, shift=1.0), _normal(g, 24, scale=0.3)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(decoding.group_norm(x, 6, w, b, activation=kind), leaves, up)
    flat = lambda t: t.detach().double().reshape(2, 99, 24)
    x, w, b, up = flat(x), w.detach().double(), b.detach().double(), flat(up)
    exact = ref.Norm(x.float(), 6, w.float(), b.float(), 1e-5, kind).grads(x.float(), up)
    h = 1e-4
    for i, name in enumerate(("x", "weight", "bias")):
        d = exact[name][0] / exact[name][0].square().mean().sqrt()
        values = []
        for sign in (1, -1):
            args = [x, w, b]
            args[i] = args[i] + sign * h * d
            v = args[0].reshape(2, 99, 6, 4)
            unit = (v - v.mean((1, 3), keepdim=True)) / (v.var((1, 3), unbiased=False, keepdim=True) + 1e-5).sqrt()
            values.append((ref.activate(unit.reshape(2, 99, 24) * args[1] + args[2], kind) * up).sum().item())
        slope = (values[0] - values[1]) / (2 * h)
        mine = (grads[i].double().reshape(d.shape) * d).sum().item()
        bound = (exact[name][1] * d.abs()).sum().item() + 1e-6 * abs(slope)
        print(kind, name, slope, mine, bound, flush=True)
        assert bound <= 0.05 * abs(slope)
        assert abs(slope - mine) <= bound
