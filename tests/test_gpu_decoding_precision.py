"""How near the decoder's results come to 64 bits where rounding is a choice:
the input gradients of 16-bit types, float16's range, float's activations."""

import pytest
import torch

import decoding_reference as ref
from dsl_splat_amd import decoding

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _normal(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


# One-pass backwards, then widths whose gradient at the activation's argument
# goes through memory, into products of every kind.
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("rows,inner,outer", [(20000, 32, 128), (20000, 128, 128), (3000, 33, 97), (4000, 256, 512),
                                              (4001, 300, 70), (2500, 512, 64), (900, 300, 600), (2000, 300, 201),
                                              (1500, 520, 700), (3000, 40, 257)])
def test_input_gradients_err_by_their_own_rounding(rows, inner, outer, dtype):
    """dz enters dx with an error of UNIT^2 in each term, so that of the result's
    one rounding, UNIT, is all that is left: the two norms agree to UNIT, far
    inside 2%."""
    print("linear", rows, inner, outer, dtype, flush=True)
    g = torch.Generator().manual_seed(rows + inner + outer)
    x, w = _normal(g, rows, inner, dtype=dtype), _normal(g, outer, inner, scale=inner ** -0.5, dtype=dtype)
    b, up = _normal(g, outer, scale=0.2, dtype=dtype), _normal(g, rows, outer, dtype=dtype)
    for kind, checkpoint in (("silu", None), ("gelu", "int8")):
        leaf = x.detach().requires_grad_(True)
        (got,) = torch.autograd.grad(decoding.linear(leaf, w, b, activation=kind, checkpoint=checkpoint), leaf, up)
        seen = ref.kept(x) if checkpoint else x
        want = ref.linear_grads(seen, w, b, up, kind)["x"][0]
        least = (want.to(dtype).double() - want).norm()
        assert (got.double() - want).norm() <= 1.02 * least, (kind, ((got.double() - want).norm() / least).item())


@pytest.mark.parametrize("inner,outer", [(40, 72), (300, 140)])
@pytest.mark.parametrize("kind", ("silu", "gelu"))
def test_gradients_beyond_the_range_of_float16(kind, inner, outer):
    """A slope above one takes an upstream gradient near float16's largest value
    past it, on the way to results that are well inside."""
    print("linear", kind, inner, outer, flush=True)
    g = torch.Generator().manual_seed(5)
    x = _normal(g, 1200, inner, dtype=torch.float16)
    w = _normal(g, outer, inner, scale=0.01 * inner ** -0.5, dtype=torch.float16)
    # Where the slope is largest.
    b = torch.full((outer,), {"silu": 2.4, "gelu": 1.4}[kind], dtype=torch.float16, device=DEV)
    up = torch.zeros((1200, outer), dtype=torch.float16, device=DEV)
    up[5, 3], up[5, 4], up[700, 9] = 65504.0, -65504.0, 65504.0
    x[5], x[700] = x[5] * 2 ** -5, x[700] * 2 ** -5
    leaves = [t.requires_grad_(True) for t in (x, w)]
    got = torch.autograd.grad(decoding.linear(*leaves, b, activation=kind), leaves, up)
    grads = ref.linear_grads(x.detach(), w.detach(), b, up, kind)
    for name, value in zip(("x", "weight"), got):
        ref.check(name, value, *grads[name])


@pytest.mark.parametrize("kind", ("silu", "gelu"))
@pytest.mark.parametrize("spread", (0.5, 2.0, 8.0))
def test_float_activations_are_as_exact_as_elementary_operations(kind, spread):
    """z passes through a product with one weight of 1, so the error is the
    activation's: in norm no more than half again what torch's exp, erf and
    divisions in 32 bits leave."""
    print(kind, spread, flush=True)
    g = torch.Generator().manual_seed(7)
    z = _normal(g, 1 << 18, 1, scale=spread)
    one = torch.ones((1, 1), device=DEV)
    leaf = z.detach().requires_grad_(True)
    y = decoding.linear(leaf, one, activation=kind)
    (dz,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    if kind == "silu":
        s = torch.sigmoid(z)
        plain = z * s, s * (1 + z * (1 - s))
    else:
        p = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        plain = z * p, p + z * torch.exp(-0.5 * z * z) * (2 * torch.pi) ** -0.5
    exact = ref.activate(z.double(), kind), ref.slope(z.double(), kind)
    for name, got, other, want in zip(("value", "slope"), (y.detach(), dz), plain, exact):
        mine, theirs = (got.double() - want).norm().item(), (other.double() - want).norm().item()
        print(name, mine / want.norm().item(), theirs / want.norm().item(), flush=True)
        assert mine <= 1.5 * theirs, (name, mine, theirs)


@pytest.mark.parametrize("kind", ("silu", "gelu"))
def test_float_activations_at_their_ends(kind):
    """Far arguments: z or 0, slopes 1 or 0, what is not finite as by the formula."""
    inf, nan = float("inf"), float("nan")
    z = torch.tensor([0.0, -0.0, 90.0, -90.0, 300.0, -300.0, 1e19, -1e19, 3e38, -3e38, inf, nan], device=DEV)[:, None]
    one = torch.ones((1, 1), device=DEV)
    leaf = z.detach().requires_grad_(True)
    y = decoding.linear(leaf, one, activation=kind)
    (dz,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    y, dz = y.detach().flatten(), dz.flatten()
    assert torch.equal(y[2:10:2], z[2:10:2, 0]) and (y[3:10:2].abs() < 1e-30).all() and not y[:2].any()
    assert torch.equal(dz[:2], torch.full((2,), 0.5, device=DEV))
    assert torch.equal(dz[2:10:2], torch.ones(4, device=DEV)) and (dz[3:10:2].abs() < 1e-30).all()
    assert y[10] == inf and y[11].isnan() and dz[11].isnan()
