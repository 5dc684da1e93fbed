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
    b = torch.full((outer,), {"silu": 2.4, "gelu": 1.4}[kind], dtype=torch.float16, device=DEV)  # where the slope is largest
    up = torch.zeros((1200, outer), dtype=torch.float16, device=DEV)
    up[5, 3], up[5, 4], up[700, 9] = 65504.0, -65504.0, 65504.0
    x[5], x[700] = x[5] * 2 ** -5, x[700] * 2 ** -5
    leaves = [t.requires_grad_(True) for t in (x, w)]
    got = torch.autograd.grad(decoding.linear(*leaves, b, activation=kind), leaves, up)
    grads = ref.linear_grads(x.detach(), w.detach(), b, up, kind)
    for name, value in zip(("x", "weight"), got):
        ref.check(name, value, *grads[name])
