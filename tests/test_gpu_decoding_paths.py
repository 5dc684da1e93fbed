"""The products of the feature decoder over the widths and row counts at which
their kernels change, and what the parameters' gradients owe to the halves that
the gradient at the activation's argument is split into."""

import pytest
import torch
from torch.autograd import forward_ad

import decoding_reference as ref
from dsl_splat_amd import decoding

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = (torch.float32, torch.bfloat16, torch.float16)
KINDS = ("none", "relu", "silu", "gelu")


def _normal(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def _case(rows, inner, outer, dtype, residual=False):
    g = torch.Generator().manual_seed(1000 * inner + outer + rows)
    x, w = _normal(g, rows, inner, dtype=dtype), _normal(g, outer, inner, scale=inner ** -0.5, dtype=dtype)
    b, up = _normal(g, outer, scale=0.3, dtype=dtype), _normal(g, rows, outer, dtype=dtype)
    return x, w, b, _normal(g, rows, outer, dtype=dtype) if residual else None, up


def _split_grads(x, w, b, up, kind):
    """{name: (gradient, bound)} for the weight and the bias where a 16-bit dz
    enters as two halves: the high one errs by UNIT |dz|, the low one by UNIT of
    that (or by float16's TINY), and there are twice the terms."""
    dtype = w.dtype
    lead, w, dy = x.double(), w.double(), up.double()
    b = torch.zeros(w.shape[0], dtype=torch.float64, device=w.device) if b is None else b.double()
    z = lead @ w.T + b
    err_z = (lead.shape[-1] + 2) * ref.U * (lead.abs() @ w.abs().T + b.abs())
    dz = dy * ref.slope(z, kind)
    if kind == "none":
        err = torch.zeros_like(dz)
    elif kind == "relu":
        err = dy.abs() * (z.abs() <= err_z)
    else:
        err = dy.abs() * (ref.CURVE * err_z + ref.ACT * z.abs().clamp_min(1))
        err = err + ref.U * (dz.abs() + err)
        if dtype != torch.float32:
            err = err + ref.UNIT[dtype] ** 2 * (dz.abs() + err) + ref.TINY[dtype]
    terms = (2 * dz.shape[0] + 2) * ref.U
    out = {"weight": (dz.T @ lead, err.T @ lead.abs() + terms * (dz.abs().T @ lead.abs())),
           "bias": (dz.sum(0), err.sum(0) + terms * dz.abs().sum(0))}
    return {k: (v, ref._rounded(v, e, dtype)) for k, (v, e) in out.items()}


def _check(x, w, b, r, up, kind, checkpoint=None):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = decoding.linear(*leaves, activation=kind, residual=r, checkpoint=checkpoint)
    ref.check("y", y, *ref.linear(x, w, b, r, kind))
    if checkpoint is None:  # without autograd: the same kernels
        assert torch.equal(decoding.linear(x, w, b, activation=kind, residual=r), y)
    got = dict(zip(("x", "weight", "bias"), torch.autograd.grad(y, leaves, up)))
    seen = ref.kept(x).reshape(x.shape) if checkpoint else x
    want = {**ref.linear_grads(seen, w, b, up, kind), **_split_grads(seen, w, b, up, kind)}
    for name, value in got.items():
        ref.check("grad " + name, value, *want[name])


# Every pair of widths that the one-pass backward knows, at their ends.
FUSED = [(32, 32), (9, 33), (17, 128), (32, 256), (33, 31), (64, 64), (50, 100), (64, 256), (128, 20), (65, 64),
         (128, 128), (100, 65), (256, 32), (129, 40), (200, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inner,outer", FUSED)
def test_one_pass_backward(inner, outer, dtype):
    for rows, kind in ((1, "gelu"), (191, "silu"), (2050, KINDS[(inner + outer) % 4])):
        print("linear", rows, inner, outer, dtype, kind, flush=True)
        _check(*_case(rows, inner, outer, dtype), kind)


# Rows enough for blocks that take several steps each, the last one short.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inner,outer", [(16, 24), (64, 128), (128, 128), (256, 64), (48, 256)])
def test_one_pass_backward_of_many_rows(inner, outer, dtype):
    print("linear", inner, outer, dtype, flush=True)
    _check(*_case(133333, inner, outer, dtype), "silu")


LONG = [(2000, 129, 8), (1100, 257, 9), (1500, 300, 70), (1025, 512, 259), (3001, 400, 64), (2500, 65, 300),
        (1030, 513, 40), (1500, 700, 130), (40, 600, 70), (1, 1000, 5), (2100, 300, 5), (2100, 520, 3)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer", LONG)
def test_long_and_wide_products(rows, inner, outer, dtype):
    kind = KINDS[1 + (rows + inner + outer) % 3]
    print("linear", rows, inner, outer, dtype, kind, flush=True)
    _check(*_case(rows, inner, outer, dtype, residual=True), kind)
    _check(*_case(rows, inner, outer, dtype), "none", "int8")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer", [(3000, 3, 3), (3000, 2, 100), (3000, 100, 2), (3000, 3, 400), (5000, 1, 1)])
def test_rows_shorter_than_a_vector(rows, inner, outer, dtype):
    print("linear", rows, inner, outer, dtype, flush=True)
    _check(*_case(rows, inner, outer, dtype, residual=True), "silu")
    _check(*_case(rows, inner, outer, dtype), "gelu", "int8")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inner,outer", [(300, 72), (40, 300), (600, 33)])
def test_strided_long_products(inner, outer, dtype):
    """Rows further apart than they are long, and bases off the vectors' grid."""
    print("linear", inner, outer, dtype, flush=True)
    x, w, b, r, up = _case(1300, inner, outer, dtype, residual=True)
    wide = lambda t: torch.cat((t[:, :3], t, t[:, :2]), 1)[:, 3:-2]
    _check(wide(x), w, b, wide(r), wide(up), "silu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inner,outer", [(40, 72), (300, 140)])
def test_single_gradients(inner, outer, dtype):
    """Each gradient alone is the one that all together give."""
    print("linear", inner, outer, dtype, flush=True)
    for kind in ("none", "silu"):
        x, w, b, _, up = _case(1200, inner, outer, dtype)
        tensors = {"x": x, "weight": w, "bias": b}
        leaves = [t.detach().requires_grad_(True) for t in tensors.values()]
        together = torch.autograd.grad(decoding.linear(*leaves, activation=kind), leaves, up)
        for name, whole in zip(tensors, together):
            alone = {n: t.detach().requires_grad_(n == name) for n, t in tensors.items()}
            y = decoding.linear(*alone.values(), activation=kind)
            assert torch.equal(torch.autograd.grad(y, alone[name], up)[0], whole), (kind, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inner,outer", [(40, 72), (300, 140)])
def test_infinite_gradients_stay_in_their_row_and_channel(inner, outer, dtype):
    """An infinity is not split into itself and a NaN."""
    print("linear", inner, outer, dtype, flush=True)
    x, w, b, _, up = _case(1200, inner, outer, dtype)
    up[7, 3] = float("inf")
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(decoding.linear(*leaves, activation="silu"), leaves, up)
    slope = ref.slope(x[7].double() @ w[3].double() + b[3].double(), "silu")
    hit = torch.zeros(1200, dtype=torch.bool, device=DEV)
    hit[7] = True
    assert torch.isfinite(dx[~hit]).all() and torch.equal(dx[7].double(), float("inf") * slope * w[3].double())
    assert torch.equal(dw[3].double(), float("inf") * slope * x[7].double())
    assert torch.isfinite(torch.cat((dw[:3], dw[4:]))).all()
    assert db[3].double() == float("inf") * slope and torch.isfinite(torch.cat((db[:3], db[4:]))).all()


def test_forward_mode_is_refused():
    """A tangent is never dropped without a word."""
    x, w, b, _, _ = _case(64, 16, 16, torch.float32)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises((RuntimeError, NotImplementedError)):
            decoding.linear(dual, w, b)
        with pytest.raises((RuntimeError, NotImplementedError)):
            decoding.group_norm(forward_ad.make_dual(x.reshape(8, 8, 16), torch.ones_like(x).reshape(8, 8, 16)), 4)
