"""The decoder's products on both sides of the row counts and widths at which
their kernels change."""

import pytest
import torch

from dsl_splat_amd import decoding
from test_gpu_decoding_paths import _case, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("rows", (4095, 4097, 32767, 32769))
@pytest.mark.parametrize("inner,outer", [(40, 300), (200, 128), (200, 129), (300, 260)])
def test_rows_where_kernels_change(inner, outer, rows, dtype):
    print("linear", rows, inner, outer, dtype, flush=True)
    _check(*_case(rows, inner, outer, dtype, residual=outer % 2 == 0), "silu")
    _check(*_case(rows, inner, outer, dtype), "gelu", "int8")


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("inner,outer", [(300, 132), (129, 257), (512, 300), (400, 511)])
def test_many_strided_rows_against_packed_weights(inner, outer, dtype):
    """Rows further apart than they are long, bases off the vectors' grid, a last
    block that is not full."""
    print("linear", inner, outer, dtype, flush=True)
    x, w, b, r, up = _case(33333, inner, outer, dtype, residual=True)
    wide = lambda t: torch.cat((t[:, :3], t, t[:, :2]), 1)[:, 3:-2]
    _check(wide(x), w, b, wide(r), wide(up), "silu")


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("inner,outer", [(3, 5), (16, 100), (33, 40), (100, 70), (128, 2)])
@pytest.mark.parametrize("rows", (1, 17, 1000, 4096, 4097))
def test_eight_bits_kept_by_products_of_few_and_many_rows(rows, inner, outer, dtype):
    """The codes that a product keeps are those of quantize_activations: the same
    gradients to the bit as from the values read back."""
    print("linear int8", rows, inner, outer, dtype, flush=True)
    x, w, b, _, up = _case(rows, inner, outer, dtype)
    kept = decoding.quantize_activations(x).dequantize()
    got = []
    for value, checkpoint in ((x, "int8"), (kept, None)):
        leaves = [t.detach().requires_grad_(True) for t in (value, w, b)]
        got.append(torch.autograd.grad(decoding.linear(*leaves, activation="gelu", checkpoint=checkpoint), leaves, up))
    for a, c in zip(*got):
        assert torch.equal(a, c)
