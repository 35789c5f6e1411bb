"""Norms and linear layers at the ends of their ranges: types that are mixed, arguments far out, rows without any spread."""

import pytest
import torch

from miles_amd.kernels.norm import layer_norm
from tests.operator_checks import f64, within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALVES = [torch.bfloat16, torch.float16]


def _off(t):
    """t at an address that is no multiple of 16, its rows apart: what the native host layer leaves to Python."""
    big = torch.zeros(t.shape[0], t.shape[1] + 8, dtype=t.dtype, device=DEV)
    view = big[:, 3:3 + t.shape[1]]
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("place", [torch.Tensor.contiguous, _off], ids=["contiguous", "off"])
def test_the_gradient_of_an_fp32_bias_without_a_weight_is_fp32(place, dtype):
    """Sums of 100 rows, at most 100 2^-24 of the magnitudes off before the rounding to fp32; the largest is beyond fp16."""
    g = torch.Generator().manual_seed(1)
    x, dy = (place(torch.randn((100, 96), generator=g).to(dtype).to(DEV)) for _ in range(2))
    dy[:, 5] = 1000.0
    b = torch.randn(96, generator=g).to(DEV).requires_grad_(True)
    db = torch.autograd.grad(layer_norm(x, None, b), b, dy)[0]
    assert db.dtype == torch.float32 and db[5] == 100_000
    within(db, f64(dy).sum(0), 100 * 2.0**-24 * f64(dy).abs().sum(0), "db")
