"""``linear``'s activations over the whole range of their argument: where squares and cubes overflow."""

from __future__ import annotations

import pytest
import torch

from mlx_diffuser_b200 import _native as N
from mlx_diffuser_b200 import linear

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_largest_arguments(act, dtype):
    """The value is z or 0 and the slope 1 or 0 wherever z is a number, though z^2 and z^3 overflow."""
    sizes = torch.tensor([1e4, 1e10, 3e12, 1e13, 1.7e19, 2e19, 1e25, 3e38], device=DEV)
    z = torch.cat([sizes, -sizes]).repeat(4).to(dtype)  # 64 rows: the tiles of either type
    x = z[:, None].clone().requires_grad_(True)
    one = torch.ones((1, 1), dtype=dtype, device=DEV)
    for a in (x, x[:6]):
        y = linear(a, one, activation=act)
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        n = len(a)
        up = z[:n] > 0
        assert torch.equal(y[:, 0][up], z[:n][up]) and not y[:, 0][~up].any()
        assert (dx[:n, 0][up] == 1).all() and not dx[:n, 0][~up].any()
    N.check_device_status(DEV)
