"""``linear``'s activations over the whole range of their argument, against the formulas in 64 bits,
relative to the result: what the tails keep, and where squares and cubes overflow.

Bounds, with u = 2^-24: exp, erfc, the divisions and the products around them are off by at most 16 u
together. The argument's own rounding is multiplied by the function: at most 8 u of t = 2 sqrt(2 / pi)
(z + 0.044715 z^3) by |t| for the tanh form, 2 u of z by z^2 for the normal integral. A factor below 2^-126 (the
logistic function, its slope, the integral, its density) is off by 2^-149, times what it is multiplied by: z,
and in the tanh form's slope z dt/dz."""

from __future__ import annotations

import math

import pytest
import torch

from mlx_diffuser_b200 import _native as N
from mlx_diffuser_b200 import linear

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0**-24
F64 = torch.float64


def _parts(z, name):
    """The activation, its slope, the sum of the slope's magnitudes, what the argument's rounding is
    multiplied by, in units of u, and what the slope's factor is."""
    if name == "silu":
        g, q = torch.sigmoid(z), torch.sigmoid(z) * torch.sigmoid(-z)
        return z * g, g + z * q, g + z.abs() * q, torch.zeros_like(z), z.abs()
    if name == "gelu":
        p = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        d = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * p, p + z * d, p + z.abs() * d, 2 * z * z, z.abs()
    t = math.sqrt(8 / math.pi) * (z + 0.044715 * z**3)
    g, q = torch.sigmoid(t), torch.sigmoid(t) * torch.sigmoid(-t)
    far = math.sqrt(8 / math.pi) * (1 + 3 * 0.044715 * z * z)
    return z * g, g + z * q * far, g + z.abs() * q * far, 8 * t.abs(), z.abs() * far


def _check(got, want, mag, amplified, times, z):
    # beyond 200 of it the result is below every number of the type (or the argument itself)
    rel = (16 + amplified.clamp(max=8 * 200)) * U
    bound = rel * mag + 4 * 2.0**-149 * (1 + times)
    err = (got.to(F64) - want).abs()
    assert (err <= bound).all(), (float((err / bound).max()), float(z[(err / bound).argmax()]))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("rows", [4001, 8])
def test_tails_in_fp32(act, rows):
    """z from -105 to 105: one product of x and 1, in tiles of 128 rows and by the path for few."""
    z = torch.linspace(-105, 105, 4001, device=DEV)
    if rows == 8:
        z = torch.tensor([-88.5, -80.25, -40.1, -13.3, -7.7, -3.1, 3.1, 40.1], device=DEV)
    x = z[:, None].clone().requires_grad_(True)
    one = torch.ones((1, 1), device=DEV)
    y = linear(x, one, activation=act)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    want, slope, mag, amplified, times = _parts(z.to(F64), act)
    _check(y.detach()[:, 0], want, want.abs(), amplified, z.to(F64).abs(), z)
    _check(dx[:, 0], slope, mag, amplified, times, z)


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
