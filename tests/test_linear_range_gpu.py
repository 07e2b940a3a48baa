"""``linear``'s activations over the whole range of their argument, against the formulas in 64 bits,
relative to the result: what the tails keep, and where squares and cubes overflow.

Bounds, with u = 2^-24: exp, erfc, the divisions and the products around them are off by at most 16 u
together. The argument's own rounding is multiplied by the function: at most 8 u of t = 2 sqrt(2 / pi)
(z + 0.044715 z^3) by |t| for the tanh form, 2 u of z by z^2 for the normal integral. A factor below 2^-126 (the
logistic function, its slope, the integral, its density) is off by 2^-149, times what it is multiplied by: z,
and in the tanh form's slope z dt/dz.

Gradients of 16-bit types: dz is rounded by half a step e of itself, in fp16 after it is raised, so that below
2^-28 of the largest |dy| it is off by 2^-39 of that at most; its slope by (2 k + 16) u of |x||w| + |b| through
z (the slopes' own slopes are below 1.2) and 32 u (1 + |z|) by the approximate exponential; a sum of t
products by 2 t u. The two roundings of dx and dw, dz's and the result's, are independent and of half a step each:
2^0.5 of the result's alone as a whole, and 2 with room for the rest."""

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


@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-6])
@pytest.mark.parametrize("shape", [(2048, 128, 192), (2047, 72, 331), (300, 40, 24)], ids=str)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_small_output_gradients(shape, act, size, dtype):
    """A mean loss's output gradients, down to fp16's smallest numbers."""
    m, k, n = shape
    gen = torch.Generator(device=DEV).manual_seed(m + k)

    def rand(*s, scale=1.0):
        return (torch.randn(s, device=DEV, generator=gen) * scale).to(dtype)

    x, w, b, dy = rand(m, k), rand(n, k, scale=k**-0.5), rand(n), rand(m, n, scale=size)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(linear(x, w, b, activation=act), leaves, dy)
    N.check_device_status(DEV)
    e = torch.finfo(dtype).eps / 2
    least = torch.finfo(dtype).smallest_normal * e
    with torch.no_grad():
        x64, w64, b64, g = (t.to(F64) for t in (x, w, b, dy))
        z = x64 @ w64.T + b64
        dz = g * _parts(z, act)[1]
        small = 2.0**-39 * float(g.abs().max()) if dtype == torch.float16 else 2.0**-126
        off = e * dz.abs() + small + (1 + e) * g.abs() * (
            1.2 * (2 * k + 16) * U * (x64.abs() @ w64.abs().T + b64.abs())
            + 32 * U * (1 + z.abs()))
        for name, got, want, o, mag, terms in (
            ("dx", grads[0], dz @ w64, off @ w64.abs(), dz.abs() @ w64.abs(), n),
            ("dw", grads[1], dz.T @ x64, off.T @ x64.abs(), dz.abs().T @ x64.abs(), m),
            ("db", grads[2], dz.sum(0), off.sum(0), dz.abs().sum(0), m),
        ):
            total = o + (2 * terms + 16) * U * (mag + o)
            bound = total + e * (want.abs() + total) + least
            err = (got.to(F64) - want).abs()
            assert (err <= bound).all(), (name, float((err / bound).max()))
            alone = (want.to(dtype).to(F64) - want).norm()
            assert err.norm() <= 2 * alone, (name, float(err.norm() / alone))


@pytest.mark.parametrize("shape", [(300, 40, 24), (64, 8, 7)], ids=str)
def test_output_gradients_that_are_zero_large_or_not_finite(shape):
    m, k, n = shape
    x = torch.ones((m, k), device=DEV, dtype=torch.float16, requires_grad=True)
    w = torch.full((n, k), 1 / k, device=DEV, dtype=torch.float16, requires_grad=True)
    y = linear(x, w, activation="gelu_tanh")
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y), retain_graph=True)
    assert not dx.any() and not dw.any()
    dy = torch.zeros_like(y)
    dy[3, 2] = 60000.0  # slope 1.083: more than the type holds, though not its products with w
    dx, = torch.autograd.grad(y, x, dy, retain_graph=True)
    want = 60000 * float(_parts(torch.ones(1, dtype=F64), "gelu_tanh")[1]) * float(w[2, 0].detach())
    assert (dx[3].to(F64) - want).abs().max() <= 2.0**-9 * want and not dx[:3].any()
    dy[3, 2] = float("inf")
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert torch.isinf(dx[3]).all() and not dx[4:].any() and not dx[:3].any()
    assert torch.isinf(dw[2]).all() and not dw[3:].any() and not dw[:2].any()


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gradients_are_taken_at_the_unrounded_argument(act, dtype):
    """Around the slope's zero an argument rounded to the type would show: half a step of z, times a second
    derivative near one, where dz and its own rounding all but vanish."""
    gen = torch.Generator(device=DEV).manual_seed(3)
    root = {"silu": -1.2784645, "gelu": -0.7517916, "gelu_tanh": -0.7524614}[act]
    x = (root + 0.02 * torch.randn((4096, 1), device=DEV, generator=gen)).to(dtype)
    w = torch.full((1, 1), 1.0234375, dtype=dtype, device=DEV)  # products need twice the type's bits
    x.requires_grad_(True)
    y = linear(x, w, activation=act)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    e = torch.finfo(dtype).eps / 2
    with torch.no_grad():
        z, w64 = x.to(F64) * w.to(F64), w.to(F64)
        dz = _parts(z, act)[1]
        off = e * dz.abs() + (1 + e) * (1.2 * 18 * U * z.abs() + 32 * U * (1 + z.abs()))
        if dtype == torch.float16:
            off += 2.0**-39  # the least of what it was raised to
        want = dz * w64
        err = (dx.to(F64) - want).abs()
        bound = off * w64 + e * (want.abs() + off * w64) + 2.0**-25
        assert (err <= bound).all(), float((err / bound).max())
        # and this would not pass at the rounded argument
        rounded = _parts(z.to(dtype).to(F64), act)[1] * w64
        assert ((rounded - want).abs() > bound).double().mean() > 0.25
