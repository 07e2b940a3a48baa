"""``dropout`` on the GPU: the same elements as the generator in numpy drops, one rounding, and the same mask in
the backward pass.

Bounds: the factor is rounded to fp32 (2^-24), the product and the sum to fp32 (2^-24 each), the
result to its type (half a step)."""

from __future__ import annotations

import pytest
import torch

from mlx_diffuser_b200 import dropout
from tests.philox import factors, numbers

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0**-24
F64 = torch.float64
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
SEED = 0x9F3A5C7712345678


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def _factors(shape, p, seed=SEED, subsequence=0):
    n = int(torch.Size(shape).numel())
    return torch.from_numpy(factors(n, p, seed, subsequence)).to(DEV).view(shape)


def _check(got, x, f, r=None):
    want = x.to(F64) * f
    bound = 2 * U * want.abs()
    if r is not None:
        want = want + r.to(F64)
        bound = bound + U * want.abs()
    bound = bound * 1.01 + torch.finfo(got.dtype).eps / 2 * (want.abs() + bound)
    assert got.dtype == x.dtype and got.shape == x.shape
    assert ((got.to(F64) - want).abs() <= bound + torch.finfo(got.dtype).smallest_normal * 2**-10).all()
    if r is None:
        assert torch.equal(got == 0, (f == 0) | (x == 0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5), (64, 64), (301, 331), (5, 7, 513),
                                   (4097, 1024)])
def test_against_the_generator(shape, dtype):
    x, r = _rand(shape, dtype, 1), _rand(shape, dtype, 2, 2.0)
    for p in (0.1, 0.5):
        f = _factors(shape, p)
        _check(dropout(x, p, SEED), x, f)
        _check(dropout(x, p, SEED, residual=r), x, f, r)


def test_share_and_subsequence():
    x = torch.ones((1000, 1000), device=DEV)
    for p in (0.0, 2.0**-17, 2.0**-16, 0.25, 0.9, 1 - 2.0**-17, 1.0):
        y = dropout(x, p, SEED)
        assert torch.equal(y, _factors(x.shape, p).float())
    a, b = (dropout(x, 0.5, SEED, subsequence=s) for s in (2**40 + 3, 4))
    assert torch.equal(a, _factors(x.shape, 0.5, SEED, 2**40 + 3).float())
    assert torch.equal(b, _factors(x.shape, 0.5, SEED, 4).float())
    # independent: a quarter of the elements is kept in both (six standard deviations)
    both = ((a > 0) & (b > 0)).double().mean().item()
    assert abs(both - 0.25) < 6 * (0.25 * 0.75 / 1e6) ** 0.5


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients(dtype):
    for shape in ((5, 7), (331, 72), (1000, 129)):
        x, r = _rand(shape, dtype, 3).requires_grad_(True), _rand(shape, dtype, 4).requires_grad_(True)
        dy = _rand(shape, dtype, 5)
        f = _factors(shape, 0.3)
        dx, dr = torch.autograd.grad(dropout(x, 0.3, SEED, residual=r), (x, r), dy)
        _check(dx, dy, f)
        assert torch.equal(dr, dy)
        # a gradient that is broadcast, and one that is a transposed view
        (dx,) = torch.autograd.grad(dropout(x, 0.3, SEED).sum(), (x,))
        _check(dx, torch.ones(shape, device=DEV, dtype=dtype), f)
        (dx,) = torch.autograd.grad(dropout(x, 0.3, SEED), (x,), dy.t().contiguous().t())
        _check(dx, dy, f)


def test_values_that_are_dropped():
    """A dropped element is zero whatever it was; kept infinities and NaN stay."""
    x = torch.full((4096,), float("nan"), device=DEV)
    x[1::2] = float("inf")
    f = _factors(x.shape, 0.5)
    y = dropout(x, 0.5, SEED)
    assert torch.equal(y == 0, f == 0)
    assert torch.equal(y[f > 0].isnan(), x[f > 0].isnan())


def test_views_and_alignment():
    base = _rand((64, 65), torch.bfloat16, 6)
    flat = base.flatten()
    for x in (base.t(), base[:, 1:], base[::3], flat[1:], flat[3:1027], base[0], base[:0]):
        f = _factors(x.shape, 0.5)
        _check(dropout(x, 0.5, SEED), x, f)
        _check(dropout(x, 0.5, SEED, residual=x), x, f, x)


def test_seed_in_device_memory():
    x = _rand((100, 72), torch.float32, 7).requires_grad_(True)
    seed = torch.tensor([SEED - 2**64], device=DEV)
    want = dropout(x, 0.5, SEED)
    assert torch.equal(dropout(x, 0.5, seed), want)
    # changed before the backward pass: its mask would be another
    y = dropout(x, 0.5, seed)
    seed += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    # a captured step with another seed at every replay; torch cannot capture a backward pass while an
    # eager graph of the same leaf is alive on another stream
    del y
    x = x.detach().requires_grad_(True)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.autograd.grad(dropout(x, 0.5, seed).sum(), (x,))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y = dropout(x, 0.5, seed)
            (dx,) = torch.autograd.grad(y, (x,), torch.ones_like(y))
    torch.cuda.synchronize()
    for s in (5, 2**63 + 11):
        seed.fill_(s if s < 2**63 else s - 2**64)
        graph.replay()
        torch.cuda.synchronize()
        f = _factors(x.shape, 0.5, s)
        _check(y.detach(), x.detach(), f)
        assert torch.equal(dx, f.float())


def test_elements_past_32_bits():
    """Element numbers beyond 2^32 have their own random numbers."""
    n = 2**32 + 4096
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    y = dropout(x, 0.5, SEED)
    for first in (2**31 - 2048, 2**32 - 2048, n - 4096):
        want = torch.from_numpy(numbers(4096, SEED, 0, first) >= 32768).to(DEV)
        assert torch.equal(y[first:first + 4096] > 0, want)
