"""``route`` on the GPU: choices, order, offsets and places equal a stable sort's, whatever the ties, masks,
types and sizes; weights and their gradients against 64 bits.

Bounds (U = 2^-24): l - m is off by U |l - m| and the exponential by 2 ulp, a sum of up to 1024 of them
by 40 U (32 in a lane, five steps over the warp, the quotient): a weight by (48 + 2 |l - m|) U. The
gradient adds the warp sum of w dw, 40 U of the terms' magnitudes, twice."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mlx_diffuser_b200 import _native as N
from mlx_diffuser_b200 import ExpertRoutes, route

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0**-24
F64 = torch.float64
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _logits(n, e, dtype, seed, masked=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = 2 * torch.randn((n, e), device=DEV, generator=g)
    if masked:
        x[torch.rand((n, e), device=DEV, generator=g) < 0.2] = float("-inf")
        x[torch.rand((n,), device=DEV, generator=g) < 0.1] = float("-inf")
    return x.to(dtype)


def _oracle(logits, k):
    """experts, order, offsets, place, and the chosen logits, by numpy's stable sorts."""
    v = logits.detach().double().cpu().numpy()
    n, e = v.shape
    best = np.argsort(-v, axis=1, kind="stable")[:, :k]
    picked = np.take_along_axis(v, best, 1)
    experts = np.where(np.isneginf(picked), -1, best)
    keys = np.where(experts < 0, e, experts).reshape(-1)
    order = np.argsort(keys, kind="stable")
    place = np.empty(n * k, np.int64)
    place[order] = np.arange(n * k)
    place = np.where(experts < 0, -1, place.reshape(n, k))
    offsets = np.concatenate([[0], np.cumsum(np.bincount(keys, minlength=e + 1)[:e])])
    return experts, order, offsets, place, picked


def _check(r, logits, k, normalize=True):
    n, e = logits.shape
    experts, order, offsets, place, picked = _oracle(logits, k)
    assert (r.rows, r.choices, r.num_experts) == (n, k, e)
    for name, want in (("experts", experts), ("order", order), ("offsets", offsets), ("place", place)):
        got = getattr(r, name)
        assert got.dtype == torch.int32
        assert np.array_equal(got.cpu().numpy(), want), name
    l = torch.from_numpy(picked).to(DEV)
    all_ = l if normalize else logits.detach().to(F64)
    top = all_.amax(1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)  # subtracted first: a lowest value swallows a logarithm
    w = torch.exp(l - top) / torch.exp(all_ - top).sum(1, keepdim=True).clamp(min=1.0)
    far = torch.where(l == float("-inf"), 0.0, top - l)
    far = torch.nan_to_num(far, nan=0.0) + 20  # the others' distances, in the sum: e^-20 of it past that
    err = (r.weights.detach().to(F64) - w).abs()
    assert (err <= (48 + 2 * far) * U * w + 2.0**-126).all()
    return w


@pytest.mark.parametrize("e", [1, 2, 8, 31, 32, 33, 64, 100, 128, 256, 300, 1024])
@pytest.mark.parametrize("dtype", DTYPES)
def test_choices(e, dtype):
    for n in (1, 3, 100, 1000):
        for k in sorted({1, 2, min(e, 8), min(e, 32)}):
            if k > e:
                continue
            logits = _logits(n, e, dtype, n + k + e)
            for normalize in (True, False):
                _check(route(logits, k, normalize=normalize), logits, k, normalize)
    N.check_device_status(DEV)


@pytest.mark.parametrize("n,e,k", [(8191, 16, 2), (8193, 16, 2), (40662, 64, 4), (40662, 8, 2),
                                   (100003, 5, 3), (5000, 1024, 32), (300001, 256, 1)])
def test_many_rows(n, e, k):
    for dtype in (torch.float32, torch.bfloat16):
        logits = _logits(n, e, dtype, 7)
        _check(route(logits, k), logits, k)


def test_ties_zeros_and_lowest_values():
    x = torch.zeros((5, 40), device=DEV)
    x[1, ::2] = -0.0  # equal to zero
    x[2] = torch.finfo(torch.float32).min  # a mask of the lowest value is a logit like others
    x[3, 7:] = torch.finfo(torch.float32).min
    x[4] = float("-inf")
    r = route(x, 10)
    _check(r, x, 10)
    assert r.experts[0].tolist() == r.experts[1].tolist() == r.experts[2].tolist() == list(range(10))
    assert (r.weights[2] == r.weights[0]).all()
    assert (r.experts[4] == -1).all() and (r.weights[4] == 0).all()
    one = torch.full((70000, 6), 1.5, device=DEV)
    _check(route(one, 3), one, 3)


def test_not_finite():
    """NaN counts as the largest and gives NaN weights; +inf as in a softmax. Other rows do not see it."""
    x = _logits(4, 33, torch.float32, 1, masked=False)
    x[1, 20], x[2, 5] = float("nan"), float("inf")
    for normalize in (True, False):
        r = route(x, 3, normalize=normalize)
        assert r.experts[1, 0] == 20 and r.experts[2, 0] == 5
        assert r.weights[1].isnan().all() and r.weights[2].isnan().any()
        assert torch.isfinite(r.weights[[0, 3]]).all()
        assert ((r.place >= 0) & (r.place < 12)).all()
        assert r.offsets[-1] == 12 and torch.equal(r.order.sort().values.cpu(), torch.arange(12).int())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("normalize", [True, False])
def test_gradients(dtype, normalize):
    for n, e, k in ((1, 1, 1), (7, 8, 2), (33, 64, 32), (200, 100, 4), (50, 1024, 8)):
        logits = _logits(n, e, dtype, e).requires_grad_(True)
        r = route(logits, k, normalize=normalize)
        w = _check(r, logits, k, normalize)
        g = torch.Generator(device=DEV).manual_seed(3)
        dw = torch.randn((n, k), device=DEV, generator=g)
        (got,) = torch.autograd.grad(r.weights, (logits,), dw)
        dw64 = dw.to(F64)
        dot, size = (w * dw64).sum(1, keepdim=True), (w * dw64).abs().sum(1, keepdim=True)
        want, bound = torch.zeros_like(logits, dtype=F64), torch.zeros_like(logits, dtype=F64)
        at = r.experts.long().clamp(min=0)
        if normalize:
            want.scatter_add_(1, at, w * (dw64 - dot))
        else:
            l = logits.detach().to(F64)
            total = torch.logsumexp(l, 1, keepdim=True)
            p = torch.exp(l - torch.where(total == float("-inf"), 0.0, total))
            want.scatter_add_(1, at, w * dw64)
            want, bound = want - p * dot, bound + p * size
        bound.scatter_add_(1, at, w * (dw64.abs() + size))
        # logits here differ by less than 20: a weight is off by (48 + 2 * 40) U
        bound = 400 * U * bound + 1.01 * torch.finfo(dtype).eps / 2 * want.abs() + \
            torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert got.dtype == dtype and ((got.to(F64) - want).abs() <= bound).all()


def test_gradients_against_differences():
    logits = _logits(20, 12, torch.float32, 5, masked=False).requires_grad_(True)
    g = torch.Generator(device=DEV).manual_seed(6)
    dw, way = (torch.randn(s, device=DEV, generator=g) for s in ((20, 3), (20, 12)))
    for normalize in (True, False):
        r = route(logits, 3, normalize=normalize)
        (grad,) = torch.autograd.grad(r.weights, (logits,), dw)
        step = 2.0**-10  # no choice changes
        a, b = (route(logits.detach() + s * step * way, 3, normalize=normalize) for s in (1, -1))
        assert torch.equal(a.experts, b.experts) and torch.equal(a.experts, r.experts)
        slope = float(((a.weights - b.weights).to(F64) * dw).sum()) / (2 * step)
        scale = float(dw.abs().sum())
        assert abs(slope - float((grad.to(F64) * way).sum())) <= (200 * U / step + 20 * step**2) * scale


def test_views_and_no_rows():
    wide = _logits(50, 100, torch.bfloat16, 8)
    for x in (wide[:, 3:40], wide[::2], wide.t()[:50], wide[:0], wide[:, :1].expand(50, 20)):
        _check(route(x, 2), x, 2)
    x = wide[:, 3:40].detach().requires_grad_(True)
    (g,) = torch.autograd.grad(route(x, 2).weights.sum(), (x,))
    assert g.shape == x.shape


def test_captured_and_on_another_stream():
    logits = _logits(20000, 32, torch.float32, 9)
    other = _logits(20000, 32, torch.float32, 10)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    held = logits.clone()
    with torch.cuda.stream(stream):
        _check(route(held, 2), logits, 2)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            r = route(held, 2)
    for x in (other, logits):
        held.copy_(x)
        torch.cuda.synchronize()
        graph.replay()
        eager = route(other, 2)
        torch.cuda.synchronize()
        _check(r, x, 2)
        _check(eager, other, 2)
    assert isinstance(r, ExpertRoutes)
