"""``expert_linear`` on the GPU against its formulas in 64 bits: every path (few positions, fp32 tiles,
tensor cores, padded copies), form, activation, type and gradient, with experts that have all rows,
some or none.

Bounds (U = 2^-24, half = half a step of the type): an fp32 sum of k products is off by at most
(2 k + 32) U of the sum of magnitudes (tensor cores may drop the last place of each addition). The
activations' slopes are below 1.13, their second derivatives below 1.2, and they and the few operations
around them are off by 32 U of the values involved. Results that are weighted and added are held in fp32. dz is rounded to the type before the
products."""

from __future__ import annotations

import dataclasses
import math

import pytest
import torch

from mlx_diffuser_b200 import ExpertRoutes, _native as N
from mlx_diffuser_b200 import expert_linear, linear, route

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0**-24
F64 = torch.float64
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = [None, "silu", "gelu", "gelu_tanh"]
CURVE = 1.2


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def _act(z, name):
    if name == "silu":
        g = torch.sigmoid(z)
        return z * g, g * (1 + z * (1 - g))
    if name == "gelu":
        p = torch.special.ndtr(z)
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(8 / math.pi)
        g = torch.sigmoid(c * (z + 0.044715 * z**3))
        return z * g, g + z * g * (1 - g) * c * (1 + 3 * 0.044715 * z * z)
    return z, torch.ones_like(z)


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def _routes(n, e, k, seed=0, how="mixed"):
    g = torch.Generator(device=DEV).manual_seed(seed + 100)
    x = torch.randn((n, e), device=DEV, generator=g)
    if how == "mixed":  # uneven shares, and rows without an expert
        x += 1.5 * torch.randn((e,), device=DEV, generator=g)
        x[torch.rand((n,), device=DEV, generator=g) < 0.1] = float("-inf")
    elif how == "one":  # one expert has everything that it can
        x[:, e // 2] += 100
    elif how == "none":
        x[:] = float("-inf")
    return route(x, k)


class _Reference:
    """The formulas in 64 bits, with bounds."""

    def __init__(self, x, w, b, routes, act, gather, combine):
        self.args = x, w, b, routes, act, gather, combine
        n, k = routes.experts.shape
        e, o, i = w.shape
        dtype = x.dtype
        self.token = (routes.order.long() // k)
        self.spans = list(zip(routes.offsets.tolist()[:-1], routes.offsets.tolist()[1:]))
        self.p = routes.weights.detach().to(F64)
        self.place = routes.place.long()
        x64 = x.detach().to(F64)
        self.xp = x64[self.token] if gather else x64
        self.z = torch.zeros((n * k, o), dtype=F64, device=DEV)
        mag = torch.zeros_like(self.z)
        for j, (s, t) in enumerate(self.spans):
            self.z[s:t] = self.xp[s:t] @ w[j].detach().to(F64).T
            mag[s:t] = self.xp[s:t].abs() @ w[j].detach().to(F64).abs().T
            if b is not None:
                self.z[s:t] += b[j].detach().to(F64)
                mag[s:t] += b[j].detach().to(F64).abs()
        self.r, self.slope = _act(self.z, act)
        self.z_bound = (2 * i + 32) * U * mag
        behind = self.spans[-1][1]
        self.r[behind:] = 0
        self.r_bound = 1.13 * self.z_bound + 32 * U * (self.r.abs() + self.z.abs())
        self.r_bound[behind:] = 0
        bound = self.r_bound
        if combine:
            there = (self.place >= 0)[..., None]
            at = self.place.clamp(min=0)
            terms = self.r[at] * self.p[..., None] * there
            self.out = terms.sum(1)
            self.bound = (bound[at] * self.p[..., None] * there).sum(1) + 2 * k * U * terms.abs().sum(1)
            self.bound = self.bound * 1.01 + 1.01 * _half(dtype) * self.out.abs() + _tiny(dtype)
        else:
            self.out, self.bound = self.r, bound + _half(dtype) * 1.01 * self.r.abs() + _tiny(dtype)

    def gradients(self, dy):
        x, w, b, routes, act, gather, combine = self.args
        dtype = x.dtype
        h = 1.01 * _half(dtype)
        n, k = routes.experts.shape
        e, o, i = w.shape
        dy = dy.to(F64)
        share = self.p.reshape(-1)[routes.order.long()][:, None]
        dr = dy[self.token] * share if combine else dy.clone()
        behind = self.spans[-1][1]
        dr[behind:] = 0
        dz = dr * self.slope
        off = 4 * U * dz.abs()
        if act is not None:
            off = off + dr.abs() * (CURVE * self.z_bound + 32 * U * (1 + self.z.abs()))
        held = off + (h * dz.abs() if act is not None or combine else 0)
        dx, dx_bound = torch.zeros_like(self.xp), torch.zeros_like(self.xp)
        dw, dw_bound = (torch.zeros(w.shape, dtype=F64, device=DEV) for _ in range(2))
        db, db_bound = (torch.zeros((e, o), dtype=F64, device=DEV) for _ in range(2))
        for j, (s, t) in enumerate(self.spans):
            w64 = w[j].detach().to(F64)
            dx[s:t] = dz[s:t] @ w64
            dx_bound[s:t] = (held[s:t] + (2 * o + 32) * U * dz[s:t].abs()) @ w64.abs()
            dw[j] = dz[s:t].T @ self.xp[s:t]
            dw_bound[j] = (held[s:t] + (2 * (t - s) + 32) * U * dz[s:t].abs()).T @ self.xp[s:t].abs()
            db[j] = dz[s:t].sum(0)
            db_bound[j] = (off[s:t] + (t - s + 32) * U * dz[s:t].abs()).sum(0)
        if gather:
            at, there = self.place.clamp(min=0), (self.place >= 0)[..., None]
            dx_bound = ((dx_bound[at] + k * U * dx[at].abs()) * there).sum(1)
            dx = (dx[at] * there).sum(1)
        dx_bound = dx_bound * 1.01 + h * dx.abs() + _tiny(dtype)
        out = {"x": (dx, dx_bound), "weight": (dw, dw_bound + h * dw.abs() + _tiny(dtype)),
               "bias": (db, db_bound + h * db.abs() + _tiny(dtype))}
        if combine:
            there = self.place >= 0
            at = self.place.clamp(min=0)
            dp = torch.einsum("no,njo->nj", dy, self.r[at]) * there
            size = torch.einsum("no,njo->nj", dy.abs(), self.r[at].abs())
            dp_bound = torch.einsum("no,njo->nj", dy.abs(), self.r_bound[at]) + (o + 32) * U * size
            out["weights"] = (dp, dp_bound * there)
        return out


def _close(got, want, bound, what):
    err = (got.detach().to(F64) - want).abs()
    assert got.shape == want.shape, what
    assert not torch.isnan(err).any(), what
    assert (err <= bound).all(), (what, float((err / bound.clamp(min=1e-300)).max()))


def _inputs(n, e, k, i, o, dtype, gather, seed=0):
    x = _rand((n if gather else n * k, i), dtype, seed + 1)
    return x, _rand((e, o, i), dtype, seed + 2, i**-0.5), _rand((e, o), dtype, seed + 3, 0.5)


FORMS = [(True, False), (False, True), (True, True), (False, False)]  # gather, combine
SHAPES = [
    # rows, experts, choices, inputs, outputs
    (1, 4, 2, 64, 200), (1, 16, 1, 331, 517), (3, 5, 2, 8, 1), (7, 3, 3, 1, 9), (16, 8, 2, 512, 256),  # few
    (17, 2, 2, 64, 64), (40, 40, 1, 72, 136), (200, 3, 1, 128, 256), (301, 7, 2, 331, 517),
    (1000, 8, 2, 256, 64), (129, 1, 1, 64, 40), (2000, 5, 3, 40, 1031), (5000, 4, 2, 1024, 512),
    (64, 300, 2, 96, 64),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
def test_forward(shape, dtype):
    n, e, k, i, o = shape
    for f, (gather, combine) in enumerate(FORMS):
        x, w, b = _inputs(n, e, k, i, o, dtype, gather, f)
        act, bias = ACTS[f], (b if f != 1 else None)
        for how in ("mixed", "one"):
            routes = _routes(n, e, k, f, how)
            got = expert_linear(x, w, routes, bias, activation=act, gather=gather, combine=combine)
            assert got.dtype == dtype
            ref = _Reference(x, w, bias, routes, act, gather, combine)
            _close(got, ref.out, ref.bound, (how, gather, combine))
    N.check_device_status(DEV)


def _step(x, w, b, routes, dy, act, gather, combine):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    b = None if b is None else b.detach().requires_grad_(True)
    p = routes.weights.detach().requires_grad_(combine)
    routes = dataclasses.replace(routes, weights=p)
    y = expert_linear(x, w, routes, b, activation=act, gather=gather, combine=combine)
    leaves = {"x": x, "weight": w, "bias": b, "weights": p if combine else None}
    leaves = {name: t for name, t in leaves.items() if t is not None}
    return y, dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))


@pytest.mark.parametrize("shape", [(1, 4, 2, 64, 200), (7, 3, 2, 33, 65), (40, 40, 1, 72, 136),
                                   (301, 7, 2, 331, 517), (1000, 8, 2, 256, 64), (129, 1, 1, 64, 40),
                                   (3000, 4, 2, 512, 768), (64, 300, 2, 96, 64)], ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients(shape, dtype):
    n, e, k, i, o = shape
    for f, (gather, combine) in enumerate(FORMS):
        x, w, b = _inputs(n, e, k, i, o, dtype, gather, f)
        for act in (ACTS[f], ACTS[(f + 2) % 4]):
            routes = _routes(n, e, k, f)
            dy = _rand((n if combine else n * k, o), dtype, 50)
            bias = b if f != 2 else None
            y, grads = _step(x, w, bias, routes, dy, act, gather, combine)
            ref = _Reference(x, w, bias, routes, act, gather, combine)
            _close(y, ref.out, ref.bound, "y")
            for name, (g, bound) in ref.gradients(dy).items():
                if name in grads:
                    _close(grads[name], g, bound, (name, act, gather, combine))
    N.check_device_status(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", ["one", "none"])
def test_experts_without_rows(dtype, how):
    for n in (9, 300):
        for gather, combine in FORMS:
            x, w, b = _inputs(n, 6, 1, 72, 136, dtype, gather)
            routes = _routes(n, 6, 1, 0, how)
            dy = _rand((n, 136), dtype, 51)
            y, grads = _step(x, w, b, routes, dy, "silu", gather, combine)
            ref = _Reference(x, w, b, routes, "silu", gather, combine)
            _close(y, ref.out, ref.bound, "y")
            for name, (g, bound) in ref.gradients(dy).items():
                if name in grads:
                    _close(grads[name], g, bound, name)
            idle = [j for j in range(6) if how == "none" or j != 3]
            assert (grads["weight"][idle] == 0).all() and (grads["bias"][idle] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_neighbours_values_stay_with_it(dtype):
    """NaN in one expert's weights and rows reaches no other expert's results or gradients: tiles
    run past an expert's rows and matrices."""
    n, e, i, o = 300, 4, 72, 200
    routes = _routes(n, e, 1, 3, "even")
    spans = list(zip(routes.offsets.tolist()[:-1], routes.offsets.tolist()[1:]))
    for bad in range(e):
        s, t = spans[bad]
        x, w, b = _inputs(n, e, 1, i, o, dtype, False)
        dy = _rand((n, o), dtype, 52)
        want_y, want = _step(x, w, b, routes, dy, "gelu", False, False)
        x[s:t], w[bad], dy[s:t] = float("nan"), float("nan"), float("inf")
        y, grads = _step(x, w, b, routes, dy, "gelu", False, False)
        others = torch.ones(n, dtype=torch.bool, device=DEV)
        others[s:t] = False
        rest = [j for j in range(e) if j != bad]
        assert torch.equal(y[others], want_y[others]) and y[s:t].isnan().all()
        if dtype != torch.float16:
            assert torch.equal(grads["x"][others], want["x"][others])
            assert torch.equal(grads["weight"][rest], want["weight"][rest])
            assert torch.equal(grads["bias"][rest], want["bias"][rest])
            continue
        # fp16's dz is raised by a power of two that goes by the largest finite |dy|, here another one: values
        # below 2^-28 of it round differently, by at most 2^-39 of it each, which is far below the bounds'
        # own smallest step (2^-24) after 200 products with weights below 1
        x, w, b = _inputs(n, e, 1, i, o, dtype, False)
        dy = _rand((n, o), dtype, 52)
        exact = _Reference(x, w, b, routes, "gelu", False, False).gradients(dy)
        for name, at in (("x", others), ("weight", rest), ("bias", rest)):
            _close(grads[name][at], *(v[at] for v in exact[name]), name)


def test_same_as_linear_for_one_expert():
    for dtype in DTYPES:
        x, w, b = _inputs(500, 1, 1, 128, 256, dtype, True)
        routes = _routes(500, 1, 1, 0, "even")
        got = expert_linear(x, w, routes, b, activation="silu", gather=True)
        want = linear(x, w[0], b[0], activation="silu").to(F64)
        mag = x.to(F64).abs() @ w[0].to(F64).abs().T + b.to(F64).abs()
        bound = 2 * _half(dtype) * 1.01 * want.abs() + 2 * 1.13 * (2 * 128 + 32) * U * mag
        assert ((got.to(F64) - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_views(dtype):
    n, e, k, i, o = 120, 5, 2, 64, 72
    routes = _routes(n, e, k)
    x, w, b = _inputs(n, e, k, i, o, dtype, True)
    want = expert_linear(x, w, routes, b, gather=True)
    wide = torch.zeros((n, 3 * i), dtype=dtype, device=DEV)
    big = torch.zeros((e, o + 3, i + 8), dtype=dtype, device=DEV)
    for shift in (0, 1, 8):
        wide[:, shift:shift + i] = x
        big[:, 1:o + 1, shift:shift + i] = w
        got = expert_linear(wide[:, shift:shift + i], big[:, 1:o + 1, shift:shift + i], routes, b, gather=True)
        assert torch.equal(got, want)
    # (experts, K, N) weights, transposed; columns and experts that are repeated
    got = expert_linear(x, w.transpose(1, 2).contiguous().transpose(1, 2), routes, b, gather=True)
    assert torch.equal(got, want)
    got = expert_linear(x, w[:1].expand(e, o, i), routes, b[:1].expand(e, o), gather=True)
    assert torch.equal(got, expert_linear(x, w[:1].repeat(e, 1, 1), routes, b[:1].repeat(e, 1), gather=True))
    dy = _rand((n * k, o), dtype, 3)
    _, a = _step(x, w, b, routes, dy, None, True, False)
    _, c = _step(x, w, b, routes, dy.t().contiguous().t(), None, True, False)
    assert all(torch.equal(a[name], c[name]) for name in a)
    shifted = torch.zeros(n * k * o + 1, dtype=dtype, device=DEV)[1:].view(n * k, o)
    shifted.copy_(dy)  # off its 16-byte boundary
    _, c = _step(x, w, b, routes, shifted, None, True, False)
    assert all(torch.equal(a[name], c[name]) for name in a)


def test_empty_sizes():
    for dtype in DTYPES:
        for n, i, o in ((0, 64, 64), (40, 0, 64), (40, 64, 0), (100, 0, 7)):
            for gather, combine in FORMS:
                routes = _routes(n, 3, 2)
                x, w, b = _inputs(n, 3, 2, max(i, 1), o, dtype, gather)
                x, w = x[:, :i], w[:, :, :i]
                dy = _rand((n if combine else 2 * n, o), dtype, 3)
                y, grads = _step(x, w, b, routes, dy, "silu", gather, combine)
                ref = _Reference(x, w, b, routes, "silu", gather, combine)
                _close(y, ref.out, ref.bound, "y")
                for name, (g, bound) in ref.gradients(dy).items():
                    if name in grads:
                        _close(grads[name], g, bound, name)


def test_small_gradients_in_half_precision():
    """Gradients of a mean over many outputs lie where fp16 has few bits left: dz is raised first."""
    n, e, k, i, o = 600, 4, 2, 128, 256
    x, w, b = _inputs(n, e, k, i, o, torch.float16, True)
    routes = _routes(n, e, k)
    for combine in (False, True):
        dy = _rand((n if combine else n * k, o), torch.float16, 9, 2.0**-12)
        _, grads = _step(x, w, b, routes, dy, "gelu", True, combine)
        ref = _Reference(x, w, b, routes, "gelu", True, combine)
        for name, (g, bound) in ref.gradients(dy).items():
            _close(grads[name], g, bound, name)


def test_any_subset_of_gradients():
    n, e, k, i, o = 200, 4, 2, 64, 72
    x, w, b = _inputs(n, e, k, i, o, torch.bfloat16, True)
    routes = _routes(n, e, k)
    dy = _rand((n, o), torch.bfloat16, 4)
    _, want = _step(x, w, b, routes, dy, "silu", True, True)
    full = {"x": x, "weight": w, "bias": b, "weights": routes.weights}
    for mask in range(1, 16):
        t = {name: v.detach().requires_grad_(bool(mask >> j & 1))
             for j, (name, v) in enumerate(full.items())}
        y = expert_linear(t["x"], t["weight"], dataclasses.replace(routes, weights=t["weights"]), t["bias"],
                          activation="silu", gather=True, combine=True)
        names = [name for j, name in enumerate(full) if mask >> j & 1]
        got = torch.autograd.grad(y, [t[name] for name in names], dy)
        assert all(torch.equal(a, want[name]) for a, name in zip(got, names))


def test_same_results_every_time():
    n, e, k, i, o = 3000, 8, 2, 256, 512
    x, w, b = _inputs(n, e, k, i, o, torch.bfloat16, True)
    routes = _routes(n, e, k)
    dy = _rand((n, o), torch.bfloat16, 5)
    y, first = _step(x, w, b, routes, dy, "gelu", True, True)
    for _ in range(3):
        y2, again = _step(x, w, b, routes, dy, "gelu", True, True)
        assert torch.equal(y, y2) and all(torch.equal(first[name], again[name]) for name in first)


def test_routes_of_other_makings():
    """Entries that are no slot or position count as nothing and are reported; offsets are taken into
    range. Two choices of a row may be the same expert."""
    n, e, k, i, o = 100, 4, 2, 64, 72
    x, w, _ = _inputs(n, e, k, i, o, torch.bfloat16, True)
    twice = torch.arange(n * k, dtype=torch.int32, device=DEV)
    r = ExpertRoutes(torch.full((n, k), 2, dtype=torch.int32, device=DEV),
                     torch.full((n, k), 0.5, device=DEV), twice,
                     torch.tensor([0, 0, 0, n * k, n * k], dtype=torch.int32, device=DEV),
                     twice.view(n, k))
    y = expert_linear(x, w, r, gather=True, combine=True)
    want = linear(x, w[2])
    assert torch.equal(y, want)
    N.check_device_status(DEV)
    bad = dataclasses.replace(r, order=torch.where(twice % 3 == 0, 10**6, twice - 400 * (twice % 3 == 1)).int())
    y = expert_linear(x, w, bad, gather=True)
    with pytest.raises(RuntimeError, match="out of range"):
        N.check_device_status(DEV)
    assert (y[0::3] == 0).all() and (y[1::3] == 0).all()
    assert torch.equal(y[2::3], want.repeat_interleave(2, 0)[2::3])
    bad = dataclasses.replace(r, place=torch.where(twice % 2 == 0, -5, 10**6).int().view(n, k))
    assert (expert_linear(x, w, bad, gather=True, combine=True) == 0).all()
    bad = dataclasses.replace(r, offsets=torch.tensor([-7, 50, 20, 10**9, 3], dtype=torch.int32, device=DEV))
    y = expert_linear(x, w, bad, gather=True)
    # an offset below one before it is that one: experts 0 and 2 have positions 0 to 49 and the others
    rows = [linear(x, w[j]).repeat_interleave(2, 0) for j in (0, 2)]
    assert torch.equal(y[:50], rows[0][:50]) and torch.equal(y[50:], rows[1][50:])
    for dtype in DTYPES:
        x2, w2, b2 = _inputs(n, e, k, i, o, dtype, False)
        good = dataclasses.replace(r, offsets=torch.tensor([0, 50, 50, n * k, n * k], dtype=torch.int32, device=DEV))
        dy = _rand((n * k, o), dtype, 2)
        a, c = (_step(x2, w2, b2, q, dy, "silu", False, False) for q in (bad, good))
        assert torch.equal(a[0], c[0]) and all(torch.equal(a[1][name], c[1][name]) for name in c[1])
    _step(x, w, _rand((e, o), torch.bfloat16, 1), bad, _rand((n, o), torch.bfloat16, 2), "silu", True, True)
    torch.cuda.synchronize()


def test_routes_made_under_inference_mode():
    n, e, k, i, o = 90, 4, 2, 64, 72
    x, w, b = _inputs(n, e, k, i, o, torch.bfloat16, True)
    logits, dy = _rand((n, e), torch.float32, 3), _rand((n, o), torch.bfloat16, 4)
    want = _step(x, w, b, route(logits, k), dy, "silu", True, True)
    with torch.inference_mode():
        held = route(logits.clone(), k)
        assert held.order.is_inference()
        y = expert_linear(x, w, held, b, activation="silu", gather=True, combine=True)
    assert torch.equal(y, want[0])
    xg = x.detach().requires_grad_(True)
    y = expert_linear(xg, w, held, b, activation="silu", gather=True, combine=True)
    (dx,) = torch.autograd.grad(y, (xg,), dy)
    assert torch.equal(dx, want[1]["x"])


def test_gradients_against_differences():
    n, e, k, i, o = 12, 3, 2, 20, 24
    x, w, b = _inputs(n, e, k, i, o, torch.float32, True)
    routes = _routes(n, e, k, 0, "even")
    dy = _rand((n, o), torch.float32, 6)
    _, grads = _step(x, w, b, routes, dy, "gelu", True, True)
    step = 2.0**-9
    for name, t in (("x", x), ("weight", w), ("bias", b), ("weights", routes.weights)):
        way = _rand(t.shape, torch.float32, 7)
        sides = []
        for sign in (1, -1):
            moved = t + sign * step * way
            y = expert_linear(moved if name == "x" else x, moved if name == "weight" else w,
                              dataclasses.replace(routes, weights=moved) if name == "weights" else routes,
                              moved if name == "bias" else b, activation="gelu", gather=True, combine=True)
            sides.append(float((y.to(F64) * dy).sum()))
        slope = float((grads[name].to(F64) * way).sum())
        scale = float(dy.abs().sum())
        # outputs below 8 with (2 i + 64) U each, and the curvature's share of a central difference
        bound = (8 * (2 * i + 64) * U / step + step**2 * 200) * scale
        assert abs((sides[0] - sides[1]) / (2 * step) - slope) <= bound, name


def test_block_of_experts_with_its_router():
    """The operators as they are used together: border, router, both products, border; gradients of
    everything against the same steps in 64 bits."""
    from mlx_diffuser_b200 import block_norm

    n, c, e, k, hidden = 700, 64, 6, 2, 128
    # the choice of experts must not hang on a rounding: logits from fixed values
    logits = _rand((n, e), torch.float32, 20)
    args = {"x": _rand((n, c), torch.float32, 21), "branch": _rand((n, c), torch.float32, 22),
            "logits": logits, "gate": _rand((c,), torch.float32, 23), "scale": _rand((c,), torch.float32, 24, 0.3),
            "shift": _rand((c,), torch.float32, 25, 0.3), "up": _rand((e, hidden, c), torch.float32, 26, c**-0.5),
            "up_bias": _rand((e, hidden), torch.float32, 27), "down": _rand((e, c, hidden), torch.float32, 28, 0.1)}

    def own(a):
        y, h = block_norm(a["x"], a["branch"], gate=a["gate"], scale=a["scale"], shift=a["shift"])
        r = route(a["logits"], k)
        z = expert_linear(y, a["up"], r, a["up_bias"], activation="gelu_tanh", gather=True)
        f = expert_linear(z, a["down"], r, combine=True)
        return block_norm(h, f, norm="rms", gate=a["gate"])

    def plain(a):
        def layer(v):
            return torch.nn.functional.layer_norm(v, (c,), eps=1e-6)

        h = a["x"] + a["gate"] * a["branch"]
        y = layer(h) * (1 + a["scale"]) + a["shift"]
        top, at = torch.topk(a["logits"], k)
        p = torch.softmax(top, -1)
        f = 0
        for j in range(k):
            z = torch.einsum("nc,nhc->nh", y, a["up"][at[:, j]]) + a["up_bias"][at[:, j]]
            z = torch.nn.functional.gelu(z, approximate="tanh")
            f = f + p[:, j, None] * torch.einsum("nh,nch->nc", z, a["down"][at[:, j]])
        h = h + a["gate"] * f
        return h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt(), h

    dy, dh = _rand((n, c), torch.float32, 30), _rand((n, c), torch.float32, 31)
    out = []
    for run, t in ((own, torch.float32), (plain, F64)):
        leaves = {name: v.to(t).requires_grad_(True) for name, v in args.items()}
        y, h = run(leaves)
        out.append([y, h, *torch.autograd.grad((y, h), list(leaves.values()), (dy.to(t), dh.to(t)))])
    for name, got, want in zip(("y", "h", *args), *out):
        # a dozen fp32 steps over sums of up to 700 terms: 2^-24 * 1400 of the whole
        err = float((got.detach().to(F64) - want.detach()).norm() / want.detach().norm())
        assert err <= 1400 * U, (name, err)
    N.check_device_status(DEV)


def test_captured_step_and_two_at_once():
    n, e, k, i, o = 900, 6, 2, 128, 192
    x, w, b = _inputs(n, e, k, i, o, torch.bfloat16, True)
    logits = _rand((n, e), torch.float32, 40)
    dy = _rand((n, o), torch.bfloat16, 41)
    routes = route(logits, k)
    want = _step(x, w, b, routes, dy, "silu", True, True)
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            _step(x, w, b, route(logits, k), dy, "silu", True, True)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(_step(x, w, b, route(logits, k), dy, "silu", True, True))
            graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = _step(x, w, b, routes, dy, "silu", True, True)
        torch.cuda.synchronize()
        for y, grads in (*outs, eager):
            assert torch.equal(y, want[0])
            assert all(torch.equal(grads[name], want[1][name]) for name in want[1])
    N.check_device_status(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
def test_most_experts(dtype):
    for n in (50, 3000):
        x, w, b = _inputs(n, 1024, 2, 40, 48, dtype, True)
        routes = _routes(n, 1024, 2)
        dy = _rand((n, 48), dtype, 8)
        y, grads = _step(x, w, b, routes, dy, "gelu", True, True)
        ref = _Reference(x, w, b, routes, "gelu", True, True)
        _close(y, ref.out, ref.bound, "y")
        for name, (g, bound) in ref.gradients(dy).items():
            _close(grads[name], g, bound, name)


def test_results_past_32_bits():
    """Offsets beyond 2^31 elements of the results: the last rows are what their formula gives."""
    n, e, i, o = 2**19 + 3, 4, 64, 4112
    x, w, b = _inputs(n, e, 1, i, o, torch.bfloat16, True)
    logits = torch.zeros((n, e), device=DEV)
    logits[torch.arange(n, device=DEV), torch.arange(n, device=DEV) * e // n] = 1  # in the experts' order
    routes = route(logits, 1)
    y = expert_linear(x, w, routes, b, activation="silu", gather=True)
    rows = x[-64:].to(F64)
    z = rows @ w[e - 1].to(F64).T + b[e - 1].to(F64)
    bound = (2 * i + 64) * U * (rows.abs() @ w[e - 1].to(F64).abs().T + b[e - 1].to(F64).abs())
    want = _act(z, "silu")[0]
    _close(y[-64:], want, 1.2 * bound + 1.01 * _half(torch.bfloat16) * want.abs() + _tiny(torch.bfloat16), "y")
    del y
    y = expert_linear(x, w[:, :2056], routes, b[:, :2056], gather=True, combine=True)
    want = z[:, :2056]
    _close(y[-64:], want, bound[:, :2056] + 1.01 * _half(torch.bfloat16) * want.abs() + _tiny(torch.bfloat16), "y")


def _made(chosen, e, offsets=None):
    """Routes of the given experts (-1: none), made by hand: a row may name one expert more than once."""
    n, k = len(chosen), len(chosen[0])
    keys = torch.tensor(chosen).flatten()
    keys = torch.where(keys < 0, e, keys)
    order = torch.sort(keys, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(n * k)
    place = torch.where(keys < e, place, -1).view(n, k)
    if offsets is None:
        offsets = [0, *torch.bincount(keys, minlength=e + 1)[:e].cumsum(0).tolist()]
    weights = torch.rand((n, k), generator=torch.Generator().manual_seed(n + k)) + 0.1
    return ExpertRoutes(*(t.to(DEV, kind) for t, kind in (
        (torch.tensor(chosen), torch.int32), (weights, torch.float32), (order, torch.int32),
        (torch.tensor(offsets), torch.int32), (place, torch.int32))))


def _poison(*shapes):
    """Memory that the next tensors of these shapes are likely to get is filled with NaN."""
    held = [torch.full(shape, float("nan"), dtype=t, device=DEV)
            for shape in (*shapes, (2**15,), (2**21,)) for t in DTYPES for _ in range(4)]
    del held


def _check_all(x, w, b, routes, act, gather, combine, seed=60):
    n, k = routes.experts.shape
    o = w.shape[1]
    dy = _rand((n if combine else n * k, o), x.dtype, seed)
    _poison((n, o), (n * k, o), (n * k, x.shape[1]), x.shape, w.shape)
    y, grads = _step(x, w, b, routes, dy, act, gather, combine)
    ref = _Reference(x, w, b, routes, act, gather, combine)
    _close(y, ref.out, ref.bound, "y")
    for name, (g, bound) in ref.gradients(dy).items():
        if name in grads:
            _close(grads[name], g, bound, (name, act, gather, combine))
    _poison((n, o), (n * k, o))
    with torch.no_grad():
        again = expert_linear(x, w, routes, b, activation=act, gather=gather, combine=combine)
    assert torch.equal(y, again)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("chosen", [[2, 2], [1, 3, 1], [0] * 8, [3, 2, 3, -1, 2], [1] * 9, [2] * 32,
                                    [0, 1, 2, 3] * 8, [1] * 40], ids=lambda c: f"{len(c)}:{c[:4]}")
def test_one_row_that_names_an_expert_more_than_once(dtype, chosen):
    e = 4
    for i, o in ((64, 200), (33, 65), (64, 1)):
        for f, (gather, combine) in enumerate(FORMS):
            x, w, b = _inputs(1, e, len(chosen), i, o, dtype, gather, f)
            _check_all(x, w, b if f else None, _made([chosen], e), ACTS[f], gather, combine)
    N.check_device_status(DEV)


@pytest.mark.parametrize("how", ["checkpoint", "host"])
def test_saved_tensors_that_come_back_as_others(how):
    from mlx_diffuser_b200 import dropout
    from tests.test_block_norm_gpu import _hooked

    n, e, k, i, o = 200, 4, 2, 64, 72
    x, w, b = (t.requires_grad_(True) for t in _inputs(n, e, k, i, o, torch.bfloat16, True))
    logits = _rand((n, e), torch.float32, 5).requires_grad_(True)
    wide = _rand((e, o, 2 * i), torch.bfloat16, 6).requires_grad_(True)

    def run(x, w, b, logits, wide):
        r = route(2 * logits, k)
        z = expert_linear(x * 2, wide[:, :, i:], r, b, activation="silu", gather=True)
        z = expert_linear(z, w.transpose(1, 2), r, combine=True)
        return dropout(z, 0.25, torch.tensor(3, device=DEV), residual=x)

    leaves, outs = [x, w, b, logits, wide], []
    dy = _rand((n, i), torch.bfloat16, 7)
    for j in range(2):
        y = _hooked(how, run, *leaves) if j else run(*leaves)
        spill = [torch.full((n * k, 2 * i), float("nan"), device=DEV) for _ in range(16)]
        outs.append((y, *torch.autograd.grad(y, leaves, dy)))
        del spill
    for a, c in zip(*outs):
        assert torch.equal(a, c)
    N.check_device_status(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, offsets", [(100, [10, 50, 50, 120, 120]), (100, [200, 200, 200, 200, 200]),
                                        (700, [1, 300, 300, 1300, 1399]), (700, [1400, 1400, 1400, 1400, 1400]),
                                        (3, [1, 2, 2, 4, 5]), (1, [1, 1, 2, 2, 2]), (2, [4, 4, 4, 4, 4])],
                         ids=str)
def test_positions_that_no_expert_has(dtype, n, offsets):
    """Before the first offset and behind the last one: zeros, in the results and in x's gradient, and a place
    there counts as none. Nothing is read that was not written."""
    e = 4
    g = torch.Generator().manual_seed(n)
    routes = _made(torch.randint(0, e, (n, 2), generator=g).tolist(), e, offsets)
    for i, o in ((64, 72), (33, 65)):
        for f, (gather, combine) in enumerate(FORMS):
            x, w, b = _inputs(n, e, 2, i, o, dtype, gather, f)
            _check_all(x, w, b, routes, ACTS[f], gather, combine)
    N.check_device_status(DEV)


@pytest.mark.parametrize("scale", [2.0**-14, 1.0, 17.0, 500.0, 2.0**20])
def test_large_and_small_weights_in_half_precision(scale):
    """dz holds the products of dy and the weights: their range is taken into account, not dy's alone."""
    n, e, k, i, o = 300, 4, 2, 72, 136
    x, w, b = _inputs(n, e, k, i, o, torch.float16, True)
    routes = _routes(n, e, k)
    routes = dataclasses.replace(routes, weights=routes.weights * scale)
    for act in (None, "gelu"):
        # the result itself has to stay in the type's range
        x1, w1 = (x, w * min(1.0, 2.0**-9 * 500 / scale)) if act is None else (x * 2.0**-10, w)
        dy = _rand((n, o), torch.float16, 9, 2.0**-4 / max(1.0, scale / 100))
        _, grads = _step(x1, w1, None, routes, dy, act, True, True)
        ref = _Reference(x1, w1, None, routes, act, True, True)
        for name, (g, bound) in ref.gradients(dy).items():
            if name in grads:
                assert torch.isfinite(grads[name]).all(), (name, act)
                _close(grads[name], g, bound, (name, act))


def test_a_weight_that_is_no_number_stays_with_its_row():
    n, e, k, i, o = 300, 4, 2, 72, 136
    x, w, b = _inputs(n, e, k, i, o, torch.float16, True)
    routes = _routes(n, e, k, 0, "even")
    dy = _rand((n, o), torch.float16, 9)
    want = _Reference(x, w, b, routes, "silu", True, True).gradients(dy)["x"]
    for bad in (float("inf"), float("nan")):
        weights = routes.weights.clone()
        weights[7] = bad
        y, grads = _step(x, w, b, dataclasses.replace(routes, weights=weights), dy, "silu", True, True)
        others = torch.arange(n, device=DEV) != 7
        assert torch.isfinite(y[others]).all() and not torch.isfinite(grads["x"][7]).any()
        _close(grads["x"][others], *(v[others] for v in want), bad)


@pytest.mark.parametrize("outputs", [64, 65])
@pytest.mark.parametrize("dtype", DTYPES)
def test_long_sums_behind_the_weights_gradients(dtype, outputs):
    """One sum on the tensor cores loses its last place at each of its k / 16 additions, always downwards.
    x in [1, 2) with 7 bits behind the point and weights there with 5: products have 12 and a run of
    512 of them is below 2^11, 23 bits, exact. What is left is the runs' addition, k / 512 roundings of U
    each (fp32 products: k / 16 of them, and one more at the end of a thread's own terms). In one sum the
    result needs 28 bits: 1,024 cuts of half a place of 2 U on average, at half of the sum's size each, are
    500 U."""
    n, e, k = 40, 2, 16384
    g = torch.Generator(device=DEV).manual_seed(4)
    x = (1 + torch.randint(0, 128, (n, k), device=DEV, generator=g) / 128).to(dtype)
    w = (1 + torch.randint(0, 32, (e, outputs, k), device=DEV, generator=g) / 32).to(dtype)
    routes = _routes(n, e, 1, 0, "even")
    expert = routes.experts[:, 0].long()
    for column in (0, 37, outputs - 1):
        dy = torch.zeros((n, outputs), dtype=dtype, device=DEV)
        dy[:, column] = 1  # the gradient is the column of the results
        p = routes.weights.detach().requires_grad_(True)
        y = expert_linear(x, w, dataclasses.replace(routes, weights=p), gather=True, combine=True)
        (got,) = torch.autograd.grad(y, (p,), dy)
        want = (x.to(F64) * w.to(F64)[expert, column]).sum(1)
        bound = (k / 512 + 1 if dtype != torch.float32 else k / 16 + 1) * U * want
        _close(got[:, 0], want, bound, column)


@pytest.mark.parametrize("shape", [(3000, 4, 2, 1100, 512), (700, 3, 1, 2048, 264), (200, 8, 2, 520, 200),
                                   (900, 2, 1, 331, 1000), (60, 5, 2, 4160, 136)], ids=str)
@pytest.mark.parametrize("dtype", DTYPES[1:])
def test_gradients_with_long_sums(shape, dtype):
    n, e, k, i, o = shape
    for f, (gather, combine) in enumerate(FORMS):
        x, w, b = _inputs(n, e, k, i, o, dtype, gather, f)
        routes = _routes(n, e, k, f)
        dy = _rand((n if combine else n * k, o), dtype, 50)
        for act in (None, ACTS[1 + f % 3]):
            y, grads = _step(x, w, b, routes, dy, act, gather, combine)
            ref = _Reference(x, w, b, routes, act, gather, combine)
            _close(y, ref.out, ref.bound, "y")
            for name, (g, bound) in ref.gradients(dy).items():
                if name in grads:
                    _close(grads[name], g, bound, (name, act, gather, combine))
    N.check_device_status(DEV)


def test_captured_step_with_long_sums_and_two_at_once():
    n, e, k, i, o = 700, 6, 2, 1100, 192
    x, w, b = _inputs(n, e, k, i, o, torch.bfloat16, True)
    routes = _routes(n, e, k)
    dy = _rand((n, o), torch.bfloat16, 41)
    for act in (None, "silu"):
        want = _step(x, w, b, routes, dy, act, True, True)
        streams = [torch.cuda.Stream() for _ in range(2)]
        graphs, outs = [], []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                _step(x, w, b, routes, dy, act, True, True)
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=s):
                    outs.append(_step(x, w, b, routes, dy, act, True, True))
                graphs.append(g)
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            eager = _step(x, w, b, routes, dy, act, True, True)
            torch.cuda.synchronize()
            for y, grads in (*outs, eager):
                assert torch.equal(y, want[0])
                assert all(torch.equal(grads[name], want[1][name]) for name in want[1])
    N.check_device_status(DEV)
