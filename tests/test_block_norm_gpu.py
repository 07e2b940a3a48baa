"""``block_norm`` on the GPU against its formulas in 64 bits, over the row widths where the kernel changes its
layout, each option, and the gradients of all that it reads.

Bounds (U = 2^-24, half = half a step of the feature type). A thread adds at most 32 elements of a row
before the sums are joined pairwise and over eight warps, so a row's sums are off by at most 64 U of
the sums of magnitudes, and the mean and rstd, with the square root and quotients, by 96 U. N(v) is then
off by e = 96 U (mean|v| rstd + |N(v)|). y and h are compared at the h that came back, so that one
rounding does not hide in the next. In the gradients the row means carry e into D: each of the terms
dy a, mean(dy a), N mean(dy a N) is off by at most 400 U of its magnitude with e's two parts taken
as 1 + |N| (the inputs' mean|v| rstd is below 1). What is normed twice has those bounds twice. The column
sums of n rows add n + 64 roundings."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mlx_diffuser_b200 import _native as N
from mlx_diffuser_b200 import block_norm
from tests.philox import factors

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0**-24
F64 = torch.float64
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
SEED = 0x1234567890ABCDEF
COEFS = ("weight", "bias", "branch_weight", "gate", "scale", "shift")


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _case(n, c, dtype, seed, batch=3, per_batch=True, names=COEFS, kind=None):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rand(shape, mean, scale, t):
        return (mean + scale * torch.randn(shape, device=DEV, generator=g)).to(t)

    a = {"x": rand((n, c), 0.0, 2.0, dtype), "branch": rand((n, c), 0.1, 1.0, dtype)}
    rows = (batch, c) if per_batch else (c,)
    for name, shape, mean, scale in (
            ("weight", (c,), 1.0, 0.3), ("bias", (c,), 0.0, 0.3), ("branch_weight", (c,), 1.0, 0.3),
            ("gate", rows, 0.3, 0.5), ("scale", rows, 0.0, 0.3), ("shift", rows, 0.0, 0.3)):
        r = rand(shape, mean, scale, kind or dtype)
        if name in names:
            a[name] = r
    a["branch_norm"] = "branch_weight" in names
    coords = torch.zeros((n, 4), dtype=torch.int32, device=DEV)
    coords[:, 0] = torch.randint(0, batch, (n,), device=DEV, generator=g).sort().values
    a["coords"] = coords
    if per_batch:
        a["batch_size"] = batch
    dy, dh = rand((n, c), 0.0, 1.0, dtype), rand((n, c), 0.0, 1.0, dtype)
    return a, dy, dh


def _norm(v, kind, eps=1e-6):
    """N(v), rstd, and what N may be off by."""
    m = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    r = ((v - m).square().mean(1, keepdim=True) + eps).rsqrt()
    unit = (v - m) * r
    return unit, r, 96 * U * (v.abs().mean(1, keepdim=True) * r + unit.abs())


class _Reference:
    """The formulas in 64 bits at the given h, with bounds."""

    def __init__(self, a, h, norm="layer", residual_scale=1.0, dropout=0.0, seed=0, subsequence=0):
        self.a, self.kind = a, norm
        dtype = a["x"].dtype
        n, c = a["x"].shape
        b = a["coords"][:, 0].long()
        inside = ((b >= 0) & (b < a.get("batch_size", 1 << 30)))[:, None]
        every = not any(a[k].ndim == 2 for k in ("gate", "scale", "shift") if k in a)
        if every:
            inside = torch.ones_like(inside)

        def row(name, missing):
            if name not in a:
                return torch.full((1, c), missing, device=DEV, dtype=F64)
            t = a[name].detach().to(F64)
            if t.ndim == 2 and t.shape[0] > 1:
                t = t[b.clamp(0, len(t) - 1)]
            if name in ("gate", "scale", "shift"):
                t = torch.where(inside, t, missing)
            return t.expand(n, c) if t.ndim == 2 and t.shape[0] > 1 else t.reshape(-1, c)

        f = 1.0
        if dropout:
            f = torch.from_numpy(factors(n * c, dropout, seed, subsequence)).to(DEV).view(n, c)
        x, d = a["x"].detach().to(F64), a["branch"].detach().to(F64) * f
        w, beta, wb = row("weight", 1.0), row("bias", 0.0), row("branch_weight", 1.0)
        gate, sc, sh = row("gate", 1.0), row("scale", 0.0), row("shift", 0.0)
        ud, rd, ed = _norm(d, norm) if a["branch_norm"] else (d, None, 4 * U * d.abs())
        gg = residual_scale * gate * wb
        self.h = x + gg * ud
        self.h_bound = 1.01 * _half(dtype) * self.h.abs() + (gg.abs() * ed) * 1.1 \
            + 8 * U * (x.abs() + (gg * ud).abs())
        h = h.to(F64)
        u, r, e = _norm(h, norm)
        self.y = (u * w + beta) * (1 + sc) + sh
        mul = w * (1 + sc)
        self.y_bound = 1.01 * _half(dtype) * self.y.abs() + 1.1 * e * mul.abs() \
            + 8 * U * ((u * mul).abs() + (beta * (1 + sc)).abs() + sh.abs())
        self.parts = dict(b=b, inside=inside, f=f, w=w, beta=beta, wb=wb, gate=gate, sc=sc, ud=ud,
                          rd=rd, gg=gg, u=u, r=r, mul=mul, alpha=residual_scale)

    def gradients(self, dy, dh):
        """{name: (gradient, bound)}"""
        p, a = self.parts, self.a
        dtype = a["x"].dtype
        half = 1.01 * _half(dtype)
        dy = torch.zeros_like(p["u"]) if dy is None else dy.to(F64)
        dh = torch.zeros_like(p["u"]) if dh is None else dh.to(F64)

        def back(g, size, u, r):
            m2 = (g * u).mean(1, keepdim=True)
            out = g - u * m2
            if self.kind == "layer":
                out = out - g.mean(1, keepdim=True)
            wide = (size * (1 + u.abs())).mean(1, keepdim=True)
            return r * out, r * (size + (1 + u.abs()) * wide)

        g = dy * p["mul"]
        D, size = back(g, g.abs(), p["u"], p["r"])
        D, size = D + dh, size + dh.abs()
        out = {"x": (D, half * D.abs() + 400 * U * size)}
        dd, dsize = D * p["gg"], size * p["gg"].abs()
        if a["branch_norm"]:
            dd, dsize = back(dd, dsize, p["ud"], p["rd"])
        dd, dsize = dd * p["f"], dsize * p["f"]
        out["branch"] = (dd, half * dd.abs() + 1000 * U * dsize)

        n = len(D)
        step = (n + 64) * U
        unit_size = 1 + p["u"].abs()
        d_size = (1 + p["ud"].abs()) if a["branch_norm"] else p["ud"].abs()

        def put(name, term, size):
            """Sums of `term` over the rows that share a row of `name`."""
            if name not in a:
                return
            t = a[name]
            size = size * (step + 500 * U)
            if name in ("gate", "scale", "shift"):
                term, size = (torch.where(p["inside"], v, 0.0) for v in (term, size))
            if t.ndim == 2 and t.shape[0] > 1:
                at = p["b"].clamp(0, t.shape[0] - 1)
                s, z = (torch.zeros(t.shape, dtype=F64, device=DEV).index_add_(0, at, v)
                        for v in (term, size))
            else:
                s, z = (v.sum(0).reshape(t.shape) for v in (term, size))
            out[name] = (s, 1.01 * _half(t.dtype) * s.abs() + z)

        one = (1 + p["sc"])
        put("weight", dy * one * p["u"], (dy * one).abs() * unit_size)
        put("bias", dy * one, (dy * one).abs())
        put("shift", dy, dy.abs())
        put("scale", dy * (p["u"] * p["w"] + p["beta"]),
            dy.abs() * (unit_size * p["w"].abs() + p["beta"].abs()))
        put("gate", D * p["ud"] * p["wb"] * p["alpha"], size * d_size * (p["wb"] * p["alpha"]).abs())
        put("branch_weight", D * p["ud"] * p["gate"] * p["alpha"],
            size * d_size * (p["gate"] * p["alpha"]).abs())
        return out


def _close(got, want, bound, what):
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps  # a subnormal step
    err = (got.detach().to(F64) - want).abs()
    assert not torch.isnan(err).any(), what
    assert (err <= bound + tiny).all(), (what, (err / (bound + tiny)).max().item())


def _step(a, dy, dh, **options):
    leaves = {k: v.detach().requires_grad_(True) for k, v in a.items()
              if isinstance(v, torch.Tensor) and k != "coords"}
    y, h = block_norm(**{**a, **leaves}, **options)
    outs = [(t, g) for t, g in ((y, dy), (h, dh)) if g is not None]
    grads = torch.autograd.grad([t for t, _ in outs], list(leaves.values()), [g for _, g in outs],
                                allow_unused=True)
    return y, h, dict(zip(leaves, grads))


def _compare(a, dy, dh, **options):
    y, h, grads = _step(a, dy, dh, **options)
    ref = _Reference(a, h, **options)
    _close(h, ref.h, ref.h_bound, "h")
    _close(y, ref.y, ref.y_bound, "y")
    want = ref.gradients(dy, dh)
    assert set(want) == set(grads)
    for name, (g, bound) in want.items():
        assert grads[name].shape == a[name].shape and grads[name].dtype == a[name].dtype
        _close(grads[name], g, bound, name)
    with torch.no_grad():
        y2, h2 = block_norm(**a, **options)
    assert torch.equal(y, y2) and torch.equal(h, h2)
    N.check_device_status(DEV)


WIDTHS = [1, 2, 8, 63, 64, 72, 128, 129, 256, 257, 264, 512, 520, 1000, 1024, 1031, 2048, 2056, 2057,
          4096, 8192]


@pytest.mark.parametrize("c", WIDTHS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_widths(c, dtype):
    for n in (1, 37):
        a, dy, dh = _case(n, c, dtype, c + n, batch=min(3, n))
        _compare(a, dy, dh)
    a, dy, dh = _case(23, c, dtype, c, batch=2)
    _compare(a, dy, dh, norm="rms", residual_scale=0.5, dropout=0.25, seed=SEED, subsequence=9)


@pytest.mark.parametrize("names", [(), ("weight",), ("bias",), ("gate",), ("scale",), ("shift",),
                                   ("branch_weight",), ("gate", "scale", "shift"),
                                   ("weight", "bias", "gate"), ("branch_weight", "gate")])
def test_options(names):
    for i, norm in enumerate(("layer", "rms")):
        for per_batch in (True, False):
            a, dy, dh = _case(301, 136, torch.float32, 10 + i, 4, per_batch, names)
            _compare(a, dy, dh, norm=norm)
            a["branch_norm"] = True
            _compare(a, dy, None, norm=norm, residual_scale=-0.25)
            _compare(a, None, dh, norm=norm, dropout=0.5, seed=SEED)


@pytest.mark.parametrize("kind", DTYPES)
def test_types_of_coefficients(kind):
    for dtype in DTYPES:
        a, dy, dh = _case(65, 264, dtype, 3, kind=kind)
        _compare(a, dy, dh)


def test_many_rows():
    a, dy, dh = _case(20011, 256, torch.bfloat16, 4, batch=5)
    _compare(a, dy, dh, dropout=0.1, seed=SEED)


# Rows of 33 to 128 eights, and 64 rows an SM: a pipeline of bulk copies per warp.
@pytest.mark.parametrize("c", [264, 512, 520, 1000, 1024])
@pytest.mark.parametrize("dtype", DTYPES)
def test_pipelined_rows(c, dtype):
    n = 64 * torch.cuda.get_device_properties(DEV).multi_processor_count + 37
    for i, norm in enumerate(("layer", "rms")):
        a, dy, dh = _case(n, c, dtype, c + i, batch=3)
        _compare(a, dy, dh, norm=norm, residual_scale=0.5)
        del a["branch_weight"]
        a["branch_norm"] = False
        _compare(a, dy, dh, norm=norm, dropout=0.25, seed=SEED, subsequence=9)


def test_pipelined_rows_of_many_batch_elements():
    """Blocks whose rows have more batch elements than tables; rows in any order; some without one; one of
    the results without a gradient; nothing per batch element."""
    n = 64 * torch.cuda.get_device_properties(DEV).multi_processor_count + 5
    a, dy, dh = _case(n, 264, torch.bfloat16, 15, batch=700)
    _compare(a, dy, None)
    _compare(a, None, dh)
    g = torch.Generator(device=DEV).manual_seed(16)
    a["coords"][:, 0] = torch.randint(0, 700, (n,), device=DEV, generator=g)
    _compare(a, dy, dh, norm="rms")
    a["coords"][::7, 0] = 700
    a["coords"][3::7, 0] = -1
    with pytest.raises(RuntimeError, match="out of range"):
        _compare(a, dy, dh)
    for names in ((), ("weight",), ("gate",)):
        a, dy, dh = _case(n, 264, torch.bfloat16, 17, per_batch=False, names=names)
        _compare(a, dy, dh)
    # rows apart, and the same results every time
    a, dy, dh = _case(n, 264, torch.bfloat16, 18, batch=2)
    wide = torch.zeros((n, 600), dtype=torch.bfloat16, device=DEV)
    wide[:, 8:272], wide[:, 280:544] = a["x"], a["branch"]
    b = {**a, "x": wide[:, 8:272], "branch": wide[:, 280:544]}
    first, again = _step(a, dy, dh), _step(b, dy, dh)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    assert all(torch.equal(first[2][k], again[2][k]) for k in first[2])


def test_coordinates_made_under_inference_mode():
    a, dy, dh = _case(100, 64, torch.float32, 19)
    want = _step(a, dy, dh)
    with torch.inference_mode():
        held = a["coords"].clone()
        assert held.is_inference()
        y, h = block_norm(**{**a, "x": a["x"].clone()})
    assert torch.equal(y, want[0]) and torch.equal(h, want[1])
    got = _step({**a, "coords": held}, dy, dh)
    assert all(torch.equal(got[2][k], want[2][k]) for k in want[2])


def test_unsorted_and_bad_batch_elements():
    """Rows of batch elements in any order, some without one: not modulated, reported, and their
    gradients reach x, branch and the weights only."""
    for n in (301, 20001):
        a, dy, dh = _case(n, 72, torch.float32, 5, batch=7)
        g = torch.Generator(device=DEV).manual_seed(6)
        a["coords"][:, 0] = torch.randint(0, 7, (n,), device=DEV, generator=g)
        _compare(a, dy, dh)
        a["coords"][::5, 0] = torch.tensor([-1, 7, 2**31 - 1, -2**31], dtype=torch.int32,
                                           device=DEV).repeat(n)[: len(a["coords"][::5])]
        with pytest.raises(RuntimeError, match="out of range"):
            _compare(a, dy, dh)
        a["coords"][:, 0] = 9  # none has one
        with pytest.raises(RuntimeError, match="out of range"):
            _compare(a, dy, dh)


def test_empty_batch_elements_and_many_of_them():
    a, dy, dh = _case(64, 40, torch.float32, 7, batch=500)
    _compare(a, dy, dh)
    a["coords"][:, 0] = 499
    _compare(a, dy, dh)


def test_sums_do_not_depend_on_the_run():
    a, dy, dh = _case(9001, 256, torch.bfloat16, 8, batch=4)
    first = _step(a, dy, dh)
    for _ in range(3):
        again = _step(a, dy, dh)
        assert all(torch.equal(first[2][k], again[2][k]) for k in first[2])


def test_strides_shapes_and_no_rows():
    a, dy, dh = _case(60, 64, torch.bfloat16, 9, batch=2)
    want = block_norm(**a)
    wide = torch.zeros((60, 200), dtype=torch.bfloat16, device=DEV)
    six = torch.zeros((2, 6 * 64), dtype=torch.bfloat16, device=DEV)
    for shift in (0, 1, 8):
        b = dict(a)
        for name, at in (("x", shift), ("branch", shift + 72)):
            wide[:, at:at + 64] = a[name]
            b[name] = wide[:, at:at + 64]
        for i, name in enumerate(("gate", "scale", "shift")):
            six[:, 128 * i:128 * i + 64] = a[name]
            b[name] = six[:, 128 * i:128 * i + 64]
        got = block_norm(**b)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    b = {**a, "x": a["x"].view(3, 20, 64), "branch": a["branch"].view(3, 20, 64)}
    got = block_norm(**b)
    assert got[0].shape == (3, 20, 64) and torch.equal(got[1].view(60, 64), want[1])
    b = {**a, "x": a["x"].t().contiguous().t(), "branch": a["branch"].t().contiguous().t()}
    assert all(torch.equal(p, q) for p, q in zip(block_norm(**b), want))
    empty = {**a, "x": a["x"][:0], "branch": a["branch"][:0], "coords": a["coords"][:0]}
    y, h, grads = _step(empty, dy[:0], dh[:0])
    assert y.shape == h.shape == (0, 64)
    assert all((grads[k] == 0).all() for k in COEFS)
    none = torch.zeros((4, 0), device=DEV)
    assert block_norm(none, none)[0].shape == (4, 0)


def test_rows_of_zeros_and_not_finite():
    x = torch.zeros((4, 64), device=DEV)
    x[1, 3], x[2, 5] = float("nan"), float("inf")
    y, h = block_norm(x, torch.zeros_like(x))
    assert (y[0] == 0).all() and (y[3] == 0).all()
    assert y[1].isnan().all() and y[2].isnan().any()
    for norm in ("layer", "rms"):  # a branch of zeros under its own norm has finite gradients
        b = torch.zeros((4, 64), device=DEV, requires_grad=True)
        y, h = block_norm(torch.ones_like(b), b, norm=norm, branch_norm=True)
        (g,) = torch.autograd.grad((y, h), (b,), (torch.ones_like(y), torch.ones_like(h)))
        assert torch.isfinite(g).all()


def test_dropout_drops_what_dropout_drops():
    from mlx_diffuser_b200 import dropout

    for c in (72, 63):
        b = torch.ones((50, c), device=DEV)
        _, h = block_norm(torch.zeros_like(b), b, dropout=0.5, seed=SEED, subsequence=3)
        assert torch.equal(h, dropout(b, 0.5, SEED, subsequence=3))


def test_gradients_against_differences():
    a, dy, dh = _case(6, 40, torch.float32, 11, batch=2)
    _, _, grads = _step(a, dy, dh, dropout=0.25, seed=SEED)
    g = torch.Generator(device=DEV).manual_seed(12)
    for name, grad in grads.items():
        way = torch.randn(a[name].shape, device=DEV, generator=g)
        step = 2.0**-7
        sides = []
        for sign in (1, -1):
            y, h = block_norm(**{**a, name: a[name] + sign * step * way}, dropout=0.25, seed=SEED)
            sides.append(float((y.to(F64) * dy).sum() + (h.to(F64) * dh).sum()))
        slope = float((grad.to(F64) * way).sum())
        # outputs' roundings over the step, and the third derivative's share of the central difference
        scale = float((dy.to(F64).abs().sum() + dh.to(F64).abs().sum()))
        bound = 256 * U * scale / step + step**2 * scale * 20
        assert abs((sides[0] - sides[1]) / (2 * step) - slope) <= bound, name


def test_captured_step_beside_an_eager_one():
    a, dy, dh = _case(500, 256, torch.bfloat16, 13, batch=3)
    want = _step(a, dy, dh)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _step(a, dy, dh)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = _step(a, dy, dh)
    torch.cuda.synchronize()
    for _ in range(2):
        graph.replay()
        again = _step(a, dy, dh)
        torch.cuda.synchronize()
        for out in (got, again):
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
            assert all(torch.equal(out[2][k], want[2][k]) for k in want[2])


def test_rows_past_32_bits():
    """Offsets beyond 2^31 elements, forward and backward: the last rows are what they are by themselves."""
    n, c = 2**21 + 5, 1032
    for width in (c, 1024):  # the direct and the pipelined kernel
        a, dy, dh = _case(64, width, torch.bfloat16, 20, batch=2)
        last = n - 64
        big = {k: torch.zeros((n, width), dtype=torch.bfloat16, device=DEV) for k in ("x", "branch")}
        for k, t in big.items():
            t[last:] = a[k]
        coords = torch.zeros((n, 4), dtype=torch.int32, device=DEV)
        coords[last:] = a["coords"]
        g = torch.zeros((n, width), dtype=torch.bfloat16, device=DEV)
        g[last:] = dy
        b = {**a, **{k: t.requires_grad_(True) for k, t in big.items()}, "coords": coords}
        y, h = block_norm(**b)
        dx, db = torch.autograd.grad((y, h), (big["x"], big["branch"]), (g, g))
        ref = _Reference(a, h[last:].detach())
        _close(h[last:], ref.h, ref.h_bound, "h")
        _close(y[last:], ref.y, ref.y_bound, "y")
        want = ref.gradients(dy, dy)
        _close(dx[last:], *want["x"], "dx")
        _close(db[last:], *want["branch"], "dbranch")
        del b, big, y, h, dx, db, g


def _hooked(how, run, *leaves):
    if how == "checkpoint":
        from torch.utils.checkpoint import checkpoint

        return checkpoint(run, *leaves, use_reentrant=False)
    with torch.autograd.graph.save_on_cpu(pin_memory=how == "pinned"):
        return run(*leaves)


@pytest.mark.parametrize("how", ["checkpoint", "host", "pinned"])
def test_saved_tensors_that_come_back_as_others(how):
    """Coefficients formed inside the region and rows apart: the backward pass gets tensors at other addresses
    with other strides, and the first ones' memory is gone."""
    n, c = 300, 72
    g = torch.Generator(device=DEV).manual_seed(23)
    leaves = [torch.randn(s, device=DEV, generator=g).requires_grad_(True)
              for s in ((n, 3 * c), (2, 16), (16, 3 * c), (c,))]
    coords = torch.zeros((n, 4), dtype=torch.int32, device=DEV)
    coords[n // 3:, 0] = 1

    def run(rows, cond, weight, norm):
        gate, scale, shift = (cond @ weight).chunk(3, 1)
        return block_norm(rows[:, :c], rows[:, 2 * c:], gate=gate, scale=scale, shift=shift,
                          weight=2 * norm, branch_norm=True, branch_weight=norm + 1, coords=coords,
                          dropout=0.25, seed=torch.tensor(7, device=DEV))

    outs = []
    for i in range(2):
        y, h = _hooked(how, run, *leaves) if i else run(*leaves)
        spill = [torch.full((n, 3 * c), float("nan"), device=DEV) for _ in range(8)]  # over what was freed
        outs.append((y, h, *torch.autograd.grad((y, h), leaves, (y.detach(), h.detach()))))
        del spill
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    N.check_device_status(DEV)


@pytest.mark.parametrize("batch", [7, 8, 31, 32, 33, 1000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_over_many_batch_elements(batch, dtype):
    """Rows of coefficients per batch element beside rows that all share, elements without rows, rows without
    an element, and no rows at all; the sums are the same every time."""
    for n, c in ((2000, 72), (333, 63), (40, 1024)):
        a, dy, dh = _case(n, c, dtype, batch + c, batch)
        a["coords"][n // 2:, 0] = batch - 1
        _compare(a, dy, dh, dropout=0.25, seed=SEED)
        for shared in ("gate", "scale", "shift"):
            _compare({**a, shared: a[shared][0].contiguous()}, dy, dh, norm="rms", residual_scale=0.5)
        first, again = _step(a, dy, dh), _step(a, dy, dh)
        assert all(torch.equal(first[2][k], again[2][k]) for k in first[2])
        a["coords"][::3, 0] = batch
        with pytest.raises(RuntimeError, match="out of range"):
            _compare(a, dy, dh)
        empty = {**a, "x": a["x"][:0], "branch": a["branch"][:0], "coords": a["coords"][:0]}
        _, _, grads = _step(empty, dy[:0], dh[:0])
        assert all((grads[k] == 0).all() for k in COEFS)
        a, dy, dh = _case(n, c, dtype, batch, batch, names=("gate", "scale", "shift"))
        _compare(a, dy, dh)  # nothing that is summed over the batch elements
