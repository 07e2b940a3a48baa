"""``rms_norm`` on the GPU against its formula in 64 bits: the residual's addition, the 8-bit output
and the gradients, over the row widths where the kernel changes its layout.

Bounds: a rounding to the type t is off by at most ``finfo(t).eps / 2`` of the value. fp32 sums of k
terms are off by at most k 2^-24 of the sum of the terms' magnitudes; a thread adds at most 64
elements of a row before the sums are joined pairwise, so 96 covers a row's sum of squares, the
square root, the quotient and the products."""

from __future__ import annotations

import pytest
import torch

from mlx_diffuser_b200 import _native as N
from mlx_diffuser_b200 import rms_norm

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0**-24
ROW = 96 * U
F64 = torch.float64


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _inputs(n, c, dtype, seed, residual=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn((n, c), device=DEV, generator=g).to(dtype)
    r = (2 * torch.randn((n, c), device=DEV, generator=g)).to(dtype) if residual else None
    w = 1 + 0.3 * torch.randn(c, device=DEV, generator=g)
    return x, r, w


def _reference(x, r, w, eps=1e-6):
    """h as the operator defines it (one rounding of the exact sum), y and u in 64 bits."""
    h = x.to(F64) if r is None else (x.to(F64) + r.to(F64)).to(x.dtype).to(F64)
    rstd = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    u = h * rstd
    return h, rstd, u, u * w.to(F64)


WIDTHS = [1, 2, 7, 8, 63, 64, 72, 256, 331, 512, 520, 1024, 1031, 2048, 4096, 8192]


@pytest.mark.parametrize("c", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_forward(c, dtype):
    for n in (1, 37):
        for residual in (False, True):
            x, r, w = _inputs(n, c, dtype, c + n, residual)
            out = rms_norm(x, w, residual=r)
            y, h = out if residual else (out, x)
            rh, _, _, ry = _reference(x, r, w)
            assert torch.equal(h.to(F64), rh)
            err = (y.to(F64) - ry).abs()
            assert (err <= (_half(dtype) + ROW) * ry.abs() + torch.finfo(dtype).tiny).all()


@pytest.mark.parametrize("n,c", [(5, 72), (5, 331), (9600, 512)])
def test_eight_bit_output_of_the_smallest_numbers(n, c):
    """Rows whose scale is a subnormal number, or would be zero. The scale is then off by half of the
    smallest number, 2^-150, and the value it stands for by at most 448 times that, next to half a
    step of e4m3 (2^-4 of the value, or 2^-10 scales below its normal range)."""
    x, _, _ = _inputs(n, c, torch.bfloat16, 9, False)
    for size in (1e-36, 1e-40, 3e-44):
        w = torch.full((c,), size, device=DEV)
        w[::3] = 0
        q, scale = rms_norm(x, w, quantize=True)
        _, _, _, y = _reference(x, None, w)
        got, s = q.float().to(F64), scale.to(F64)[:, None]
        assert torch.isfinite(got).all() and (scale > 0).all() and not got[:, ::3].any()
        # y is a multiple of 2^-149 too
        off = (2.0**-4 + ROW) * y.abs() + 2.0**-10 * s + 450 * 2.0**-149
        assert ((got * s - y).abs() <= off).all()


@pytest.mark.parametrize("c", [1, 7, 64, 72, 331, 1024, 2048, 8192])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_eight_bit_output(c, dtype):
    x, r, w = _inputs(41, c, dtype, c, True)
    x[3] = 0
    r[3] = 0  # a row of zeros
    (q, scale), h = rms_norm(x, w, residual=r, quantize=True)
    rh, _, _, ry = _reference(x, r, w)
    assert q.dtype == torch.float8_e4m3fn and scale.dtype == torch.float32
    assert torch.equal(h.to(F64), rh)
    top = ry.abs().amax(-1)
    want = torch.where(top == 0, torch.ones_like(top), top / 448)
    assert ((scale.to(F64) - want).abs() <= (ROW + U) * want).all()
    assert scale[3] == 1 and not q[3].float().any()
    back = q.to(F64) * scale.to(F64)[:, None]
    # half a step of e4m3: 2^-4 of the value, 2^-10 of the scale below the normal range
    bound = (2.0**-4 + 2 * ROW) * ry.abs() + (2.0**-10 + ROW) * want[:, None]
    assert ((back - ry).abs() <= bound).all()
    assert (q.float().abs().amax(-1)[top > 0] == 448).all()
    alone, s2 = rms_norm(h, w, quantize=True)
    assert torch.equal(alone.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, scale)


@pytest.mark.parametrize("c", [1, 7, 8, 64, 72, 331, 512, 1024, 1031, 4096, 8192])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_gradients(c, dtype):
    for n, residual in ((1, True), (173, False), (173, True)):
        x, r, w = _inputs(n, c, dtype, 3 * c + n, residual)
        g = torch.Generator(device=DEV).manual_seed(c)
        dy, dh = (torch.randn((n, c), device=DEV, generator=g).to(dtype) for _ in range(2))
        leaves = [t.requires_grad_(True) for t in (x, r, w) if t is not None]
        out = rms_norm(x, w, residual=r)
        if residual:
            dx, dr, dw = torch.autograd.grad(out, leaves, (dy, dh))
            assert torch.equal(dx, dr)
        else:
            dx, dw = torch.autograd.grad(out, leaves, dy)
        with torch.no_grad():
            _, rstd, u, _ = _reference(x, r, w)
            gw = dy.to(F64) * w.to(F64)
            gu = gw * u
            want = rstd * (gw - u * gu.mean(-1, keepdim=True))
            mag = rstd * (gw.abs() + u.abs() * gu.abs().mean(-1, keepdim=True))
            if residual:
                want = want + dh.to(F64)
                mag = mag + dh.to(F64).abs()
            err = (dx.to(F64) - want).abs()
            assert (err <= _half(dtype) * want.abs() + 4 * ROW * mag + torch.finfo(dtype).tiny).all()
            terms = dy.to(F64) * u
            err = (dw.to(F64) - terms.sum(0)).abs()
            assert dw.dtype == torch.float32
            assert (err <= (n * U + ROW) * terms.abs().sum(0) + 1e-30).all()


@pytest.mark.parametrize("c", [264, 512, 516, 768, 1000, 1024])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_many_rows(c, dtype):
    """Enough rows for the warps' pipelines, the last round not full, rows with a stride."""
    n = 4 * 16 * torch.cuda.get_device_properties(DEV).multi_processor_count + 77
    x, r, w = _inputs(n, c, dtype, c, True)
    wide = torch.zeros((n, c + 8), dtype=dtype, device=DEV)
    wide[:, :c] = x
    x = wide[:, :c]
    rh, rstd, u, ry = _reference(x, r, w)
    y, h = rms_norm(x, w, residual=r)
    assert torch.equal(h.to(F64), rh)
    assert ((y.to(F64) - ry).abs() <= (_half(dtype) + ROW) * ry.abs()
            + torch.finfo(dtype).tiny).all()
    (q, s), h2 = rms_norm(x, w, residual=r, quantize=True)
    top = ry.abs().amax(-1)
    assert torch.equal(h2, h) and ((s.to(F64) - top / 448).abs() <= (ROW + U) * top / 448).all()
    back = q.to(F64) * s.to(F64)[:, None]
    assert ((back - ry).abs() <= (2.0**-4 + 2 * ROW) * ry.abs()
            + (2.0**-10 + ROW) * (top / 448)[:, None]).all()
    alone = rms_norm(x, w)
    ra = _reference(x, None, w)[3]
    assert ((alone.to(F64) - ra).abs() <= (_half(dtype) + ROW) * ra.abs()
            + torch.finfo(dtype).tiny).all()
    g = torch.Generator(device=DEV).manual_seed(c)
    dy, dh = (torch.randn((n, c), device=DEV, generator=g).to(dtype) for _ in range(2))
    for residual in (True, False):
        leaves = [t.requires_grad_(True) for t in ((x.detach(), r, w) if residual
                                                   else (x.detach(), w))]
        out = rms_norm(leaves[0], w, residual=r if residual else None)
        grads = torch.autograd.grad(out, leaves, (dy, dh) if residual else dy)
        with torch.no_grad():
            _, rstd, u, _ = _reference(x, r if residual else None, w)
            gw = dy.to(F64) * w.to(F64)
            gu = gw * u
            want = rstd * (gw - u * gu.mean(-1, keepdim=True))
            mag = rstd * (gw.abs() + u.abs() * gu.abs().mean(-1, keepdim=True))
            if residual:
                want, mag = want + dh.to(F64), mag + dh.to(F64).abs()
            err = (grads[0].to(F64) - want).abs()
            assert (err <= _half(dtype) * want.abs() + 4 * ROW * mag
                    + torch.finfo(dtype).tiny).all()
            terms = dy.to(F64) * u
            err = (grads[-1].to(F64) - terms.sum(0)).abs()
            assert (err <= (n * U + ROW) * terms.abs().sum(0)).all()
    N.check_device_status(DEV)


def test_gradient_against_differences():
    x, r, w = _inputs(5, 24, torch.float32, 9)
    x, r, w = (t.requires_grad_(True) for t in (x, r, w))
    g = torch.Generator(device=DEV).manual_seed(1)
    dy, dh = (torch.randn((5, 24), device=DEV, generator=g, dtype=torch.float32) for _ in range(2))
    grads = torch.autograd.grad(rms_norm(x, w, residual=r), (x, r, w), (dy, dh))

    def loss(a, b, c):  # the formula in 64 bits, without the rounding of h
        h = a + b
        y = h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * c
        return (y * dy.to(F64)).sum() + (h * dh.to(F64)).sum()

    args = [t.detach().to(F64) for t in (x, r, w)]
    for i, grad in enumerate(grads):
        step = torch.randn(args[i].shape, device=DEV, generator=g).to(F64)
        up, down = ([a + (s * 1e-5 * step if i == j else 0) for j, a in enumerate(args)]
                    for s in (1, -1))
        want = (loss(*up) - loss(*down)) / 2e-5
        # differences: 1e-10 of third derivatives (order 10 here); fp32 sums of 120 terms
        assert abs((grad.to(F64) * step).sum() - want) <= 1e-5 * (grad.to(F64) * step).abs().sum()


def test_strided_rows_other_shapes_and_weight_types():
    g = torch.Generator(device=DEV).manual_seed(2)
    wide = torch.randn((30, 200), device=DEV, generator=g).to(torch.bfloat16)
    w = torch.rand(64, device=DEV, generator=g).to(torch.bfloat16)
    for view in (wide[:, 64:128], wide[:, 3:67], wide[::2, :64], wide.t()[:64].t(),
                 wide[:1].expand(30, 200)[:, :64]):
        assert torch.equal(rms_norm(view, w), rms_norm(view.contiguous(), w.float()))
    cube = torch.randn((3, 5, 64), device=DEV, generator=g)
    y, h = rms_norm(cube, residual=cube)
    assert y.shape == cube.shape and torch.equal(h, cube + cube)
    (q, s), _ = rms_norm(cube, residual=cube, quantize=True)
    assert q.shape == cube.shape and s.shape == (3, 5)
    row = rms_norm(cube[0, 0])
    assert row.shape == (64,) and torch.equal(row, rms_norm(cube)[0, 0])
    wb = w.clone().requires_grad_(True)
    (dw,) = torch.autograd.grad(rms_norm(wide[:, 64:128], wb).float().sum(), wb)
    assert dw.dtype == torch.bfloat16
    # only one of the two results is used further
    x = cube.clone().requires_grad_(True)
    r = cube.clone().requires_grad_(True)
    y, h = rms_norm(x, residual=r)
    a = torch.autograd.grad(h.sum(), (x, r), retain_graph=True)
    assert torch.equal(a[0], torch.ones_like(x)) and torch.equal(a[1], a[0])
    b = torch.autograd.grad(y.sum(), x)[0]
    assert torch.isfinite(b).all()


def test_empty_and_not_finite_rows():
    for shape in ((0, 64), (5, 0), (0, 0)):
        x = torch.zeros(shape, device=DEV)
        assert rms_norm(x).shape == shape
        y, h = rms_norm(x, residual=x)
        assert y.shape == shape and h.shape == shape
        q, s = rms_norm(x, quantize=True)
        assert q.shape == shape and s.shape == shape[:1]
    x = torch.zeros((0, 64), device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    dx, dw = torch.autograd.grad(rms_norm(x, w).sum(), (x, w))
    assert dx.shape == (0, 64) and not dw.any()
    x = torch.randn((4, 1024), device=DEV)
    x[1, 7] = float("nan")
    x[2, 1000] = float("inf")
    y = rms_norm(x)
    q, s = rms_norm(x, quantize=True)
    assert torch.isfinite(y[0]).all() and torch.isfinite(y[3]).all()
    assert torch.isnan(y[1]).all() and torch.isnan(y[2, 1000]) and not y[2, :1000].any()
    assert torch.equal(torch.isnan(s).cpu(), torch.tensor([False, True, True, False]))
    assert torch.isnan(q[1].float()).all() and torch.isnan(q[2].float()).all()


def test_other_stream_and_graph():
    x, r, w = _inputs(300, 1024, torch.bfloat16, 4)
    want = rms_norm(x, w, residual=r)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        got = rms_norm(x, w, residual=r)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rms_norm(x, w, residual=r, quantize=True)
    x.copy_(x.flip(0))
    graph.replay()
    (q, s), h = out
    (q2, s2), h2 = rms_norm(x, w, residual=r, quantize=True)
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8))
    assert torch.equal(s, s2) and torch.equal(h, h2)
    N.check_device_status(DEV)
