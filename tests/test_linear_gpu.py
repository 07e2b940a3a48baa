"""``linear`` on the GPU against its formula in 64 bits: every path (few rows, fp32 tiles, tensor
cores, split k, padded copies), activation, type and gradient.

Bounds: with ``mag = |x| |w|^T``, an fp32 sum of k products is off by at most (2 k + 16) 2^-24 mag:
tensor cores may drop the last place of each addition instead of rounding it (2^-23 a step).
The activations' slopes are below 1.13 and they and the few operations around them are off by
at most 16 2^-24 of the values involved. A rounding to t is off by ``finfo(t).eps / 2``."""

from __future__ import annotations

import math

import pytest
import torch

from mlx_diffuser_b200 import _native as N
from mlx_diffuser_b200 import linear, rms_norm

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0**-24
F64 = torch.float64
ACTS = [None, "silu", "gelu", "gelu_tanh"]


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _act(z, name):
    """The activation, its slope and a bound of the slope's own slope."""
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


CURVE = 1.2  # the activations' second derivatives are below it


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def _check_forward(got, x, w, b, r, act, xs=None, ws=None):
    dtype = got.dtype
    k = x.shape[1]
    x64, w64 = x.to(F64), w.to(F64)
    if xs is not None:
        x64 = x64 * xs.to(F64)[:, None]
    if ws is not None:
        w64 = w64 * ws.to(F64)[:, None]
    z, mag = x64 @ w64.T, x64.abs() @ w64.abs().T
    if b is not None:
        z, mag = z + b.to(F64), mag + b.to(F64).abs()
    y, _ = _act(z, act)
    if r is not None:
        y, mag = y + r.to(F64), mag + r.to(F64).abs()
    bound = _half(dtype) * y.abs() + 1.13 * (2 * k + 32) * U * mag + torch.finfo(dtype).tiny
    err = (got.to(F64) - y).abs()
    assert (err <= bound).all(), float((err / bound).max())
    # and as a whole: the rounding alone is eps / (2 sqrt 3) at most in the mean
    if y.numel() >= 64:
        rel = float(err.norm() / y.norm())
        assert rel <= _half(dtype) + (4e-6 if dtype == torch.float32 else 0), rel


SHAPES = [
    (1, 8, 5), (2, 256, 2048), (8, 331, 517), (3, 1, 1), (5, 4096, 64),  # few rows
    (9, 64, 64), (128, 64, 256), (129, 72, 264), (257, 331, 517), (300, 128, 40),
    (1000, 8, 1024), (640, 1031, 33), (2000, 512, 768),
    (40, 4096, 64), (130, 2049, 130),  # few tiles: k is split
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_forward(shape, dtype):
    m, k, n = shape
    x, w = _rand((m, k), dtype, 1), _rand((n, k), dtype, 2, k**-0.5)
    b, r = _rand((n,), dtype, 3), _rand((m, n), dtype, 4)
    for i, act in enumerate(ACTS):
        bias, res = (b if i != 1 else None), (r if i % 2 else None)
        got = linear(x, w, bias, activation=act, residual=res)
        assert got.dtype == dtype and got.shape == (m, n)
        _check_forward(got, x, w, bias, res, act)
    N.check_device_status(DEV)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("out", [torch.float16, torch.bfloat16])
def test_eight_bit_operands(shape, out):
    m, k, n = shape
    # 2^-6 steps: every product and most sums are exact, so nothing hides behind rounding
    x = _rand((m, k), torch.float32, 5).to(torch.float8_e4m3fn)
    w = _rand((n, k), torch.float32, 6).to(torch.float8_e4m3fn)
    xs = torch.rand(m, device=DEV) + 0.5
    ws = (torch.rand(n, device=DEV) + 0.5) * k**-0.5
    b, r = _rand((n,), out, 7), _rand((m, n), out, 8)
    for act, scales, res in ((None, (xs, ws), None), ("gelu_tanh", (xs, ws), r),
                             ("silu", (None, ws), r), ("gelu", (xs, None), None)):
        got = linear(x, w, b, activation=act, residual=res, x_scale=scales[0],
                     weight_scale=scales[1])
        assert got.dtype == out
        _check_forward(got, x, w, b, res, act, *scales)
    assert linear(x, w).dtype == torch.bfloat16
    N.check_device_status(DEV)


@pytest.mark.parametrize("shape", [(1, 8, 5), (7, 331, 64), (9, 64, 64), (129, 72, 264),
                                   (257, 331, 517), (2000, 256, 128), (64, 40, 1031)], ids=str)
@pytest.mark.parametrize("act", ACTS, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_gradients(shape, act, dtype):
    m, k, n = shape
    x, w = _rand((m, k), dtype, 11), _rand((n, k), dtype, 12, k**-0.5)
    b, r, dy = _rand((n,), dtype, 13), _rand((m, n), dtype, 14), _rand((m, n), dtype, 15)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    y = linear(x, w, b, activation=act, residual=r)
    dx, dw, db, dr = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        _check_forward(y, x, w, b, r, act)
        assert torch.equal(dr, dy)
        x64, w64, g = x.to(F64), w.to(F64), dy.to(F64)
        z = x64 @ w64.T + b.to(F64)
        zmag = x64.abs() @ w64.abs().T + b.to(F64).abs()
        dz = g * _act(z, act)[1]
        # dz is rounded to t, and so is the z it is computed from
        h = _half(dtype)
        dz_off = h * dz.abs()
        if act is not None:
            dz_off = (1 + h) * dz_off + g.abs() * (CURVE * (h * z.abs() + (2 * k + 16) * U * zmag)
                                                   + 32 * U * (1 + z.abs()))
        for got, want, off, mag, terms in (
            (dx, dz @ w64, dz_off @ w64.abs(), dz.abs() @ w64.abs(), n),
            (dw, dz.T @ x64, dz_off.T @ x64.abs(), dz.abs().T @ x64.abs(), m),
            (db, dz.sum(0), dz_off.sum(0), dz.abs().sum(0), m),
        ):
            assert got.dtype == dtype and got.shape == want.shape
            bound = (h * want.abs() + (1 + h) * off + (2 * terms + 16) * U * (mag + off)
                     + torch.finfo(dtype).tiny)
            err = (got.to(F64) - want).abs()
            assert (err <= bound).all(), float((err / bound).max())
    N.check_device_status(DEV)


@pytest.mark.parametrize("act", ACTS, ids=str)
def test_gradient_against_differences(act):
    x, w = _rand((9, 20), torch.float32, 21), _rand((12, 20), torch.float32, 22, 0.3)
    b, dy = _rand((12,), torch.float32, 23), _rand((9, 12), torch.float32, 24)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(linear(x, w, b, activation=act), leaves, dy)
    args = [t.detach().to(F64) for t in leaves]

    def loss(a, c, d):
        return (_act(a @ c.T + d, act)[0] * dy.to(F64)).sum()

    for i, grad in enumerate(grads):
        step = _rand(args[i].shape, torch.float32, 30 + i).to(F64)
        up, down = ([a + (s * 1e-5 * step if i == j else 0) for j, a in enumerate(args)]
                    for s in (1, -1))
        want = (loss(*up) - loss(*down)) / 2e-5
        assert abs((grad.to(F64) * step).sum() - want) <= 2e-5 * (grad.to(F64) * step).abs().sum()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views_shapes_and_partial_gradients(dtype):
    wide = _rand((200, 300), dtype, 31)
    w = _rand((96, 64), dtype, 32, 0.125)
    for view in (wide[:, 64:128], wide[:, 3:67], wide[::3, 8:72], wide.t()[:64].t(),
                 wide[:1].expand(200, 300)[:, :64]):
        a, b = linear(view, w), linear(view.contiguous(), w)
        assert torch.equal(a, b)
    big = _rand((96, 200), dtype, 33, 0.125)
    assert torch.equal(linear(wide[:, :64], big[:, 5:69]),
                       linear(wide[:, :64], big[:, 5:69].contiguous()))
    res = _rand((200, 400), dtype, 34)
    assert torch.equal(linear(wide[:, :64], w, residual=res[:, 1:97]),
                       linear(wide[:, :64], w, residual=res[:, 1:97].contiguous()))
    cube = _rand((4, 50, 64), dtype, 35)
    got = linear(cube, w, residual=res[:, :96].reshape(4, 50, 96))
    assert got.shape == (4, 50, 96)
    assert torch.equal(got.reshape(200, 96), linear(cube.reshape(200, 64), w,
                                                    residual=res[:, :96]))
    assert linear(cube[0, 0], w).shape == (96,)
    # gradients of some inputs only, through a view and a broadcast bias
    bias = _rand((1,), dtype, 36).requires_grad_(True)
    wg = w.clone().requires_grad_(True)
    y = linear(cube, wg, bias.expand(96), activation="silu")
    db, = torch.autograd.grad(y, bias, torch.ones_like(y), retain_graph=True)
    dw, = torch.autograd.grad(y, wg, torch.ones_like(y))
    assert db.shape == (1,) and dw.shape == w.shape
    xg = wide.clone().requires_grad_(True)
    dx, = torch.autograd.grad(linear(xg[:, 5:69], w).sum(), xg)
    assert not dx[:, :5].any() and dx[:, 5:69].any()
    N.check_device_status(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_empty_sides(dtype):
    for m, k, n in ((0, 8, 16), (4, 8, 0), (40, 0, 16), (3, 0, 16), (0, 0, 0)):
        x, w = _rand((m, k), dtype, 41), _rand((n, k), dtype, 42)
        b, r = _rand((n,), dtype, 43), _rand((m, n), dtype, 44)
        leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
        y = linear(x, w, b, activation="silu", residual=r)
        dx, dw, db, _ = torch.autograd.grad(y, leaves, torch.ones_like(y))
        with torch.no_grad():
            if y.numel():  # no products: the bias and the residual are left
                _check_forward(y, x, w, b, r, "silu")
            assert dx.shape == x.shape and dw.shape == w.shape and db.shape == b.shape
            if m == 0:
                assert not dw.any() and not db.any()
            if n == 0:
                assert not dx.any()
    N.check_device_status(DEV)


def test_rows_behind_the_last_are_left_alone():
    """Tiles reach past the last row and column; nothing there is written."""
    lib = N.load()
    m, k, n = 130, 72, 136
    x, w = _rand((m, k), torch.bfloat16, 51), _rand((n, k), torch.bfloat16, 52)
    room = torch.full((m * n + 4096,), 7.0, dtype=torch.bfloat16, device=DEV)
    nbytes = lib.sv_linear_workspace_bytes(N.SV_LINEAR_FORWARD, m, k, n, 2, 0)
    ws = N.workspace(nbytes, DEV)
    rc = lib.sv_linear_forward(x.data_ptr(), k, w.data_ptr(), k, None, None, 0, None, None, m, k, n,
                               2, 2, 0, room.data_ptr(), None, ws.data_ptr(), nbytes,
                               N.status_word(DEV).data_ptr(), N.stream(DEV))
    N.check(rc, "linear")
    assert torch.equal(room[: m * n].view(m, n), linear(x, w))
    assert (room[m * n:] == 7).all()


def test_not_finite_values_stay_in_their_rows():
    x, w = _rand((300, 128), torch.bfloat16, 61), _rand((64, 128), torch.bfloat16, 62)
    clean = linear(x, w, activation="gelu_tanh")
    x[17, 3] = float("nan")
    x[290, 5] = float("inf")
    got = linear(x, w, activation="gelu_tanh")
    keep = torch.ones(300, dtype=torch.bool, device=DEV)
    keep[[17, 290]] = False
    assert torch.equal(got[keep], clean[keep])
    assert torch.isnan(got[17]).all() and not torch.isfinite(got[290]).all()
    big = torch.tensor([[-300.0], [-30.0], [30.0], [300.0]], device=DEV)
    one = torch.ones((1, 1), device=DEV)
    for act in ("silu", "gelu", "gelu_tanh"):
        y = linear(big, one, activation=act)
        assert torch.isfinite(y).all() and y[3] == 300 and y[0].abs() == 0


def test_two_streams_and_two_graphs():
    x, w = _rand((1500, 512), torch.bfloat16, 71), _rand((512, 512), torch.bfloat16, 72, 0.05)
    x2 = _rand((1500, 512), torch.bfloat16, 73)
    want, want2 = linear(x, w, activation="silu"), linear(x2, w, activation="silu")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    outs = [[], []]
    for _ in range(4):
        for i, (s, a) in enumerate(zip(streams, (x, x2))):
            with torch.cuda.stream(s):
                outs[i].append(linear(a, w, activation="silu"))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs[0])
    assert all(torch.equal(o, want2) for o in outs[1])
    few, tall = x[:40], x[:, :8].contiguous()  # split k, padded copies: both use workspaces
    narrow = _rand((512, 7), torch.bfloat16, 74)
    graphs, results = [], []
    for a in (few, x2[:40]):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append((linear(a, w), linear(tall[:, :7], narrow)))
        graphs.append(g)
    for g in graphs:
        g.replay()
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for (a, b), src in zip(results, (few, x2[:40])):
        assert torch.equal(a, linear(src, w)) and torch.equal(b, linear(tall[:, :7], narrow))
    N.check_device_status(DEV)


def test_norm_then_eight_bit_projection():
    """The 8-bit norm feeds the 8-bit projection: the two together against the formula on the values
    that the norm's output stands for."""
    x, r = _rand((333, 256), torch.bfloat16, 81), _rand((333, 256), torch.bfloat16, 82)
    w = _rand((128, 256), torch.float32, 83, 1 / 16)
    ws = w.abs().amax(1) / 448
    w8 = (w / ws[:, None]).to(torch.float8_e4m3fn)
    b = _rand((128,), torch.bfloat16, 84)
    (q, s), h = rms_norm(x, residual=r, quantize=True)
    got = linear(q, w8, b, activation="gelu_tanh", residual=h[:, :128], x_scale=s, weight_scale=ws)
    _check_forward(got, q, w8, b, h[:, :128], "gelu_tanh", s, ws)


def test_sparse_linear_with_epilogue():
    from mlx_diffuser_b200.layers.resblock import SparseLinear
    from mlx_diffuser_b200.layers.sparse import SparseTensor

    layer = SparseLinear(64, 96).to(DEV)
    f, r = _rand((50, 64), torch.bfloat16, 91), _rand((50, 96), torch.bfloat16, 92)
    coords = torch.zeros((50, 4), dtype=torch.int32, device=DEV)
    coords[:, 1] = torch.arange(50)
    x = SparseTensor(f, coords)
    w, b = layer.weight.to(torch.bfloat16), layer.bias.to(torch.bfloat16)
    assert torch.equal(layer(x).features, torch.nn.functional.linear(f, w, b))
    got = layer(x, activation="gelu_tanh", residual=r)
    assert got.cache is x.cache
    _check_forward(got.features, f, w, b, r, "gelu_tanh")
