"""The biased attention in fp16 / bf16 where magnitudes span many powers of two: tables that fall steeply,
rows whose output gradient lies far above the others', small output gradients and weights. Every
entry is held to what its own terms allow, not to the largest of the head.

Bounds, with u = 2^-24 and e = eps / 2 of the type: a score is off by (2 dim + 32) u of the magnitudes in
it, so a weight p by twice that (and its row's largest) of itself; dP by (2 dim + 16) u of |dout||v|; delta, a
mean of dP over rows, by as much of the row's mean of |dout||v| and by what the output keeps of the
forward pass, at most e^2 of |dout||out| twice over and half of the rest's smallest number (2^-25 of
2^-11 in fp16). So a score gradient is off by

    ds_off = |ds| (p's) + p (dP's + delta's),

none of it rounded to the type. A bucket of the table sums its terms in units of at most 2^-16 of its own
largest term, half a unit a pair, and is rounded once.

As operands of the second products weights and score gradients are rounded to the type, by e of
themselves. In fp16 they are raised first: below 2^-27 of a row's (or, for dv, of 1) a weight is off by 2^-38
of that at most, a score gradient below 2^-28 of its row's largest by 2^-39 of that."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mlx_diffuser_b200 import SparseTensor, _native as N
from mlx_diffuser_b200 import position_buckets, sparse_self_attention
from mlx_diffuser_b200.layers.sparse import attention_windows
from tests.test_position_bias_gpu import _close, _reference

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0**-24
F64 = torch.float64
HALVES = [torch.float16, torch.bfloat16]


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _least(dtype):
    """Half of the smallest subnormal number, which any rounding to the type may be off by."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def _voxels(n, grid, seed):
    cells = np.random.default_rng(seed).choice(grid**3, n, replace=False)
    rows = np.stack([np.zeros(n, np.int64), *np.unravel_index(cells, (grid,) * 3)], 1)
    return torch.from_numpy(rows.astype(np.int32)).to(DEV)


def _falling_table(heads, side, step, dtype):
    """-step for every voxel between query and key."""
    d = torch.arange(-side, side + 1, device=DEV).abs()
    far = d[:, None, None] + d[None, :, None] + d[None, None]
    return (-step * far.float()).to(dtype).expand(heads, -1, -1, -1).contiguous()


def _terms(coords, q, k, v, table, lut, window, dout):
    """Per window: its rows, the buckets [L, L], and p, ds and ds_off [heads, L, L]."""
    e = _half(q.dtype)
    small = 2.0**-36 if q.dtype == torch.float16 else 2.0**-126
    q, k, v, flat, dout = (t.detach().to(F64) for t in (q, k, v, table.flatten(1), dout))
    reach, nb, dim = lut.numel() // 2, table.shape[-1], q.shape[-1]
    x = SparseTensor(torch.zeros((len(coords), 1), device=DEV), coords)
    for rows in attention_windows(x, window).as_list():
        rows = rows.long()
        c = coords[rows, 1:].long()
        b = torch.zeros((len(rows),) * 2, dtype=torch.long, device=DEV)
        for a in range(3):
            d = (c[None, :, a] - c[:, None, a]).clamp(-reach, reach)
            b = b * nb + lut.long()[d + reach]
        qs, ks, vs, gs = (t[rows].transpose(0, 1) for t in (q, k, v, dout))
        s = qs @ ks.transpose(1, 2) * dim**-0.5 + flat[:, b]
        s_off = (2 * dim + 32) * U * (qs.abs() @ ks.abs().transpose(1, 2) * dim**-0.5 + s.abs())
        p = torch.softmax(s, -1)
        dp = gs @ vs.transpose(1, 2)
        mag = gs.abs() @ vs.abs().transpose(1, 2)
        delta = (p * dp).sum(-1, keepdim=True)
        out = p @ vs
        ds = p * (dp - delta)
        p_rel = 2 * s_off + 2 * s_off.amax(-1, keepdim=True) + 8 * U
        kept = (2 * e * e * gs.abs() * (p @ vs.abs()) + small * gs.abs()).sum(-1, keepdim=True)
        d_off = ((p * p_rel) @ vs.abs() * gs.abs()).sum(-1, keepdim=True) + kept + \
            (2 * dim + 2 * len(rows)) * U * (p * mag).sum(-1, keepdim=True) + \
            2 * dim * U * (gs.abs() * out.abs()).sum(-1, keepdim=True)
        ds_off = ds.abs() * p_rel + p * ((2 * dim + 16) * U * (mag + delta.abs()) + d_off)
        yield rows, b, p, ds, ds_off


def _check_table(coords, q, k, v, table, lut, window, dout, got):
    heads, cells = q.shape[1], table.shape[-1] ** 3
    want, off, top, count = (torch.zeros((heads, cells), dtype=F64, device=DEV) for _ in range(4))
    for _, b, _, ds, ds_off in _terms(coords, q, k, v, table, lut, window, dout):
        b = b.flatten().expand(heads, -1)
        want.scatter_add_(1, b, ds.flatten(1))
        off.scatter_add_(1, b, ds_off.flatten(1))
        count.scatter_add_(1, b, torch.ones_like(ds).flatten(1))
        top.scatter_reduce_(1, b, (ds.abs() + ds_off).flatten(1), "amax")
    off += 2.0**-17 * top * count
    bound = off + _half(q.dtype) * (want.abs() + off) + _least(q.dtype)
    err = (got.flatten(1).to(F64) - want).abs()
    assert (err <= bound).all(), float((err / bound).max())
    return want, bound


def _attend(coords, q, k, v, table, lut, window, dout):
    x = SparseTensor(torch.zeros((len(coords), 1), device=DEV), coords)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
    out = sparse_self_attention(x, *leaves[:3], window_size=window, position_bias=leaves[3],
                                position_buckets=lut)
    grads = torch.autograd.grad(out, leaves, dout)
    N.check_device_status(DEV)
    return out.detach(), *grads


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("step", [0.75, 1.5])
def test_table_that_falls_steeply(step, dtype):
    """The far buckets' score gradients lie 2^30 and more below the near ones', and are no less exact."""
    coords = _voxels(2500, 16, 1)
    lut = position_buckets(7, 7, device=DEV)
    q, k, v, dout = (_rand((2500, 2, 32), dtype, i) for i in range(4))
    table = _falling_table(2, 7, step, dtype)
    got = _attend(coords, q, k, v, table, lut, 8, dout)[4]
    want, bound = _check_table(coords, q, k, v, table, lut, 8, dout, got)
    known = bound < want.abs()
    assert known.double().mean() > 0.5 and got.flatten(1)[known].all()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("window,n", [(8, 2500), (None, 1500)])
def test_table_beside_one_large_output_gradient(window, n, dtype):
    """One row's output gradient 10^4 times the others': the buckets it does not reach are as exact as
    without it, and those it does to a share of their own terms."""
    coords = _voxels(n, 16, 2)
    reach = 7 if window else 15
    lut = position_buckets(reach, reach if window else 8, device=DEV)
    side = int(lut.max()) // 2
    q, k, v, dout = (_rand((n, 2, 32), dtype, 10 + i) for i in range(4))
    if dtype == torch.float16:
        dout *= 0.25  # so that the large one is finite in the type
    dout[n // 2] *= 1e4
    table = _rand((2, *(2 * side + 1,) * 3), dtype, 14)
    got = _attend(coords, q, k, v, table, lut, window, dout)[4]
    _check_table(coords, q, k, v, table, lut, window, dout, got)


@pytest.mark.parametrize("dtype", HALVES)
def test_table_beside_a_value_that_is_not_finite(dtype):
    """Only the buckets of its own pairs lose their gradient: ds_ij holds dout_i and no other row's."""
    coords = _voxels(1200, 16, 3)
    far = torch.tensor([[0, 40, 40, 40], [0, 41, 40, 40]], dtype=torch.int32, device=DEV)
    coords = torch.cat([coords, far])
    n = len(coords)
    lut = position_buckets(7, 7, device=DEV)
    q, k, v, dout = (_rand((n, 2, 32), dtype, 20 + i) for i in range(4))
    table = _rand((2, 15, 15, 15), dtype, 24)
    clean = _attend(coords, q, k, v, table, lut, 8, dout)[4]
    dout[-1, 1, 3] = float("inf")
    got = _attend(coords, q, k, v, table, lut, 8, dout)[4]
    touched = torch.zeros((2, 15, 15, 15), dtype=torch.bool, device=DEV)
    touched[1, 6:8, 7, 7] = True  # from it to the other row and to itself: -1 and 0 along x
    assert torch.equal(got[~touched], clean[~touched])
    assert not torch.isfinite(got[touched]).any()


def _check_rows(coords, q, k, v, table, lut, window, dout, got, whole=2.0):
    """out, dq, dk and dv against the formula, entry by entry, and (the errors of single operands being
    independent) as a whole: an operand's rounding and the result's, each half a step, give 2^0.5 of the
    result's alone; ``whole`` leaves room for ds_off and the sums. The result's is taken as what rounding
    the exact value to the type leaves."""
    dtype = q.dtype
    e, scale = _half(dtype), q.shape[-1] ** -0.5
    wants = [torch.zeros(q.shape, dtype=F64, device=DEV) for _ in range(4)]
    offs = [torch.zeros(q.shape, dtype=F64, device=DEV) for _ in range(4)]
    small_p, small_ds = (2.0**-38, 2.0**-39) if dtype == torch.float16 else (2.0**-126,) * 2
    for rows, _, p, ds, ds_off in _terms(coords, q, k, v, table, lut, window, dout):
        n = len(rows)
        qs, ks, vs, gs = (t.detach().to(F64)[rows].transpose(0, 1) for t in (q, k, v, dout))
        s_off = (2 * q.shape[-1] + 32) * U * (
            qs.abs() @ ks.abs().transpose(1, 2) * scale + table.abs().max().double())
        p_off = p * (2 * s_off + 2 * s_off.amax(-1, keepdim=True) + 8 * U + e + 2 * n * U)
        t_off = ds_off + (e + 2 * n * U) * ds.abs()
        by_query = t_off + small_ds * ds.abs().amax(-1, keepdim=True)
        by_key = t_off + small_ds * ds.abs().amax(-2, keepdim=True)
        for i, (value, off) in enumerate((
                (p @ vs, (p_off + small_p) @ vs.abs()),
                (ds @ ks * scale, by_query @ ks.abs() * scale),
                (ds.transpose(1, 2) @ qs * scale, by_key.transpose(1, 2) @ qs.abs() * scale),
                (p.transpose(1, 2) @ gs, (p_off + small_p).transpose(1, 2) @ gs.abs()))):
            wants[i][rows] = value.transpose(0, 1)
            offs[i][rows] = (off + e * (value.abs() + off)).transpose(0, 1) + _least(dtype)
    for name, a, want, off in zip(("out", "dq", "dk", "dv"), got, wants, offs):
        err = (a.to(F64) - want).abs()
        assert (err <= off).all(), (name, float((err / off).max()))
        alone = (want.to(dtype).to(F64) - want).norm()
        assert err.norm() <= whole * alone, (name, float(err.norm() / alone))


@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-4])
def test_small_output_gradients_in_half_precision(size):
    """4,096 rows that all see each other: score gradients around 2^-12 of the output's, which for a mean
    loss is below the smallest numbers of the type."""
    coords = _voxels(4096, 16, 4)
    lut = position_buckets(15, 8, device=DEV)
    q, k, v = (_rand((4096, 2, 64), torch.float16, 30 + i) for i in range(3))
    dout = _rand((4096, 2, 64), torch.float16, 33, size)
    table = _rand((2, 17, 17, 17), torch.float16, 34)
    got = _attend(coords, q, k, v, table, lut, None, dout)
    _check_rows(coords, q, k, v, table, lut, None, dout, got[:4])
    _check_table(coords, q, k, v, table, lut, None, dout, got[4])


@pytest.mark.parametrize("window", [8, None])
@pytest.mark.parametrize("dtype", HALVES)
def test_weights_far_below_the_largest(dtype, window):
    """Every row sees itself e^17 times as much as any other, and half of the rows hold nothing: their
    outputs are sums of weights around 2^-24."""
    n = 2500 if window else 3000
    coords = _voxels(n, 16, 5)
    reach = 7 if window else 15
    lut = position_buckets(reach, 3, device=DEV)
    q, k = (_rand((n, 2, 32), dtype, 40 + i, 0.1) for i in range(2))
    v = 1 + _rand((n, 2, 32), dtype, 42, 0.25)
    v[::2] = 0
    dout = _rand((n, 2, 32), dtype, 43)
    dout[1::2] = 0
    table = torch.zeros((2, 7, 7, 7), dtype=dtype, device=DEV)
    table[:, 3, 3, 3] = 17
    got = _attend(coords, q, k, v, table, lut, window, dout)
    _check_rows(coords, q, k, v, table, lut, window, dout, got[:4])
    x = SparseTensor(torch.zeros((n, 1), device=DEV), coords)
    serving = sparse_self_attention(x, q, k, v, window_size=window, position_bias=table,
                                    position_buckets=lut)
    _check_rows(coords, q, k, v, table, lut, window, dout, (serving,))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("n,window,dim", [(2500, 8, 64), (600, 2, 32), (1200, None, 64)])
def test_gradients_as_a_whole(n, window, dim, dtype):
    """Nothing but the operand's and the result's rounding: within 1.5 of the result's, where 2^0.5 is
    theirs. A delta from the rounded output, or one weight's rounding more in it, would add as much again
    in windows of a few hundred rows."""
    coords = _voxels(n, 16, 6)
    reach = 7 if window else 15
    lut = position_buckets(reach, 7, device=DEV)
    q, k, v, dout = (_rand((n, 2, dim), dtype, 60 + i) for i in range(4))
    table = _rand((2, 15, 15, 15), dtype, 64)
    got = _attend(coords, q, k, v, table, lut, window, dout)
    _check_rows(coords, q, k, v, table, lut, window, dout, got[:4], 1.5)
    _check_table(coords, q, k, v, table, lut, window, dout, got[4])


@pytest.mark.parametrize("window", [8, None])
@pytest.mark.parametrize("dtype", [torch.float32, *HALVES])
def test_row_order(dtype, window):
    """The same voxels in another order: the same results but for rounding, row by row, and the same
    table gradient, each within the bounds of the formula."""
    n = 1100
    coords = _voxels(n, 16, 7)
    reach = 7 if window else 15
    lut = position_buckets(reach, 5, device=DEV)
    q, k, v, dout = (_rand((n, 2, 32), dtype, 70 + i) for i in range(4))
    table = _rand((2, 11, 11, 11), dtype, 74)
    x = SparseTensor(torch.zeros((n, 1), device=DEV), coords)
    val, off = _reference(x, q, k, v, table, lut, window, (0, 0, 0), dout)
    for seed in range(3):
        order = torch.randperm(n, generator=torch.Generator().manual_seed(seed)).to(DEV)
        if seed == 0:
            order = torch.arange(n - 1, -1, -1, device=DEV)
        got = _attend(*(t[order].contiguous() for t in (coords, q, k, v)), table, lut, window,
                      dout[order].contiguous())
        for name, a in zip(("out", "dq", "dk", "dv"), got):
            back = torch.empty_like(a)
            back[order] = a
            _close(back, val[name], off[name], name)
        _close(got[4], val["dtable"], off["dtable"], "dtable")
