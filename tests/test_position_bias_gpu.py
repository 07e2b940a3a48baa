"""``sparse_self_attention`` with a relative position bias on the GPU against its formula in 64 bits:
window shapes from lone voxels to whole batch elements, head sizes, types, strides, gradients.

Bounds, with u = 2^-24 and e = eps / 2 of the type (a rounding is off by at most that): a score is
off by ds <= (2 dim + 32) u (scale |q||k| + |s|) with exp and the running rescales in the 32; a weight
p by p (2 ds + e), the e for the type it is multiplied in; sums of n products by 2 n u of their
magnitudes. Below the normal range these are absolute: exp may give zero for results under 2^-126,
and a rounding to the type is off by half its smallest subnormal number."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mlx_diffuser_b200 import SparseTensor, _native as N
from mlx_diffuser_b200 import linear, position_buckets, rms_norm, sparse_self_attention
from mlx_diffuser_b200.layers.sparse import attention_windows

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0**-24
F64 = torch.float64
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _voxels(n, grid, batch, seed):
    """n distinct voxels of a grid per batch element, in a random order."""
    rng = np.random.default_rng(seed)
    rows = []
    for b in range(batch):
        cells = rng.choice(grid**3, n, replace=False)
        rows.append(np.stack([np.full(n, b), *np.unravel_index(cells, (grid,) * 3)], 1))
    rows = np.concatenate(rows)
    return torch.from_numpy(rows[rng.permutation(len(rows))].astype(np.int32)).to(DEV)


def _tensor(coords):
    return SparseTensor(torch.zeros((len(coords), 1), device=DEV), coords)


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def _reference(x, q, k, v, table, lut, window, shift, dout=None):
    """The formula per window in 64 bits, with a bound for every value."""
    dtype = q.dtype
    e = _half(dtype)
    q, k, v, table = (t.detach().to(F64) for t in (q, k, v, table))
    g = None if dout is None else dout.to(F64)
    n, heads, dim = q.shape
    reach, nb, scale = lut.numel() // 2, table.shape[-1], dim**-0.5
    names = ["out"] + (["dq", "dk", "dv"] if g is not None else [])
    val = {m: torch.zeros_like(q) for m in names}
    off = {m: torch.zeros_like(q) for m in names}
    flat = table.reshape(heads, -1)
    val["dtable"], off["dtable"] = torch.zeros_like(flat), torch.zeros_like(flat)
    count = torch.zeros(nb**3, dtype=F64, device=DEV)
    top = torch.zeros(heads, dtype=F64, device=DEV)
    groups = attention_windows(_tensor(x.coords), window, shift)
    for rows in groups.as_list():
        rows = rows.long()
        size = len(rows)
        c = x.coords[rows, 1:].long()
        b = torch.zeros((size, size), dtype=torch.long, device=DEV)
        for a in range(3):
            d = (c[None, :, a] - c[:, None, a]).clamp(-reach, reach)
            b = b * nb + lut.long()[d + reach].clamp(0, nb - 1)
        qs, ks, vs = (t[rows].transpose(0, 1) for t in (q, k, v))
        s = qs @ ks.transpose(1, 2) * scale + flat[:, b]
        ds_off = (2 * dim + 32) * U * (qs.abs() @ ks.abs().transpose(1, 2) * scale + s.abs())
        p = torch.softmax(s, -1)
        p = torch.where(torch.isnan(p), torch.zeros_like(p), p)  # nothing but -inf
        ds_off = torch.where(torch.isfinite(ds_off), ds_off, torch.zeros_like(ds_off))
        p_rel = 2 * ds_off + 2 * ds_off.amax(-1, keepdim=True) + e + 8 * U
        o = p @ vs
        low = max(torch.finfo(dtype).smallest_normal * e, 2.0**-126)
        o_off = (p * p_rel + low) @ vs.abs() + 2 * size * U * (p @ vs.abs())
        val["out"][rows] = o.transpose(0, 1)
        off["out"][rows] = (o_off + e * (o.abs() + o_off)).transpose(0, 1)
        if g is None:
            continue
        gs = g[rows].transpose(0, 1)
        dp = gs @ vs.transpose(1, 2)
        delta = (p * dp).sum(-1, keepdim=True)
        w = dp - delta
        # dp's own sum, and delta from the rounded output
        w_off = (2 * dim + 16) * U * (gs.abs() @ vs.abs().transpose(1, 2)) + \
            (gs.abs() * (o_off + e * (o.abs() + o_off)) + 2 * dim * U * gs.abs() * o.abs()
             ).sum(-1, keepdim=True)
        ds = p * w
        # before its own rounding to the type, and with it
        ds32_off = (p * (p_rel - e) + 2.0**-126) * w.abs() + p * w_off
        ds_t_off = ds32_off + e * (ds.abs() + ds32_off) + low
        dv = p.transpose(1, 2) @ gs
        dv_off = (p * p_rel + low).transpose(1, 2) @ gs.abs() + 2 * size * U * \
            (p.transpose(1, 2) @ gs.abs())
        dq, dk = ds @ ks * scale, ds.transpose(1, 2) @ qs * scale
        dq_off = (ds_t_off + 2 * size * U * ds.abs()) @ ks.abs() * scale
        dk_off = (ds_t_off + 2 * size * U * ds.abs()).transpose(1, 2) @ qs.abs() * scale
        for m, value, bound in (("dq", dq, dq_off), ("dk", dk, dk_off), ("dv", dv, dv_off)):
            val[m][rows] = value.transpose(0, 1)
            off[m][rows] = (bound + (e + 4 * U) * (value.abs() + bound)).transpose(0, 1)
        val["dtable"].index_add_(1, b.flatten(), ds.flatten(1))
        off["dtable"].index_add_(1, b.flatten(), ds32_off.flatten(1))
        top = torch.maximum(top, torch.maximum(ds.abs().amax((1, 2)),
                                               2.0**-14 * delta.abs().amax((1, 2))))
        count.index_add_(0, b.flatten(), torch.ones_like(b.flatten(), dtype=F64))
    if g is not None:
        # the 16-bit kernels sum the table in fixed point: half a unit a pair, the unit 2^-17 of the
        # power of two above the head's largest |ds| (at least 2^-14 of the largest |delta|)
        # fp32: half of 2^-61 of the power of two above 2 n |g| |v|
        half_unit = 2.0**-17 * top
        if dtype == torch.float32:
            half_unit = 2.0**-61 * 2 * n * g.norm(dim=2).amax(0) * v.norm(dim=2).amax(0)
        off["dtable"] += half_unit[:, None] * count
        off["dtable"] += e * (val["dtable"].abs() + off["dtable"])
    shape = (heads, nb, nb, nb)
    val["dtable"], off["dtable"] = val["dtable"].view(shape), off["dtable"].view(shape)
    return val, off


def _close(got, want, off, what):
    err = (got.detach().to(F64) - want).abs()
    bound = off + torch.finfo(got.dtype).tiny
    assert (err <= bound).all(), (what, float((err / bound).max()))


def _run(coords, heads, dim, dtype, window, shift, reach, side, train=True, seed=0, lut=None,
         qkv=None, table=None):
    x = _tensor(coords)
    n = len(coords)
    lut = position_buckets(reach, side, device=DEV) if lut is None else lut
    nb = 2 * min(side, reach) + 1
    if qkv is None:
        qkv = [_rand((n, heads, dim), dtype, seed + i) for i in range(3)]
    if table is None:
        table = _rand((heads, nb, nb, nb), dtype, seed + 3)
    dout = _rand((n, heads, dim), dtype, seed + 4)
    args = [t.requires_grad_(train) if t.is_leaf else t for t in (*qkv, table)]
    out = sparse_self_attention(x, *args[:3], window_size=window, shift_window=shift,
                                position_bias=args[3], position_buckets=lut)
    grads = torch.autograd.grad(out, args, dout) if train else ()
    N.check_device_status(DEV)
    val, off = _reference(x, *args, lut, window, shift, dout if train else None)
    for what, got in zip(("out", "dq", "dk", "dv", "dtable"), (out, *grads)):
        assert got.dtype == dtype and got.shape == val[what].shape
        _close(got, val[what], off[what], what)
    return out, grads


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [8, 16, 24, 32, 40, 64, 100, 128])
def test_head_sizes(dim, dtype):
    _run(_voxels(150, 12, 2, dim), 3, dim, dtype, 5, (1, 2, 3), 4, 4, seed=dim)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,grid,window", [(1, 4, 2), (2, 4, None), (63, 8, 8), (64, 8, 8),
                                           (65, 8, None), (200, 40, 2), (300, 7, 7),
                                           (400, 8, None), (500, 16, 4)])
def test_window_shapes(n, grid, window, dtype):
    """Lone voxels, full tiles and one more, whole batch elements, many tiny windows."""
    _run(_voxels(n, grid, 2, n), 2, 32, dtype, window, (1, 0, 1) if window else (0, 0, 0),
         6, 3, seed=n)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_window(dtype):
    _run(_voxels(1500, 16, 1, 5), 1, 64, dtype, None, (0, 0, 0), 15, 4, seed=5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,dim", [(1, 8), (2, 64), (300, 24), (300, 128)])
def test_lone_rows(n, dim, dtype):
    """Windows of one row: the output is v, dv is dout, and the score, which changes nothing, has a
    gradient of exactly zero."""
    coords = torch.zeros((n, 4), dtype=torch.int32, device=DEV)
    coords[:, 1] = 4 * torch.arange(n, device=DEV)
    x = _tensor(coords)
    leaves = [_rand((n, 2, dim), dtype, i).requires_grad_(True) for i in range(3)]
    leaves.append(_rand((2, 7, 7, 7), dtype, 3).requires_grad_(True))
    dout = _rand((n, 2, dim), dtype, 4)
    out = sparse_self_attention(x, *leaves[:3], window_size=4, position_bias=leaves[3],
                                position_buckets=position_buckets(3, 3, device=DEV))
    dq, dk, dv, dtable = torch.autograd.grad(out, leaves, dout)
    assert torch.equal(out, leaves[2]) and torch.equal(dv, dout)
    assert not dq.any() and not dk.any() and not dtable.any()


def _parts_bytes(n, heads, dim, dtype, windows):
    return N.load().sv_window_attention_workspace_bytes(n, heads, dim, N.DTYPE_CODE[dtype], windows)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [24, 64, 100, 128])
def test_long_windows_in_parts(dim, dtype):
    """Few rows of long windows: the walk over the keys is split and joined."""
    coords = _voxels(1100, 16, 2, dim)
    if dtype != torch.float32:
        assert _parts_bytes(2200, 2, dim, dtype, 2) > 0
    _run(coords, 2, dim, dtype, None, (0, 0, 0), 15, 3, seed=dim)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_parts_with_masks_and_not_finite_values(dtype):
    """A head that sees nothing, one whose keys lie in one direction (so that some parts of a row hold
    none), and a NaN and an infinity in one of two windows."""
    coords = _voxels(1000, 16, 2, 3)
    x = _tensor(coords)
    lut = position_buckets(15, 2, device=DEV)
    table = _rand((2, 5, 5, 5), dtype, 5)
    table[0, 2:] = float("-inf")
    table[1] = float("-inf")
    q, k, v = (_rand((2000, 2, 64), dtype, 6 + i) for i in range(3))
    assert _parts_bytes(2000, 2, 64, dtype, 2) > 0

    def run():
        return sparse_self_attention(x, q, k, v, window_size=None, position_bias=table,
                                     position_buckets=lut)

    val, off = _reference(x, q, k, v, table, lut, None, (0, 0, 0))
    out = run()
    _close(out, val["out"], off["out"], "out")
    assert not out[:, 1].any()
    table[1] = 0
    val, off = _reference(x, q, k, v, table, lut, None, (0, 0, 0))
    first = torch.nonzero(coords[:, 0] == 0).flatten()
    rest = coords[:, 0] == 1
    k[first[3], 1, 4] = float("inf")
    v[first[9], 1, 7] = float("nan")
    got = run()
    _close(got[rest], val["out"][rest], off["out"][rest], "out")
    assert torch.isnan(got[~rest, 1, 7]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_windows_of_every_length(dtype):
    """Windows of 1 to 140 rows in a row, so that blocks hold several, one, and a part of one."""
    sizes = [1, 2, 31, 32, 33, 1, 63, 64, 65, 5, 127, 128, 129, 1, 1, 1, 140, 30, 3]
    rows = []
    for i, n in enumerate(sizes):
        at = np.arange(n)
        rows.append(np.stack([np.zeros(n, int), 6 * i + at // 36, at // 6 % 6, at % 6], 1))
    coords = torch.from_numpy(np.concatenate(rows).astype(np.int32)).to(DEV)
    for seed in range(2):
        order = torch.randperm(len(coords), generator=torch.Generator().manual_seed(seed)).to(DEV)
        _run(coords[order].contiguous() if seed else coords, 2, 32, dtype, 6, (0, 0, 0), 5, 5,
             seed=seed)
    # scores around -68, far below the zero that a row of zeros would score
    n = len(coords)
    base = torch.ones((1, 2, 32), device=DEV)
    q = (-12 * base + _rand((n, 2, 32), torch.float32, 8, 0.1)).to(dtype)
    k = (base + _rand((n, 2, 32), torch.float32, 9, 0.1)).to(dtype)
    _run(coords, 2, 32, dtype, 6, (0, 0, 0), 5, 5, qkv=[q, k, _rand((n, 2, 32), dtype, 10)])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reach,side", [(1, 1), (7, 7), (12, 12), (31, 5), (1023, 12)])
def test_tables(reach, side, dtype):
    _run(_voxels(220, 10, 1, reach), 2, 32, dtype, 8, (4, 4, 4), reach, side, seed=reach)


def test_one_bucket_and_a_table_for_everything():
    lut = torch.zeros(1, dtype=torch.int32, device=DEV)
    table = _rand((2, 1, 1, 1), torch.bfloat16, 3)
    _run(_voxels(100, 8, 1, 2), 2, 32, torch.bfloat16, 4, (0, 0, 0), 0, 0, lut=lut, table=table)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_views(dtype):
    coords = _voxels(180, 10, 1, 7)
    n = len(coords)
    fused = _rand((n, 3, 4, 32), dtype, 8)
    _run(coords, 4, 32, dtype, 5, (0, 0, 0), 4, 4, train=False, qkv=list(fused.unbind(1)))
    odd = _rand((n, 4 * 3 * 33 + 1), dtype, 9)[:, 1:].view(n, 4, 3, 33)
    # heads outermost in memory, and rows that start off a 16-byte boundary
    _run(coords, 4, 33, dtype, 5, (0, 0, 0), 4, 4, train=False,
         qkv=[odd[:, :, i] for i in range(3)])
    headed = _rand((4, n, 3, 32), dtype, 10).transpose(0, 1)
    leaf = headed.detach().clone(memory_format=torch.preserve_format)
    qkv = [leaf[:, :, i].requires_grad_(True) for i in range(3)]
    _run(coords, 4, 32, dtype, 5, (0, 0, 0), 4, 4, qkv=qkv)
    crossed = _rand((n, 32, 4), dtype, 11).transpose(1, 2)  # channels not contiguous
    _run(coords, 4, 32, dtype, 5, (0, 0, 0), 4, 4, train=False, qkv=[crossed] * 3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores_keep_the_softmax_finite(dtype):
    coords = _voxels(200, 9, 1, 3)
    qkv = [_rand((200, 2, 32), dtype, 20 + i, 12.0) for i in range(2)]
    qkv.append(_rand((200, 2, 32), dtype, 22))
    out, grads = _run(coords, 2, 32, dtype, None, (0, 0, 0), 8, 8, qkv=qkv)
    assert all(torch.isfinite(t).all() for t in (out, *grads))


@pytest.mark.parametrize("dtype", DTYPES)
def test_table_entries_that_mask(dtype):
    """-inf in the table: pairs out of sight, and rows that see nothing."""
    coords = _voxels(160, 8, 1, 4)
    lut = position_buckets(7, 7, device=DEV)
    table = _rand((2, 15, 15, 15), dtype, 30)
    table[0, 8:] = float("-inf")  # head 0 sees no key ahead of it along x
    table[1] = float("-inf")      # head 1 sees nothing
    out, grads = _run(coords, 2, 32, dtype, 4, (0, 0, 0), 7, 7, lut=lut, table=table)
    assert all(torch.isfinite(t).all() for t in (out, *grads))
    assert not out[:, 1].any() and not any(g[:, 1].any() for g in grads[:3])
    assert not grads[3][1].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_table_entries_of_the_lowest_value(dtype):
    """The type's lowest value masks like -inf beside ordinary entries; where a row has nothing else,
    every score is that value in fp32 (the products vanish beside it), so the weights are equal."""
    coords = _voxels(160, 8, 1, 4)
    x = _tensor(coords)
    lut = position_buckets(7, 7, device=DEV)
    low = torch.finfo(dtype).min
    table = _rand((2, 15, 15, 15), dtype, 30)
    hidden = table.clone()
    table[0, 8:], hidden[0, 8:] = low, float("-inf")
    table[1] = low
    q, k, v, dout = (_rand((160, 2, 32), dtype, 31 + i) for i in range(4))

    def run(t, qq):
        leaves = [a.clone().requires_grad_(True) for a in (qq, k, v, t)]
        out = sparse_self_attention(x, *leaves[:3], window_size=4, position_bias=leaves[3],
                                    position_buckets=lut)
        return (out, *torch.autograd.grad(out, leaves, dout))

    got, want = run(table, q), run(hidden, q)
    for a, b in zip(got[:4], want[:4]):
        assert torch.equal(a[:, 0], b[:, 0])
    assert torch.equal(got[4][0], want[4][0])
    flat = table.clone()
    flat[1] = 0
    zero = q.clone()
    zero[:, 1] = 0
    alike = run(flat, zero)  # equal scores of zero
    for i in (0, 3):  # out and dv
        assert torch.equal(got[i][:, 1], alike[i][:, 1])
    assert torch.isfinite(got[2]).all()
    assert torch.equal(got[1][:, 1], alike[1][:, 1])
    assert torch.equal(got[4][1], alike[4][1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_not_finite_values_stay_in_their_window(dtype):
    coords = _voxels(300, 12, 1, 6)
    x = _tensor(coords)
    q, k, v = (_rand((300, 2, 32), dtype, 40 + i) for i in range(3))
    table, lut = _rand((2, 7, 7, 7), dtype, 43), position_buckets(3, 3, device=DEV)

    def run(*qkv):
        leaves = [t.clone().requires_grad_(True) for t in (*qkv, table)]
        out = sparse_self_attention(x, *leaves[:3], window_size=4, position_bias=leaves[3],
                                    position_buckets=lut)
        return (out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out)))

    clean = run(q, k, v)
    val, off = _reference(x, q, k, v, table, lut, 4, (0, 0, 0), torch.ones_like(q))
    bad = 17
    near = (coords[:, 1:] // 4 == coords[bad, 1:] // 4).all(1)
    for which in range(3):
        args = [q.clone(), k.clone(), v.clone()]
        args[which][bad, 1, 5] = float("nan")
        got = run(*args)
        for a, b, what in zip(got[:4], clean[:4], ("out", "dq", "dk", "dv")):
            assert torch.equal(a[:, 0], b[:, 0])
            # rows that shared a tile with the NaN are computed again without the tile's roundings,
            # so they keep the bounds and not the bits
            _close(a[~near], val[what][~near], off[what][~near], what)
        assert torch.isnan(got[0][bad, 1, 5 if which == 2 else 0])
        assert torch.equal(got[4][0], clean[4][0]) and torch.isnan(got[4][1]).any()


def test_far_coordinates_and_duplicates():
    c = torch.tensor([[0, -2**31, 0, 5], [0, 2**31 - 1, 0, 5], [0, 0, 0, 5], [0, 0, 0, 5],
                      [0, 3, -7, 2**31 - 1]], dtype=torch.int32, device=DEV)
    for dtype in DTYPES:
        _run(c, 2, 16, dtype, None, (0, 0, 0), 31, 8, seed=3)


def test_bucket_values_outside_the_table_are_clamped():
    lut = position_buckets(3, 3, device=DEV)
    wild = lut.clone()
    wild[0], wild[6] = -5, 99
    for dtype in DTYPES:
        a = _run(_voxels(60, 5, 1, 8), 2, 16, dtype, None, (0, 0, 0), 3, 3, lut=lut)
        b = _run(_voxels(60, 5, 1, 8), 2, 16, dtype, None, (0, 0, 0), 3, 3, lut=wild)
        assert torch.equal(a[0], b[0]) and all(torch.equal(s, t) for s, t in zip(a[1], b[1]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_results_repeat_and_do_not_depend_on_the_row_order(dtype):
    coords = _voxels(700, 14, 1, 9)
    a = _run(coords, 2, 64, dtype, 7, (0, 0, 0), 6, 6)
    b = _run(coords, 2, 64, dtype, 7, (0, 0, 0), 6, 6)
    assert torch.equal(a[0], b[0]) and all(torch.equal(s, t) for s, t in zip(a[1], b[1]))


def test_gradient_against_differences():
    coords = _voxels(40, 5, 1, 11)
    x = _tensor(coords)
    lut = position_buckets(4, 2, device=DEV)
    leaves = [_rand((40, 2, 8), torch.float32, 50 + i).requires_grad_(True) for i in range(3)]
    leaves.append(_rand((2, 5, 5, 5), torch.float32, 53).requires_grad_(True))
    dout = _rand((40, 2, 8), torch.float32, 54)
    out = sparse_self_attention(x, *leaves[:3], window_size=3, position_bias=leaves[3],
                                position_buckets=lut)
    grads = torch.autograd.grad(out, leaves, dout)
    args = [t.detach().to(F64) for t in leaves]

    def loss(*a):
        val, _ = _reference(x, *a, lut, 3, (0, 0, 0))
        return (val["out"] * dout.to(F64)).sum()

    for i, grad in enumerate(grads):
        step = _rand(args[i].shape, torch.float32, 60 + i).to(F64)
        up, down = ([a + (s * 1e-5 * step if i == j else 0) for j, a in enumerate(args)]
                    for s in (1, -1))
        want = (loss(*up) - loss(*down)) / 2e-5
        assert abs((grad.to(F64) * step).sum() - want) <= 2e-5 * (grad.to(F64) * step).abs().sum()


def test_empty_tensor_and_partial_gradients():
    coords = torch.zeros((0, 4), dtype=torch.int32, device=DEV)
    x = SparseTensor(torch.zeros((0, 1), device=DEV), coords)
    lut = position_buckets(3, 3, device=DEV)
    table = _rand((2, 7, 7, 7), torch.bfloat16, 1).requires_grad_(True)
    q = torch.zeros((0, 2, 32), dtype=torch.bfloat16, device=DEV, requires_grad=True)
    out = sparse_self_attention(x, q, q, q, window_size=4, position_bias=table,
                                position_buckets=lut)
    dq, dt = torch.autograd.grad(out.sum(), (q, table))
    assert out.shape == (0, 2, 32) and dq.shape == q.shape and not dt.any()
    x = _tensor(_voxels(90, 6, 1, 12))
    for dtype in DTYPES:
        q, k, v = (_rand((90, 2, 32), dtype, 70 + i) for i in range(3))
        t = table.detach().to(dtype)
        kw = dict(window_size=4, position_buckets=lut)
        full = [a.clone().requires_grad_(True) for a in (q, k, v, t)]
        want = torch.autograd.grad(sparse_self_attention(x, *full[:3], position_bias=full[3],
                                                         **kw).sum(), full)
        for i in range(4):
            some = [a.clone() for a in (q, k, v, t)]
            some[i].requires_grad_(True)
            got, = torch.autograd.grad(sparse_self_attention(x, *some[:3], position_bias=some[3],
                                                             **kw).sum(), some[i])
            assert torch.equal(got, want[i])


def test_plan_of_a_captured_call_is_not_for_others():
    """Windows known, their plan not: the capture lays out its own, which holds nothing until a replay;
    a call outside lays out another."""
    coords = _voxels(500, 12, 1, 14)
    x = _tensor(coords)
    q, k, v = (_rand((500, 2, 32), torch.bfloat16, 90 + i) for i in range(3))
    table, lut = _rand((2, 9, 9, 9), torch.bfloat16, 93), position_buckets(4, 4, device=DEV)

    def run(t):
        return sparse_self_attention(t, q, k, v, window_size=5, position_bias=table,
                                     position_buckets=lut)

    want = run(_tensor(coords))
    attention_windows(x, 5, (0, 0, 0))
    N.status_word(DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = run(x)
    outside = run(x)
    assert torch.equal(outside, want)
    graph.replay()
    assert torch.equal(inside, want)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = run(x)
    side.synchronize()
    assert torch.equal(again, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_streams_graph_and_cached_windows(dtype):
    coords = _voxels(500, 12, 1, 13)
    x = _tensor(coords)
    q, k, v = (_rand((500, 4, 32), dtype, 80 + i) for i in range(3))
    table, lut = _rand((4, 9, 9, 9), dtype, 83), position_buckets(4, 4, device=DEV)

    def run():
        return sparse_self_attention(x, q, k, v, window_size=5, position_bias=table,
                                     position_buckets=lut)

    want = run()
    assert attention_windows(x, 5).plan is not None
    torch.cuda.synchronize()
    side = torch.cuda.Stream(DEV)
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    v.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, run()) and torch.equal(captured, -want)
    # coordinates changed in place: the plan is built again
    x.coords[:, 1] = x.coords[:, 1].flip(0)
    val, off = _reference_cached(x, q, k, v, table, lut)
    _close(run(), val, off, "out")


def _reference_cached(x, q, k, v, table, lut):
    """The formula on the windows that the tensor's cache holds, whatever its coordinates are now."""
    groups = attention_windows(x, 5)
    dim = q.shape[-1]
    e = _half(q.dtype)
    q, k, v, flat = (t.to(F64) for t in (q, k, v, table.flatten(1)))
    val, off = torch.zeros_like(q), torch.zeros_like(q)
    for rows in groups.as_list():
        rows = rows.long()
        c = x.coords[rows, 1:].long()
        d = (c[None] - c[:, None]).clamp(-4, 4)
        b = lut.long()[d + 4]
        b = (b[..., 0] * 9 + b[..., 1]) * 9 + b[..., 2]
        qs, ks, vs = (t[rows].transpose(0, 1) for t in (q, k, v))
        s = qs @ ks.transpose(1, 2) * dim**-0.5 + flat[:, b]
        p = torch.softmax(s, -1)
        val[rows] = (p @ vs).transpose(0, 1)
        off[rows] = ((4 * e + 1e-5) * (p @ vs.abs())).transpose(0, 1)
    return val, off


@pytest.mark.parametrize("dtype", DTYPES)
def test_transformer_block(dtype):
    """norm -> projection -> windowed attention -> projection with the residual -> norm -> widening
    with GELU -> narrowing with the residual, forward and backward, against the same steps in
    torch on 64-bit values. Seven rounded steps forward and as many back of values of order one."""
    n, c, heads = 600, 64, 4
    coords = _voxels(n, 12, 1, 14)
    x = _tensor(coords)
    lut = position_buckets(3, 3, device=DEV)
    names = {"f": (n, c), "res": (n, c), "g1": (c,), "qkv": (3 * c, c), "o": (c, c), "ob": (c,),
             "g2": (c,), "up": (4 * c, c), "ub": (4 * c,), "down": (c, 4 * c),
             "table": (heads, 7, 7, 7)}
    p = {}
    for i, (name, shape) in enumerate(names.items()):
        scale = shape[-1] ** -0.5 if name in ("qkv", "o", "up", "down") else 1.0
        p[name] = _rand(shape, dtype, 100 + i, scale).requires_grad_(True)
    dout = _rand((n, c), dtype, 120)

    def block(p, norm, proj, attend):
        y, h = norm(p["f"], p["g1"], p["res"])
        qkv = proj(y, p["qkv"], None, None, None).view(n, 3, heads, c // heads)
        a = attend(*qkv.unbind(1), p["table"]).reshape(n, c)
        h = proj(a, p["o"], p["ob"], None, h)
        y, h = norm(h, p["g2"], None)
        u = proj(y, p["up"], p["ub"], "gelu_tanh", None)
        return proj(u, p["down"], None, None, h)

    def own_norm(f, g, r):
        out = rms_norm(f, g, residual=r)
        return out if r is not None else (out, f)

    got = block(p, own_norm,
                lambda a, w, b, act, r: linear(a, w, b, activation=act, residual=r),
                lambda q, k, v, t: sparse_self_attention(x, q, k, v, window_size=4,
                                                         position_bias=t, position_buckets=lut))
    grads = torch.autograd.grad(got, list(p.values()), dout)

    p64 = {m: t.detach().to(F64).requires_grad_(True) for m, t in p.items()}

    def ref_norm(f, g, r):
        h = f if r is None else f + r
        return h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * g, h

    def ref_proj(a, w, b, act, r):
        z = a @ w.T + (0 if b is None else b)
        z = torch.nn.functional.gelu(z, approximate="tanh") if act else z
        return z if r is None else z + r

    def ref_attend(q, k, v, t):
        d = coords[None, :, 1:].long() - coords[:, None, 1:].long()
        b = lut.long()[d.clamp(-3, 3) + 3]
        s = torch.einsum("ihd,jhd->hij", q, k) * q.shape[-1] ** -0.5
        s = s + t.flatten(1)[:, (b[..., 0] * 7 + b[..., 1]) * 7 + b[..., 2]]
        same = (coords[:, None, 1:] // 4 == coords[None, :, 1:] // 4).all(-1)
        s = s.masked_fill(~same, float("-inf"))
        return torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v)

    want = block(p64, ref_norm, ref_proj, ref_attend)
    wants = torch.autograd.grad(want, list(p64.values()), dout.to(F64))
    # fourteen roundings in the mean square, each at most eps / 2 of its value, with gains below
    # three along the way; fp32 as one of 2^-20 for its sums
    tol = 14**0.5 * 3 * max(_half(dtype), 2.0**-20)
    for name, a, b in zip(["out", *p], (got, *grads), (want, *wants)):
        rel = float((a.to(F64) - b).norm() / b.norm())
        assert rel <= tol, (name, rel, tol)
    N.check_device_status(DEV)


@pytest.mark.parametrize("window", [5, None])
def test_training_step_in_a_graph_and_on_two_streams(window):
    """Forward and backward of norm, projection and attention captured together (their workspaces come
    from the graph's pool), replayed on other inputs, and two eager steps at once on two streams."""
    coords = _voxels(1200, 12, 1, 15)
    x = _tensor(coords)
    lut = position_buckets(4, 2, device=DEV)
    dtype = torch.bfloat16

    def inputs(seed):
        shapes = [(1200, 64), (64,), (192, 64), (192,), (2, 5, 5, 5)]
        return [_rand(s, dtype, seed + i, 0.3) for i, s in enumerate(shapes)]

    dout = _rand((1200, 2, 32), dtype, 99)

    def step(args):
        f, w, p, b, table = args
        h = rms_norm(f, w)
        q, k, v = linear(h, p, b, activation="silu").view(1200, 3, 2, 32).unbind(1)
        out = sparse_self_attention(x, q, k, v, window_size=window, position_bias=table,
                                    position_buckets=lut)
        return [out.detach(), *torch.autograd.grad(out, args, dout)]

    def eager(seed):
        return step([t.requires_grad_(True) for t in inputs(seed)])

    want = {seed: eager(seed) for seed in (100, 200)}
    static = [t.requires_grad_(True) for t in inputs(100)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(static)
    for seed in (200, 100):
        with torch.no_grad():
            for t, new in zip(static, inputs(seed)):
                t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[seed]))
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for s, seed in zip(streams, (100, 200)):
        with torch.cuda.stream(s):
            results.append(eager(seed))
    torch.cuda.synchronize()
    for seed, res in zip((100, 200), results):
        assert all(torch.equal(a, b) for a, b in zip(res, want[seed]))
    N.check_device_status(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reach", [12, 31, 1023])
def test_largest_table_with_the_widest_heads(reach, dtype):
    """25 buckets an axis and 128 channels: the most shared memory that any call takes."""
    _run(_voxels(220, 10, 1, reach), 2, 128, dtype, 8, (4, 4, 4), reach, 12, seed=reach)
