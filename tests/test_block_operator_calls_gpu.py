"""How ``rms_norm``, ``linear`` and the biased attention may be called: autograd modes, coordinates that
change, streams and graphs that share a tensor's cache."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mlx_diffuser_b200 import SparseTensor, _native as N
from mlx_diffuser_b200 import linear, position_buckets, rms_norm, sparse_self_attention

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def _voxels(n, grid, seed):
    cells = np.random.default_rng(seed).choice(grid**3, n, replace=False)
    rows = np.stack([np.zeros(n, np.int64), *np.unravel_index(cells, (grid,) * 3)], 1)
    return torch.from_numpy(rows.astype(np.int32)).to(DEV)


def _tensor(coords):
    return SparseTensor(torch.zeros((len(coords), 1), device=DEV), coords)


def _attention(n=400, dtype=torch.bfloat16, seed=0):
    """A call of the biased attention on a tensor of n rows."""
    q, k, v = (_rand((n, 2, 32), dtype, seed + i) for i in range(3))
    table, lut = _rand((2, 9, 9, 9), dtype, seed + 3), position_buckets(4, 4, device=DEV)

    def run(x, window=5):
        return sparse_self_attention(x, q, k, v, window_size=window, position_bias=table,
                                     position_buckets=lut)

    return run


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_inference_mode(dtype):
    """Tensors made under inference mode have no version counter; inside and outside of it the operators
    give what they give elsewhere."""
    coords = _voxels(400, 12, 1)
    run = _attention(dtype=dtype)
    want = run(_tensor(coords))
    f, g, w = (_rand(s, dtype, 10 + i) for i, s in enumerate([(90, 64), (64,), (32, 64)]))
    want_y, want_z = rms_norm(f, g), linear(f, w, activation="silu")
    with torch.inference_mode():
        x = _tensor(coords.clone())
        assert x.coords.is_inference()
        first, again = run(x), run(x)
        assert torch.equal(first, want) and torch.equal(again, want)
        assert torch.equal(rms_norm(f.clone(), g), want_y)
        assert torch.equal(linear(f, w.clone(), activation="silu"), want_z)
        (q8, s8), h = rms_norm(f, g, residual=f.clone(), quantize=True)
    (q8_, s8_), h_ = rms_norm(f, g, residual=f, quantize=True)
    assert torch.equal(q8.view(torch.uint8), q8_.view(torch.uint8))
    assert torch.equal(s8, s8_) and torch.equal(h, h_)
    assert torch.equal(run(x), want)  # the tensor used after the mode has ended
    with torch.inference_mode():
        assert torch.equal(run(_tensor(coords)), want)  # an ordinary tensor inside it
    N.check_device_status(DEV)


def test_training_on_windows_laid_out_under_inference_mode():
    """A tensor whose first call was under inference mode is trained on later."""
    coords = _voxels(400, 12, 2)
    lut = position_buckets(4, 4, device=DEV)
    leaves = [_rand((400, 2, 32), torch.bfloat16, i).requires_grad_(True) for i in range(3)]
    leaves.append(_rand((2, 9, 9, 9), torch.bfloat16, 3).requires_grad_(True))
    dout = _rand((400, 2, 32), torch.bfloat16, 4)

    def step(x):
        out = sparse_self_attention(x, *leaves[:3], window_size=5, position_bias=leaves[3],
                                    position_buckets=lut)
        return (out, *torch.autograd.grad(out, leaves, dout))

    want = step(_tensor(coords))
    x = _tensor(coords)
    with torch.inference_mode():
        _attention()(x)
    assert all(torch.equal(a, b) for a, b in zip(step(x), want))


@pytest.mark.parametrize("window", [5, None])
def test_changed_coordinates(window):
    """Windows and biases belong to the coordinates that the tensor holds now: changed in place, or
    another tensor's beside the same cache."""
    coords = _voxels(400, 12, 3)
    other = _voxels(400, 12, 4)
    other[200:, 0] = 1
    run = _attention()
    want, want_other = run(_tensor(coords), window), run(_tensor(other), window)
    assert not torch.equal(want, want_other)
    x = _tensor(coords.clone())
    assert torch.equal(run(x, window), want)
    y = x.replace(x.features, other)  # shares the cache
    assert y.cache is x.cache
    assert torch.equal(run(y, window), want_other)
    assert torch.equal(run(x, window), want)
    x.coords.copy_(other)
    assert torch.equal(run(x, window), want_other)
    # the same windows without a bias
    q = _rand((400, 2, 32), torch.bfloat16, 50)
    z = _tensor(coords.clone())
    sparse_self_attention(z, q, q, q, window_size=window)
    z.coords.copy_(other)
    assert torch.equal(sparse_self_attention(z, q, q, q, window_size=window),
                       sparse_self_attention(_tensor(other), q, q, q, window_size=window))
    N.check_device_status(DEV)


def test_fewer_coordinates_than_features_are_refused():
    x = _tensor(_voxels(400, 12, 5))
    x.coords = x.coords[:300]
    with pytest.raises(ValueError, match="one row per feature row"):
        _attention()(x)


def test_plan_read_on_another_stream_is_not_handed_on():
    """A plan laid out on one stream and read on another, dropped while that one still works: its memory
    stays out of the first stream's reach until the reading is done."""
    coords = _voxels(3000, 16, 6)
    run = _attention(3000)
    x = _tensor(coords)
    want = run(x)
    plan = next(g for k, g in x.cache.items() if k.startswith("attention_groups_5")).plan
    address, size = plan.data_ptr(), plan.numel()
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # about a tenth of a second
        got = run(x)
    busy = not side.query()
    del plan, x
    taken = [torch.empty(size, dtype=torch.uint8, device=DEV) for _ in range(8)]
    still = busy and not side.query()
    inside = [t for t in taken if t.data_ptr() < address + size and address < t.data_ptr() + size]
    side.synchronize()
    assert still and not inside
    assert torch.equal(got, want)


def test_captured_call_and_changed_coordinates():
    """A graph that read the cached plan replays what it captured, though another has taken the plan's
    place since."""
    coords = _voxels(400, 12, 7)
    run = _attention()
    x = _tensor(coords.clone())
    want = run(x)
    N.status_word(DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = run(x)
    x.coords.copy_(_voxels(400, 12, 8))
    changed = run(x)
    assert torch.equal(changed, run(_tensor(x.coords))) and not torch.equal(changed, want)
    junk = [torch.full((1 << 16,), 255, dtype=torch.uint8, device=DEV) for _ in range(64)]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(inside, want)
    assert len(junk) == 64 and len(x.cache["attention_groups_captured"]) == 1


def test_eight_bit_rows_without_channels_have_scales():
    """A row of nothing is a row of zeros: its scale is 1, not what was in memory before."""
    for shape in ((5, 0), (3, 4, 0), (4096, 0)):
        x = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
        dirt = [torch.full(shape[:-1], float("nan"), device=DEV) for _ in range(4)]
        del dirt
        for r in (None, x):
            out = rms_norm(x, residual=r, quantize=True)
            q, s = out if r is None else out[0]
            assert q.shape == shape and s.shape == shape[:-1]
            assert torch.equal(s, torch.ones(shape[:-1], device=DEV))
    N.check_device_status(DEV)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_training_step_with_small_gradients_in_a_graph(dtype):
    """Norm, projection and attention, forward and backward, captured and replayed on other inputs whose
    gradients are 2^-10 of the captured ones: what fp16's gradients are raised by is found at replay."""
    coords = _voxels(900, 12, 9)
    x = _tensor(coords)
    lut = position_buckets(4, 4, device=DEV)
    shapes = [(900, 64), (64,), (192, 64), (192,), (2, 9, 9, 9)]

    def inputs(seed):
        return [_rand(s, dtype, seed + i, 0.3) for i, s in enumerate(shapes)]

    def step(args, dout):
        f, g, w, b, table = args
        q, k, v = linear(rms_norm(f, g), w, b, activation="gelu").view(900, 3, 2, 32).unbind(1)
        out = sparse_self_attention(x, q, k, v, window_size=5, position_bias=table,
                                    position_buckets=lut)
        return [out.detach(), *torch.autograd.grad(out, args, dout)]

    douts = {100: _rand((900, 2, 32), dtype, 98), 200: _rand((900, 2, 32), dtype, 99, 2.0**-10)}
    want = {}
    for seed, dout in douts.items():
        want[seed] = step([t.requires_grad_(True) for t in inputs(seed)], dout)
    static, sdout = [t.requires_grad_(True) for t in inputs(100)], douts[100].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static, sdout)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(static, sdout)
    for seed in (200, 100, 200):
        with torch.no_grad():
            for t, new in zip(static, inputs(seed)):
                t.copy_(new)
            sdout.copy_(douts[seed])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[seed]))
    N.check_device_status(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(300, 40, 24), (300, 41, 23), (5, 64, 24)], ids=str)
def test_some_of_the_projections_gradients(shape, dtype):
    """Any subset of the gradients is what all of them together are, with an activation and without,
    and through an output gradient off a 16-byte boundary."""
    m, k, n = shape
    x, w, b = _rand((m, k), dtype, 1), _rand((n, k), dtype, 2, 0.2), _rand((n,), dtype, 3)
    r = _rand((m, n), dtype, 4)
    odd = _rand((m * n + 1,), dtype, 5, 1e-3)[1:].view(m, n)
    for act in (None, "silu"):
        for dy in (odd, odd.clone()):
            want = None
            for wanted in range(15, 0, -1):
                leaves = [t.clone().requires_grad_(bool(wanted >> i & 1))
                          for i, t in enumerate((x, w, b, r))]
                y = linear(*leaves[:3], activation=act, residual=leaves[3])
                some = [t for t in leaves if t.requires_grad]
                got = iter(torch.autograd.grad(y, some, dy))
                got = [next(got) if t.requires_grad else None for t in leaves]
                want = got if want is None else want
                assert all(a is None or torch.equal(a, c) for a, c in zip(got, want))
    N.check_device_status(DEV)
