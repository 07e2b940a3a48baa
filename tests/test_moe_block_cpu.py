"""What ``block_norm``, ``dropout``, ``route`` and ``expert_linear`` refuse, their random numbers and
packed arguments, and the C entry points' checks: no GPU."""

from __future__ import annotations

import ctypes
import dataclasses
import math

import numpy as np
import pytest
import torch

from mlx_diffuser_b200 import ExpertRoutes, _native as N
from mlx_diffuser_b200 import block_norm, dropout, expert_linear, route
from tests.philox import factors, numbers, philox


def test_random_numbers_are_philox():
    """The generator's published known answers, and how elements take their halves."""
    for counter, key, want in (
        ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
        ((2**32 - 1,) * 4, (2**32 - 1,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
        ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
         (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
    ):
        assert philox(np.array([counter], np.uint64), key)[0].tolist() == list(want)
    got = numbers(19, 0)
    words = philox(np.array([[i, 0, 0, 0] for i in range(3)], np.uint64), (0, 0)).reshape(-1)
    want = [int(w) >> s & 0xFFFF for w in words for s in (0, 16)]
    assert got.tolist() == want[:19]
    assert numbers(8, 7, 2**33 + 1, first=64).tolist() == numbers(72, 7, 2**33 + 1).tolist()[64:]
    f = factors(100000, 0.25, 3)
    assert set(np.unique(f)) == {0.0, 4 / 3}
    assert abs(f.mean() - 1) < 6 * math.sqrt(1 / 3 / 1e5)  # six standard deviations


def test_dropout_refusals():
    x = torch.zeros((4, 8))
    with pytest.raises(ValueError, match="unsupported dtype"):
        dropout(x.double(), 0.5, 1)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="share"):
            dropout(x, p, 1)
    for seed in (-1, 2**64, 1.5, None, True):
        with pytest.raises(ValueError, match="seed must be"):
            dropout(x, 0.5, seed)
    for seed in (torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="one int64"):
            dropout(x, 0.5, seed)
    with pytest.raises(ValueError, match="seed is on"):
        dropout(x, 0.5, torch.zeros(1, dtype=torch.int64, device="meta"))
    for s in (-1, 2**64, 1.0):
        with pytest.raises(ValueError, match="subsequence"):
            dropout(x, 0.5, 1, subsequence=s)
    for r in (x[:2], x.half()):
        with pytest.raises(ValueError, match="residual must be"):
            dropout(x, 0.5, 1, residual=r)
    with pytest.raises(ValueError, match="residual is on"):
        dropout(x, 0.5, 1, residual=torch.zeros((4, 8), device="meta"))
    with pytest.raises(RuntimeError, match="CUDA device"):
        dropout(x, 0.5, 1)


def test_block_norm_refusals():
    x = torch.zeros((6, 8))
    coords = torch.zeros((6, 4), dtype=torch.int32)
    rows, one = torch.zeros((3, 8)), torch.zeros(8)
    for bad in (x.double(), torch.tensor(1.0)):
        with pytest.raises(ValueError, match="unsupported input"):
            block_norm(bad, bad)
    with pytest.raises(ValueError, match="unknown norm"):
        block_norm(x, x, norm="batch")
    for bad in (x[:2], x.half(), x[:, :4]):
        with pytest.raises(ValueError, match="branch must be"):
            block_norm(x, bad)
    for name in ("weight", "bias"):
        for bad in (torch.zeros(7), torch.zeros(8, dtype=torch.int32), torch.zeros((1, 8)), one.double()):
            with pytest.raises(ValueError, match=f"{name} must be"):
                block_norm(x, x, **{name: bad})
    with pytest.raises(ValueError, match="branch_weight goes with"):
        block_norm(x, x, branch_weight=one)
    with pytest.raises(ValueError, match="branch_weight must be"):
        block_norm(x, x, branch_norm=True, branch_weight=torch.zeros(7))
    for name in ("gate", "scale", "shift"):
        for bad in (torch.zeros((3, 7)), torch.zeros((1, 1, 8)), torch.zeros(()), rows.long(), rows[:0]):
            with pytest.raises(ValueError, match=f"{name} must be"):
                block_norm(x, x, **{name: bad})
    with pytest.raises(ValueError, match="need the coordinates"):
        block_norm(x, x, gate=rows)
    for bad in (coords[:5], coords.long(), coords[:, :3]):
        with pytest.raises(ValueError, match="coords must be"):
            block_norm(x, x, gate=rows, coords=bad)
    with pytest.raises(ValueError, match="rows of coefficients for batch 2"):
        block_norm(x, x, gate=rows, coords=coords, batch_size=2)
    with pytest.raises(ValueError, match="2 rows, others 3"):
        block_norm(x, x, gate=rows, scale=rows[:2], coords=coords)
    for eps in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            block_norm(x, x, eps=eps)
    with pytest.raises(ValueError, match="share"):
        block_norm(x, x, dropout=1.5, seed=1)
    with pytest.raises(ValueError, match="needs a seed"):
        block_norm(x, x, dropout=0.5)
    with pytest.raises(ValueError, match="seed must be"):
        block_norm(x, x, dropout=0.5, seed=-1)
    meta = torch.zeros(8, device="meta")
    with pytest.raises(ValueError, match="weight is on"):
        block_norm(x, x, weight=meta)
    with pytest.raises(ValueError, match="coords is on"):
        block_norm(x, x, gate=rows, coords=coords.to("meta"))
    with pytest.raises(ValueError, match="branch is on"):
        block_norm(x, x.to("meta"))
    with pytest.raises(RuntimeError, match="CUDA device"):
        block_norm(x, x, gate=rows, coords=coords)


def test_route_refusals():
    x = torch.zeros((5, 8))
    for bad in (torch.zeros(8), torch.zeros((1, 5, 8)), x.double(), x.long()):
        with pytest.raises(ValueError, match="logits must be"):
            route(bad, 1)
    for bad in (x[:, :0], torch.zeros((2, 1025))):
        with pytest.raises(ValueError, match="experts"):
            route(bad, 1)
    for k in (0, 9, -1):
        with pytest.raises(ValueError, match="choices"):
            route(x, k)
    with pytest.raises(ValueError, match="1 to 32 choices"):
        route(torch.zeros((2, 64)), 33)
    with pytest.raises(RuntimeError, match="CUDA device"):
        route(x, 2)


def _routes(n=6, k=2, e=4):
    i32 = torch.int32
    return ExpertRoutes(torch.zeros((n, k), dtype=i32), torch.zeros((n, k)), torch.zeros(n * k, dtype=i32),
                        torch.zeros(e + 1, dtype=i32), torch.zeros((n, k), dtype=i32))


def test_expert_linear_refusals():
    r = _routes()
    assert (r.rows, r.choices, r.num_experts) == (6, 2, 4)
    x, xs, w, b = torch.zeros((6, 8)), torch.zeros((12, 8)), torch.zeros((4, 10, 8)), torch.zeros((4, 10))
    with pytest.raises(ValueError, match="unknown activation"):
        expert_linear(x, w, r, activation="relu", gather=True)
    with pytest.raises(ValueError, match="ExpertRoutes"):
        expert_linear(x, w, None, gather=True)
    for bx, bw in ((x[0], w), (x, w[0]), (x, torch.zeros((4, 10, 7)))):
        with pytest.raises(ValueError, match="x must have shape"):
            expert_linear(bx, bw, r, gather=True)
    with pytest.raises(ValueError, match="unsupported dtype"):
        expert_linear(x.double(), w.double(), r, gather=True)
    with pytest.raises(ValueError, match="routes ask for 6"):
        expert_linear(xs, w, r, gather=True)
    with pytest.raises(ValueError, match="routes ask for 12"):
        expert_linear(x, w, r)
    with pytest.raises(ValueError, match="3 experts, the routes 4"):
        expert_linear(x, w[:3], r, gather=True)
    with pytest.raises(ValueError, match="weight must be"):
        expert_linear(x, w.half(), r, gather=True)
    for bad in (torch.zeros(10), torch.zeros((4, 8)), b.half()):
        with pytest.raises(ValueError, match="bias must be"):
            expert_linear(x, w, r, bad, gather=True)
    for name, bad in (("weights", r.weights.half()), ("order", r.order[:5]), ("order", r.order.long()),
                      ("offsets", r.offsets.long()), ("place", r.place[:, :1])):
        with pytest.raises(ValueError, match=f"routes.{name} must be"):
            expert_linear(x, w, dataclasses.replace(r, **{name: bad}), gather=True)
    with pytest.raises(ValueError, match="bias is on"):
        expert_linear(x, w, r, b.to("meta"), gather=True)
    with pytest.raises(RuntimeError, match="CUDA device"):
        expert_linear(x, w, r, b, gather=True)


class _Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("stride", ctypes.c_int64), ("dtype", ctypes.c_int)]


class _BlockNormArgs(ctypes.Structure):
    _fields_ = [
        ("n", ctypes.c_int64), ("batch", ctypes.c_int64), ("x", ctypes.c_void_p),
        ("x_stride", ctypes.c_int64), ("branch", ctypes.c_void_p), ("branch_stride", ctypes.c_int64),
        ("h", ctypes.c_void_p), ("stats", ctypes.c_void_p), ("coords", ctypes.c_void_p),
        *((name, _Rows) for name in ("weight", "bias", "branch_weight", "gate", "scale", "shift")),
        ("dropout", ctypes.c_double), ("seed", ctypes.c_uint64), ("seed_at", ctypes.c_void_p),
        ("subsequence", ctypes.c_uint64), ("channels", ctypes.c_int), ("dtype", ctypes.c_int),
        ("layer", ctypes.c_int), ("branch_norm", ctypes.c_int), ("residual_scale", ctypes.c_float),
        ("eps", ctypes.c_float)]


class _ExpertArgs(ctypes.Structure):
    _fields_ = [
        ("n", ctypes.c_int64), ("x", ctypes.c_void_p), ("ldx", ctypes.c_int64),
        ("weight", ctypes.c_void_p), ("ldw", ctypes.c_int64), ("w_expert", ctypes.c_int64),
        *((name, ctypes.c_void_p)
          for name in ("bias", "order", "offsets", "place", "weights", "preact", "rows")),
        ("inputs", ctypes.c_int64), ("outputs", ctypes.c_int64),
        *((name, ctypes.c_int)
          for name in ("k", "experts", "dtype", "activation", "gather", "combine"))]


def test_packed_arguments_are_the_headers_structures():
    values = [7, 3, 11, 12, 13, 14, 15, 16, 17]
    rows = [100 * (i + 1) + j for i in range(6) for j in range(3)]
    tail = [0.25, 2**63 + 5, 18, 2**40, 64, 2, 1, 0, 0.5, 2.0**-20]
    a = _BlockNormArgs.from_buffer_copy(N.BLOCK_NORM_ARGS.pack(*values, *rows, *tail))
    assert ctypes.sizeof(_BlockNormArgs) == N.BLOCK_NORM_ARGS.size
    assert [getattr(a, f) for f, _ in _BlockNormArgs._fields_[:9]] == values
    got = [getattr(getattr(a, f), g) for f, _ in _BlockNormArgs._fields_[9:15] for g in ("data", "stride", "dtype")]
    assert got == rows
    assert [getattr(a, f) for f, _ in _BlockNormArgs._fields_[15:]] == tail
    assert N.BLOCK_NORM_GRADS.size == 6 * ctypes.sizeof(_Rows)
    values = list(range(1, 22))
    e = _ExpertArgs.from_buffer_copy(N.EXPERT_ARGS.pack(*values))
    assert ctypes.sizeof(_ExpertArgs) == N.EXPERT_ARGS.size
    assert [getattr(e, f) for f, _ in _ExpertArgs._fields_] == values


def _block_args(**kw):
    base = dict(n=4, batch=2, x=0, x_stride=8, branch=0, branch_stride=8, h=0, stats=0, coords=0,
                rows=[0, 0, 0] * 6, dropout=0.0, seed=0, seed_at=0, subsequence=0, channels=8, dtype=0,
                layer=1, branch_norm=0, residual_scale=1.0, eps=1e-6)
    base.update(kw)
    return N.BLOCK_NORM_ARGS.pack(*(v for name, value in base.items()
                                    for v in (value if name == "rows" else [value])))


def _expert_args(**kw):
    base = dict(n=4, x=0, ldx=8, weight=0, ldw=8, w_expert=64, bias=0, order=0, offsets=0, place=0,
                weights=0, preact=0, rows=0, inputs=8, outputs=8, k=2, experts=4, dtype=2, activation=0,
                gather=0, combine=0)
    base.update(kw)
    return N.EXPERT_ARGS.pack(*base.values())


def test_c_entry_points_check_before_any_launch():
    lib = N.load()

    def norm(**kw):
        return lib.sv_block_norm(_block_args(**kw), None, None, None)

    assert norm() == N.SV_ERR_INVALID_ARGUMENT  # null pointers
    assert norm(n=0) == N.SV_OK and norm(channels=0) == N.SV_OK
    assert norm(n=-1) == N.SV_ERR_INVALID_ARGUMENT
    assert norm(dtype=3) == N.SV_ERR_BAD_DTYPE
    assert norm(channels=8193) == N.SV_ERR_UNSUPPORTED
    assert norm(dropout=1.5) == N.SV_ERR_INVALID_ARGUMENT
    assert norm(eps=-1.0) == N.SV_ERR_INVALID_ARGUMENT
    gate = [0] * 9 + [4096, 8, 0] + [0] * 6
    assert norm(rows=gate) == N.SV_ERR_INVALID_ARGUMENT  # rows per batch element without coords
    assert norm(rows=gate, coords=4096, batch=4096) == N.SV_ERR_UNSUPPORTED
    assert norm(rows=[0] * 9 + [4096, 8, 7] + [0] * 6, coords=4096) == N.SV_ERR_BAD_DTYPE
    assert norm(rows=[0] * 6 + [4096, 0, 0] + [0] * 9) == N.SV_ERR_INVALID_ARGUMENT  # branch_weight alone
    assert lib.sv_block_norm(None, None, None, None) == N.SV_ERR_INVALID_ARGUMENT
    grads = N.BLOCK_NORM_GRADS.pack(*[0] * 18)
    assert lib.sv_block_norm_backward(_block_args(), None, None, None, None, grads, None, 0, None,
                                      None) == N.SV_OK  # nothing is wanted
    wanted = N.BLOCK_NORM_GRADS.pack(*([4096, 0, 0] + [0] * 15))
    assert lib.sv_block_norm_backward(_block_args(), None, None, None, None, wanted, None, 0, None,
                                      None) == N.SV_ERR_INVALID_ARGUMENT  # dweight without a weight
    assert lib.sv_block_norm_backward_workspace_bytes(1000, 64, 5) > 1000 * 4
    assert lib.sv_block_norm_backward_workspace_bytes(-1, 64, 5) == 0

    def drop(cells=8, dtype=0, p=0.5):
        return lib.sv_dropout(None, None, cells, dtype, p, 1, None, 0, None, None)

    assert drop() == N.SV_ERR_INVALID_ARGUMENT and drop(cells=0) == N.SV_OK
    assert drop(cells=-1) == N.SV_ERR_INVALID_ARGUMENT and drop(dtype=3) == N.SV_ERR_BAD_DTYPE
    for p in (-0.5, 2.0, float("nan")):
        assert drop(p=p) == N.SV_ERR_INVALID_ARGUMENT

    def routed(n=4, e=8, k=2, dtype=0, stride=8):
        return lib.sv_route(None, stride, n, e, k, dtype, 1, None, None, None, None, None, None, 0, None)

    assert routed() == N.SV_ERR_INVALID_ARGUMENT
    assert routed(dtype=9) == N.SV_ERR_BAD_DTYPE and routed(k=9) == N.SV_ERR_BAD_SHAPE
    assert routed(e=1025) == N.SV_ERR_UNSUPPORTED and routed(n=-1) == N.SV_ERR_INVALID_ARGUMENT
    assert routed(e=64, k=33) == N.SV_ERR_UNSUPPORTED
    assert routed(n=2**31, k=1) == N.SV_ERR_UNSUPPORTED
    assert lib.sv_route_workspace_bytes(8, 16, 2) == 0  # one block does it all
    assert lib.sv_route_workspace_bytes(40000, 16, 2) > 0

    def expert(**kw):
        return lib.sv_expert_linear(_expert_args(**kw), None, None, 0, None, None)

    assert expert() == N.SV_ERR_INVALID_ARGUMENT
    assert expert(n=0) == N.SV_OK and expert(outputs=0) == N.SV_OK
    assert expert(dtype=3) == N.SV_ERR_BAD_DTYPE and expert(activation=9) == N.SV_ERR_INVALID_ARGUMENT
    assert expert(experts=1025) == N.SV_ERR_UNSUPPORTED and expert(ldx=7) == N.SV_ERR_INVALID_ARGUMENT
    assert expert(n=2**31) == N.SV_ERR_UNSUPPORTED
    assert expert(k=0) == N.SV_ERR_INVALID_ARGUMENT
    size = lib.sv_expert_linear_workspace_bytes
    few, many = _expert_args(gather=1), _expert_args(gather=1, n=100)
    assert size(few, N.SV_LINEAR_FORWARD, 0, 0, None) == 0
    assert size(many, N.SV_LINEAR_FORWARD, 0, 0, None) >= 200 * 8 * 2  # the gathered rows
    assert size(many, N.SV_LINEAR_BACKWARD, 1, 1, None) > size(many, N.SV_LINEAR_BACKWARD, 0, 0, None)
    assert lib.sv_expert_linear_backward(few, None, None, None, None, None, None, 0, None,
                                         None) == N.SV_OK  # nothing is wanted
    assert lib.sv_expert_linear_backward(few, None, None, 4096, None, None, None, 0, None,
                                         None) == N.SV_ERR_INVALID_ARGUMENT


def test_forward_mode_tangents_are_refused():
    x, r = torch.zeros((6, 8)), _routes()
    w = torch.zeros((4, 10, 8))
    with torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: dropout(d, 0.5, 1), lambda: block_norm(d, x), lambda: route(d, 2),
                     lambda: expert_linear(d, w, r, gather=True)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_experts_epilogue_warps_meet_their_barrier_equally_often():
    """The epilogue warps meet at ex_epi_sync() once a tile. A warp whose wait has run out must not leave the
    loop over the tiles before the others, nor skip to the next tile ahead of the barrier."""
    from tests.test_kernel_waits_cpu import CSRC, _block

    with open(f"{CSRC}/expert_tc.cu") as f:
        text = f.read()
    text = text[text.index("expert_tc_kernel(const __grid_constant__") :]
    assert text.count("ex_epi_sync();") == 1
    at = text.rindex("for (int32_t t = unit", 0, text.index("ex_epi_sync();"))
    loop = _block(text, at)
    head, tail = loop.split("ex_epi_sync();")
    assert "break" not in loop and "return" not in loop and "goto" not in loop
    assert "continue" not in head
    assert tail.index("if (!ok) continue;") < tail.index("mbar_wait_bounded")
    assert "mbar_try_wait" not in loop


class _Recorder:
    """Stands for the library: keeps the packed arguments and launches nothing."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if name.endswith("_bytes"):
            return lambda *args: 256

        def entry(*args):
            self.calls.append((name, args))
            return N.SV_OK

        return entry


def test_block_norm_backward_reads_the_tensors_that_autograd_hands_it(monkeypatch):
    """Saved tensors that come back as others (a checkpoint's recomputation, copies on the host) lie at other
    addresses with other strides than those of the forward call, whose memory may be gone."""
    lib = _Recorder()
    monkeypatch.setattr(N, "load", lambda: lib)
    monkeypatch.setattr(N, "require_cuda", lambda t, name: None)
    monkeypatch.setattr(N, "call", lambda device, fn, *args: fn(*args))
    monkeypatch.setattr(N, "stream", lambda device: 0)
    monkeypatch.setattr(N, "status_word", lambda device: torch.zeros(1, dtype=torch.int32))
    back = []

    def unpack(t):  # another tensor, dense
        back.append(t.clone(memory_format=torch.contiguous_format))
        return back[-1]

    n, c = 6, 8
    wide = torch.randn((n, 24))
    six = torch.randn((3, 6 * c))
    leaves = {"x": torch.randn((n, c)), "branch": wide[:, 8:16], "weight": torch.randn(c),
              "bias": torch.randn(2 * c)[::2], "branch_weight": torch.randn(c), "gate": six[:, :c],
              "scale": six[:, c:2 * c], "shift": torch.randn((1, c))}
    leaves = {k: t.requires_grad_(True) for k, t in leaves.items()}
    coords = torch.zeros((n, 4), dtype=torch.int32)
    seed = torch.ones(1, dtype=torch.int64)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y, h = block_norm(**leaves, branch_norm=True, coords=coords, batch_size=3, dropout=0.5, seed=seed)
    torch.autograd.grad((y, h), list(leaves.values()), (torch.ones_like(y), torch.ones_like(h)))
    (first, forward), (second, backward) = lib.calls
    assert (first, second) == ("sv_block_norm", "sv_block_norm_backward")
    a = _BlockNormArgs.from_buffer_copy(forward[0])
    assert (a.branch, a.branch_stride) == (leaves["branch"].data_ptr(), 24)
    assert (a.gate.data, a.gate.stride) == (leaves["gate"].data_ptr(), 6 * c)
    b = _BlockNormArgs.from_buffer_copy(backward[0])
    held = {t.data_ptr(): t for t in back}
    for name in ("branch", "h", "stats", "coords", "seed_at"):
        assert getattr(b, name) in held, name
    assert b.branch_stride == c
    for name in ("weight", "bias", "branch_weight", "gate", "scale", "shift"):
        row = getattr(b, name)
        assert row.data in held and held[row.data].shape == leaves[name].shape, name
        assert row.stride == (c if name in ("gate", "scale") else 0), name


def test_routing_weights_that_are_not_read_get_no_gradient(monkeypatch):
    """Without the weighted sum the result does not depend on them: no zeros go back through the router."""
    lib = _Recorder()
    monkeypatch.setattr(N, "load", lambda: lib)
    monkeypatch.setattr(N, "require_cuda", lambda t, name: None)
    monkeypatch.setattr(N, "call", lambda device, fn, *args: fn(*args))
    monkeypatch.setattr(N, "stream", lambda device: 0)
    monkeypatch.setattr(N, "status_word", lambda device: torch.zeros(1, dtype=torch.int32))
    r, x = _routes(), torch.randn((6, 8), requires_grad=True)
    p = torch.rand((6, 2), requires_grad=True)
    w = torch.randn((4, 10, 8), requires_grad=True)
    for combine in (False, True):
        y = expert_linear(x, w, dataclasses.replace(r, weights=p * 1), gather=True, combine=combine)
        lib.calls.clear()
        dx, dw, dp = torch.autograd.grad(y, (x, w, p), torch.ones_like(y), allow_unused=True)
        assert dx.shape == x.shape and dw.shape == w.shape
        assert (dp is not None) == combine
        ((name, args),) = lib.calls
        assert name == "sv_expert_linear_backward" and (args[5] is not None) == combine
    y = expert_linear(x.detach(), w.detach(), dataclasses.replace(r, weights=p), gather=True)
    assert not y.requires_grad


def test_status_word_made_under_inference_mode(monkeypatch):
    """A process whose first call is under inference mode reads and clears the word outside of it."""
    zeros, cuda = torch.zeros, torch.device("cuda", 0)
    monkeypatch.setattr(torch, "zeros", lambda *args, device=None, **kw: zeros(*args, **kw))
    monkeypatch.setattr(N, "_status", {})
    with torch.inference_mode():
        word = N.status_word(cuda)
    assert not word.is_inference()
    word.fill_(N.SV_DEVICE_BAD_INDEX)
    with pytest.raises(RuntimeError, match="out of range"):
        N.check_device_status(cuda)
    N.check_device_status(cuda)
