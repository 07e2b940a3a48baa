"""Calls that ``rms_norm``, ``linear`` and the biased attention refuse before anything runs, and what their
bindings hold on to: no GPU."""

from __future__ import annotations

import weakref

import pytest
import torch
from torch.autograd import forward_ad

from mlx_diffuser_b200 import _native as N
from mlx_diffuser_b200 import (
    SparseTensor,
    linear,
    position_buckets,
    rms_norm,
    sparse_self_attention,
)


def test_forward_mode_derivatives_are_refused():
    """A tangent on any input, with and without a gradient wanted: never dropped in silence."""
    coords = torch.zeros((5, 4), dtype=torch.int32)
    x = SparseTensor(torch.zeros((5, 1)), coords)
    lut = position_buckets(1, 1)
    norm = [torch.zeros((4, 8)), torch.zeros((4, 8)), torch.ones(8)]
    proj = [torch.zeros((4, 8)), torch.zeros((6, 8)), torch.zeros(6), torch.zeros((4, 6))]
    attn = [torch.zeros((5, 2, 16)) for _ in range(3)] + [torch.zeros((2, 3, 3, 3))]
    calls = (
        (norm, lambda a, r, w: rms_norm(a, w, residual=r)),
        (proj, lambda a, w, b, r: linear(a, w, b, activation="silu", residual=r)),
        (attn, lambda q, k, v, t: sparse_self_attention(x, q, k, v, position_bias=t,
                                                        position_buckets=lut)),
    )
    for args, call in calls:
        for i in range(len(args)):
            for grad in (False, True):
                with forward_ad.dual_level():
                    some = [t.clone().requires_grad_(grad) for t in args]
                    some[i] = forward_ad.make_dual(some[i], torch.ones_like(some[i]))
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        call(*some)
        # a level without tangents is an ordinary call
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="CUDA device"):
            call(*args)
    with forward_ad.dual_level():
        a = forward_ad.make_dual(norm[0], torch.ones_like(norm[0]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            rms_norm(a, quantize=True)


class _Library:
    """In the library's place: sizes are 4096, and every other call finds its workspaces alive."""

    def __init__(self):
        self.held = []
        self.calls = []

    def __getattr__(self, name):
        if not name.startswith("sv_"):
            raise AttributeError(name)
        if name.endswith("_bytes"):
            return lambda *a: 4096

        def call(*args):
            self.calls.append(name)
            assert all(r() is not None for r in self.held), f"{name}: a workspace is gone"
            self.held.clear()
            return N.SV_OK

        return call


def test_workspaces_live_until_their_call_returns(monkeypatch):
    """The library is called without the interpreter's lock: memory that is dropped before the call goes to
    whatever another thread launches on the same stream in the meantime."""
    lib = _Library()

    def workspace(nbytes, device):
        t = torch.empty(nbytes, dtype=torch.uint8)
        lib.held.append(weakref.ref(t))
        return t

    monkeypatch.setattr(N, "load", lambda: lib)
    monkeypatch.setattr(N, "workspace", workspace)
    monkeypatch.setattr(N, "require_cuda", lambda *a: None)
    monkeypatch.setattr(N, "status_word", lambda device: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(N, "stream", lambda device: 0)
    x, w, b = (torch.zeros(s, requires_grad=True) for s in ((20, 8), (6, 8), (6,)))
    linear(x, w, b, activation="gelu").sum().backward()
    rms_norm(x, w[0].detach().requires_grad_(True)).sum().backward()
    from mlx_diffuser_b200.kernels.attention import biased_window_attention

    q, k, v = (torch.zeros((5, 2, 8), requires_grad=True) for _ in range(3))
    table = torch.zeros((2, 3, 3, 3), requires_grad=True)
    plan = torch.zeros(4096, dtype=torch.uint8)
    biased_window_attention(q, k, v, table, position_buckets(1, 1), plan, 1, 0.5).sum().backward()
    assert lib.calls == ["sv_linear_forward", "sv_linear_backward", "sv_rms_norm",
                         "sv_rms_norm_backward", "sv_window_attention",
                         "sv_window_attention_backward"]
