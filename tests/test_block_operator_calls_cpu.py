"""Calls that ``rms_norm``, ``linear`` and the biased attention refuse before anything runs: no GPU."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

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
