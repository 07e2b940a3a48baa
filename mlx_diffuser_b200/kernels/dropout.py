"""Dropout whose mask is never stored (``sv_dropout``): counter-based random numbers, formed again in the
backward pass."""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _native as N


def seed_argument(what: str, seed, subsequence: int, device: torch.device):
    """(seed, device tensor or None, subsequence) as the C entry points take them."""

    if not isinstance(subsequence, int) or not 0 <= subsequence < 2**64:
        raise ValueError(f"{what}: subsequence must be an int in [0, 2**64)")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError(f"{what}: a seed tensor holds one int64")
        if seed.device != device:
            raise ValueError(f"{what}: seed is on {seed.device}, x on {device}")
        return 0, seed, subsequence
    if isinstance(seed, bool) or not isinstance(seed, int) or not 0 <= seed < 2**64:
        raise ValueError(f"{what}: seed must be an int in [0, 2**64) or an int64 tensor")
    return seed, None, subsequence


def check_share(what: str, p) -> float:
    p = float(p)
    if not 0 <= p <= 1:
        raise ValueError(f"{what}: the dropped share must be in [0, 1], got {p}")
    return p


def _forward(x, residual, p, seed, seed_at, subsequence):
    out = torch.empty_like(x)
    dev = x.device
    rc = N.call(dev, N.load().sv_dropout, x.data_ptr(), N.ptr(residual), x.numel(),
                N.DTYPE_CODE[x.dtype], p, seed, N.ptr(seed_at), subsequence, out.data_ptr(),
                N.stream(dev))
    if rc:
        N.check(rc, "dropout")
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, seed_at, p, seed, subsequence):
        ctx.args = p, seed, subsequence
        ctx.save_for_backward(seed_at)  # changed before the backward pass: autograd raises
        return _forward(x, residual, p, seed, seed_at, subsequence)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        (seed_at,) = ctx.saved_tensors
        p, seed, subsequence = ctx.args
        dx = None
        if ctx.needs_input_grad[0]:
            dx = _forward(dout.contiguous(), None, p, seed, seed_at, subsequence)
        return dx, dout if ctx.needs_input_grad[1] else None, None, None, None, None


def dropout(
    x: torch.Tensor,
    p: float,
    seed: int | torch.Tensor,
    *,
    subsequence: int = 0,
    residual: torch.Tensor | None = None,
) -> torch.Tensor:
    """``x / (1 - p)`` where an element is kept and zero where it is dropped, plus ``residual``;
    float32, float16, bfloat16, one rounding.

    The share ``p`` is rounded to a multiple of 2^-16, and what is kept is divided by the share that is
    kept then. Which elements are dropped depends on ``seed``, ``subsequence`` and the element's number in
    row-major order only, and not on the type: the same call drops the same elements. Give every
    layer its own ``subsequence`` and every step its own ``seed``. A ``seed`` in device memory (one
    int64) can change between the replays of a captured graph; it has to keep its value until the
    backward pass has run.

    A dropped element is zero whatever it was. Gradients for ``x`` and ``residual``.
    """

    x = N.as_tensor(x)
    if x.dtype not in N.DTYPE_CODE:
        raise ValueError(f"dropout: unsupported dtype {x.dtype}")
    p = check_share("dropout", p)
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"dropout: residual must be a {tuple(x.shape)} {x.dtype} tensor, got "
                             f"{tuple(residual.shape)} {residual.dtype}")
        if residual.device != x.device:
            raise ValueError(f"dropout: residual is on {residual.device}, x on {x.device}")
    seed, seed_at, subsequence = seed_argument("dropout", seed, subsequence, x.device)
    N.refuse_tangents("dropout", x, residual)
    N.require_cuda(x, "x")
    x = x.contiguous()
    residual = None if residual is None else residual.contiguous()
    if torch.is_grad_enabled() and (
            x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, residual, N.savable(seed_at), p, seed, subsequence)
    return _forward(x, residual, p, seed, seed_at, subsequence)


__all__ = ["dropout"]
