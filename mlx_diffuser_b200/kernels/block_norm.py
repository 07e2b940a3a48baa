"""The border between two blocks of a transformer in one pass (``sv_block_norm``): dropout and norm of a
block's result, gate, residual scale and addition, then the next block's norm with its modulation
(``src/mlx_diffuser/models/trellis_slat.py:77-80`` modulates the same way), with gradients."""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from .. import _native as N
from .dropout import check_share, seed_argument
from .norm import _rows

_NONE = (0, 0, 0)  # an sv_rows without data


def _row(t: torch.Tensor) -> tuple[int, int, int]:
    """``t`` (C,), (1, C) or (B, C), rows contiguous, as an sv_rows."""

    per_batch = t.ndim == 2 and t.shape[0] > 1
    return t.data_ptr(), t.stride(0) if per_batch else 0, N.DTYPE_CODE[t.dtype]


def _laid_out(t: torch.Tensor, c: int) -> torch.Tensor:
    """Coefficients as ``_row`` takes them: contiguous rows that do not overlap."""

    if t.is_contiguous() or (
            (t.stride(-1) == 1 or c <= 1) and (t.ndim == 1 or t.stride(0) >= c)):
        return t
    return t.contiguous()


class _Call:
    """What both passes hand to the library beside their tensors. No address and no stride: the tensors that
    autograd hands to the backward pass may be others than those it was given (recomputed by a checkpoint,
    or brought back from the host)."""

    __slots__ = ("n", "c", "code", "batch", "per_batch", "p", "seed", "subsequence", "layer",
                 "branch_norm", "residual_scale", "eps")

    def pack(self, x, x_stride, branch, h, stats, coords, rows, seed_at) -> bytes:
        return N.BLOCK_NORM_ARGS.pack(
            self.n, self.batch, x, x_stride, branch.data_ptr(), max(branch.stride(0), self.c),
            h.data_ptr(),
            0 if stats is None else stats.data_ptr(), 0 if coords is None else coords.data_ptr(),
            *rows, self.p, self.seed, 0 if seed_at is None else seed_at.data_ptr(),
            self.subsequence, self.c, self.code, self.layer, self.branch_norm,
            self.residual_scale, self.eps)


def _forward(x, branch, coords, seed_at, o, rows, keep):
    n, c, dev = o.n, o.c, x.device
    h, y = x.new_empty((n, c)), x.new_empty((n, c))
    stats = torch.empty((n, 4), dtype=torch.float32, device=dev) if keep else None
    args = o.pack(x.data_ptr(), max(x.stride(0), c), branch, h, stats, coords, rows, seed_at)
    rc = N.call(dev, N.load().sv_block_norm, args, y.data_ptr(), N.status_word(dev).data_ptr(),
                N.stream(dev))
    if rc:
        N.check(rc, "block_norm")
    return y, h, stats


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, coords, seed_at, o, rows, *coefs):
        y, h, stats = _forward(x, branch, coords, seed_at, o, rows, True)
        ctx.save_for_backward(branch, h, stats, coords, seed_at, *coefs)
        ctx.options = o
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        branch, h, stats, coords, seed_at, *coefs = ctx.saved_tensors
        need_x, need_branch, _, _, _, _, *need = ctx.needs_input_grad
        if dy is None and dh is None:
            return (None,) * (6 + len(need))
        o, dev = ctx.options, h.device
        h, stats = h.contiguous(), stats.contiguous()
        coords = None if coords is None else coords.contiguous()
        if o.c:
            branch = _rows(branch, o.c)
        rows = []
        coefs = [None if t is None else _laid_out(t, o.c) for t in coefs]
        for t in coefs:
            rows += _NONE if t is None else _row(t)
        dy = None if dy is None else dy.contiguous()
        dh = None if dh is None else dh.contiguous()
        dx = torch.empty_like(h) if need_x else None
        dbranch = torch.empty_like(h) if need_branch else None
        grads = [torch.empty(t.shape, dtype=t.dtype, device=dev) if want else None
                 for t, want in zip(coefs, need)]
        wanted = []
        for t in grads:
            wanted += _NONE if t is None else _row(t)
        lib = N.load()
        nbytes, ws = 0, None
        if o.per_batch or any(need):
            nbytes = lib.sv_block_norm_backward_workspace_bytes(o.n, o.c, o.batch if o.per_batch else 0)
            ws = N.workspace(nbytes, dev)
        rc = N.call(dev, lib.sv_block_norm_backward, o.pack(0, 0, branch, h, stats, coords, rows, seed_at),
                    N.ptr(dy), N.ptr(dh), N.ptr(dx), N.ptr(dbranch), N.BLOCK_NORM_GRADS.pack(*wanted),
                    N.ptr(ws), nbytes, N.status_word(dev).data_ptr(), N.stream(dev))
        if rc:
            N.check(rc, "block_norm (backward)")
        return dx, dbranch, None, None, None, None, *grads


def block_norm(
    x: torch.Tensor,
    branch: torch.Tensor,
    *,
    norm: str = "layer",
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    scale: torch.Tensor | None = None,
    shift: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    residual_scale: float = 1.0,
    branch_norm: bool = False,
    branch_weight: torch.Tensor | None = None,
    coords: torch.Tensor | None = None,
    batch_size: int | None = None,
    dropout: float = 0.0,
    seed: int | torch.Tensor | None = None,
    subsequence: int = 0,
    eps: float = 1e-6,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(y, h)`` over the last axis of ``x``, fp32 inside::

        d = dropout(branch)
        u = N(d) * branch_weight            # with branch_norm; d itself without it
        h = x + residual_scale * gate[b] * u
        y = (N(h) * weight + bias) * (1 + scale[b]) + shift[b]

    ``h`` is the residual stream that goes on to the next border, rounded to ``x.dtype`` before it is
    normed; ``y`` is what the next block reads. ``N`` is the layer norm (``norm="layer"``) or the
    root-mean-square norm (``"rms"``), both with ``eps``.

    ``x`` and ``branch``: (..., C), alike, float32, float16 or bfloat16, C up to 8192. ``weight``,
    ``bias``, ``branch_weight``: (C,). ``gate``, ``scale``, ``shift``: (B, C) with the row picked by
    ``coords[:, 0]`` of the (rows, 4) int32 coordinates, or (C,) / (1, C) for every row; any of the
    three float types. A row whose batch index is outside ``batch_size`` (by default the largest B, at most
    4095) is left without gate, scale and shift, and :func:`check_device_status` reports it.
    ``dropout``, ``seed`` and ``subsequence`` are those of :func:`~mlx_diffuser_b200.dropout`.

    Gradients for everything but the coordinates and the seed, in fixed orders of summation.
    """

    x, branch = N.as_tensor(x), N.as_tensor(branch)
    shape, dtype, dev = x.shape, x.dtype, x.device
    if not shape or dtype not in N.DTYPE_CODE:
        raise ValueError(f"block_norm: unsupported input, shape {tuple(shape)}, dtype {dtype}")
    if norm not in ("layer", "rms"):
        raise ValueError(f"block_norm: unknown norm {norm!r}")
    c = shape[-1]
    rows = shape[0] if len(shape) == 2 else math.prod(shape[:-1])
    if branch.shape != shape or branch.dtype != dtype:
        raise ValueError(f"block_norm: branch must be a {tuple(shape)} {dtype} tensor, got "
                         f"{tuple(branch.shape)} {branch.dtype}")
    if branch_weight is not None and not branch_norm:
        raise ValueError("block_norm: branch_weight goes with branch_norm")
    grads = torch.is_grad_enabled()
    some = grads and (x.requires_grad or branch.requires_grad)
    o = _Call()
    packed, coefs, largest = [], [], 1
    for name, t, rank in (("weight", weight, 1), ("bias", bias, 1),
                          ("branch_weight", branch_weight, 1), ("gate", gate, 2),
                          ("scale", scale, 2), ("shift", shift, 2)):
        if t is None:
            packed += _NONE
            coefs.append(None)
            continue
        size = t.shape
        if not 1 <= len(size) <= rank or size[-1] != c or t.dtype not in N.DTYPE_CODE or \
                (len(size) == 2 and size[0] < 1):
            raise ValueError(f"block_norm: {name} must be a float tensor of shape "
                             + (f"(B, {c})" if rank == 2 else f"({c},)"))
        if t.device != dev:
            raise ValueError(f"block_norm: {name} is on {t.device}, x on {dev}")
        if len(size) == 2 and size[0] != 1:
            if largest not in (1, size[0]):
                raise ValueError(f"block_norm: {name} has {size[0]} rows, others {largest}")
            largest = size[0]
        t = _laid_out(t, c)
        some = some or (grads and t.requires_grad)
        coefs.append(t)
        packed += _row(t)
    batch = largest if batch_size is None else int(batch_size)
    if largest not in (1, batch):
        raise ValueError(f"block_norm: {largest} rows of coefficients for batch {batch}")
    if largest != 1:
        if coords is None:
            raise ValueError("block_norm: rows per batch element need the coordinates")
        if coords.shape != (rows, 4) or coords.dtype != torch.int32:
            raise ValueError(f"block_norm: coords must be an int32 tensor of shape ({rows}, 4)")
        if coords.device != dev:
            raise ValueError(f"block_norm: coords is on {coords.device}, x on {dev}")
        coords = coords.contiguous()
    else:
        coords = None
    if branch.device != dev:
        raise ValueError(f"block_norm: branch is on {branch.device}, x on {dev}")
    if not eps >= 0:
        raise ValueError("block_norm: eps must not be negative")
    p, seed_value, seed_at = 0.0, 0, None
    if dropout != 0:
        p = check_share("block_norm", dropout)
        if seed is None:
            raise ValueError("block_norm: dropout needs a seed")
        seed_value, seed_at, subsequence = seed_argument("block_norm", seed, subsequence, dev)
    else:
        subsequence = 0
    N.refuse_tangents("block_norm", x, branch, *coefs)
    N.require_cuda(x, "x")
    flat = len(shape) == 2
    if not (flat and x.is_contiguous()):
        x = _rows(x, c) if c else x.reshape(rows, 0)
    if not (flat and branch.is_contiguous()):
        branch = _rows(branch, c) if c else branch.reshape(rows, 0)
    o.n, o.c, o.code, o.batch, o.per_batch = rows, c, N.DTYPE_CODE[dtype], batch, largest != 1
    o.p, o.seed, o.subsequence = p, seed_value, subsequence
    o.layer, o.branch_norm = int(norm == "layer"), int(bool(branch_norm))
    o.residual_scale, o.eps = float(residual_scale), float(eps)
    if some:
        coords, seed_at = N.savable(coords), N.savable(seed_at)
        y, h = _BlockNorm.apply(x, branch, coords, seed_at, o, packed, *coefs)
    else:
        y, h, _ = _forward(x, branch, coords, seed_at, o, packed, False)
    return (y, h) if flat else (y.reshape(shape), h.reshape(shape))


__all__ = ["block_norm"]
