"""The border between two blocks of a transformer in one pass (``sv_block_norm``): dropout and norm of a
block's result, gate, residual scale and addition, then the next block's norm with its modulation
(``src/mlx_diffuser/models/trellis_slat.py:77-80`` modulates the same way), with gradients."""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from .. import _native as N
from .dropout import check_share, seed_argument
from .norm import _rows

_COEFS = ("weight", "bias", "branch_weight", "gate", "scale", "shift")


def _row(t: torch.Tensor | None) -> N.Rows:
    if t is None:
        return N.Rows(None, 0, 0)
    per_batch = t.ndim == 2 and t.shape[0] > 1
    return N.Rows(t.data_ptr(), t.stride(0) if per_batch else 0, N.DTYPE_CODE[t.dtype])


def _per_batch(coefs) -> bool:
    return any(t is not None and t.ndim == 2 and t.shape[0] > 1 for t in coefs)


def _arguments(branch, h, stats, coords, coefs, o) -> N.BlockNormArgs:
    n, c = h.shape
    a = N.BlockNormArgs(
        n=n, batch=o["batch"], branch=branch.data_ptr(), branch_stride=max(branch.stride(0), c),
        h=h.data_ptr(), stats=N.ptr(stats), coords=N.ptr(coords), dropout=o["p"], seed=o["seed"],
        subsequence=o["subsequence"], channels=c, dtype=N.DTYPE_CODE[h.dtype], layer=o["layer"],
        branch_norm=o["branch_norm"], residual_scale=o["residual_scale"], eps=o["eps"])
    for name, t in zip(_COEFS, coefs):
        setattr(a, name, _row(t))
    return a


def _forward(x, branch, coords, seed_at, coefs, o, keep):
    n, c = x.shape
    h, y = x.new_empty((n, c)), x.new_empty((n, c))
    stats = x.new_empty((n, 4), dtype=torch.float32) if keep else None
    a = _arguments(branch, h, stats, coords, coefs, o)
    a.x, a.x_stride, a.seed_at = x.data_ptr(), max(x.stride(0), c), N.ptr(seed_at)
    with N.on_device(x.device):
        rc = N.load().sv_block_norm(ctypes.byref(a), y.data_ptr(),
                                    N.status_word(x.device).data_ptr(), N.stream(x.device))
    N.check(rc, "block_norm")
    return y, h, stats


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, coords, seed_at, o, *coefs):
        y, h, stats = _forward(x, branch, coords, seed_at, coefs, o, True)
        ctx.save_for_backward(branch, h, stats, coords, seed_at, *coefs)
        ctx.options = o
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        branch, h, stats, coords, seed_at, *coefs = ctx.saved_tensors
        need_x, need_branch, _, _, _, *need = ctx.needs_input_grad
        if dy is None and dh is None:
            return (None,) * len(ctx.needs_input_grad)
        n, c = h.shape
        dev = h.device
        o = ctx.options
        dy = None if dy is None else dy.contiguous()
        dh = None if dh is None else dh.contiguous()
        dx = h.new_empty((n, c)) if need_x else None
        dbranch = h.new_empty((n, c)) if need_branch else None
        grads = [torch.empty(t.shape, dtype=t.dtype, device=dev) if want else None
                 for t, want in zip(coefs, need)]
        a = _arguments(branch, h, stats, coords, coefs, o)
        a.seed_at = N.ptr(seed_at)
        g = N.BlockNormGrads(*(_row(t) for t in grads))
        lib = N.load()
        with N.on_device(dev):
            batch = o["batch"] if _per_batch(coefs) else 0
            nbytes = lib.sv_block_norm_backward_workspace_bytes(n, c, batch)
            ws = N.workspace(nbytes, dev) if batch or any(need) else None
            rc = lib.sv_block_norm_backward(
                ctypes.byref(a), N.ptr(dy), N.ptr(dh), N.ptr(dx), N.ptr(dbranch), ctypes.byref(g),
                N.ptr(ws), nbytes, N.stream(dev))
        N.check(rc, "block_norm (backward)")
        return dx, dbranch, None, None, None, *grads


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
    if x.ndim < 1 or x.dtype not in N.DTYPE_CODE:
        raise ValueError(f"block_norm: unsupported input, shape {tuple(x.shape)}, dtype {x.dtype}")
    if norm not in ("layer", "rms"):
        raise ValueError(f"block_norm: unknown norm {norm!r}")
    c = x.shape[-1]
    rows = math.prod(x.shape[:-1])
    if branch.shape != x.shape or branch.dtype != x.dtype:
        raise ValueError(f"block_norm: branch must be a {tuple(x.shape)} {x.dtype} tensor, got "
                         f"{tuple(branch.shape)} {branch.dtype}")
    if branch_weight is not None and not branch_norm:
        raise ValueError("block_norm: branch_weight goes with branch_norm")
    for name, t in (("weight", weight), ("bias", bias), ("branch_weight", branch_weight)):
        if t is not None and (t.shape != (c,) or t.dtype not in N.DTYPE_CODE):
            raise ValueError(f"block_norm: {name} must be a float tensor of shape ({c},)")
    largest = 1
    for name, t in (("gate", gate), ("scale", scale), ("shift", shift)):
        if t is None:
            continue
        if t.ndim not in (1, 2) or t.shape[-1] != c or t.dtype not in N.DTYPE_CODE:
            raise ValueError(f"block_norm: {name} must be a float tensor of shape (B, {c})")
        largest = max(largest, t.shape[0] if t.ndim == 2 else 1)
    batch = largest if batch_size is None else int(batch_size)
    for name, t in (("gate", gate), ("scale", scale), ("shift", shift)):
        if t is not None and t.ndim == 2 and t.shape[0] not in (1, batch):
            raise ValueError(f"block_norm: {name} has {t.shape[0]} rows for batch {batch}")
    if largest > 1:
        if coords is None:
            raise ValueError("block_norm: rows per batch element need the coordinates")
        if coords.shape != (rows, 4) or coords.dtype != torch.int32:
            raise ValueError(f"block_norm: coords must be an int32 tensor of shape ({rows}, 4)")
    else:
        coords = None
    for name, t in (("branch", branch), ("weight", weight), ("bias", bias), ("gate", gate),
                    ("branch_weight", branch_weight), ("scale", scale), ("shift", shift),
                    ("coords", coords)):
        if t is not None and t.device != x.device:
            raise ValueError(f"block_norm: {name} is on {t.device}, x on {x.device}")
    if not eps >= 0:
        raise ValueError("block_norm: eps must not be negative")
    p = check_share("block_norm", dropout)
    seed_value, seed_at = 0, None
    if p > 0:
        if seed is None:
            raise ValueError("block_norm: dropout needs a seed")
        seed_value, seed_at, subsequence = seed_argument("block_norm", seed, subsequence, x.device)
    else:
        subsequence = 0
    N.refuse_tangents("block_norm", x, branch, weight, bias, branch_weight, gate, scale, shift)
    N.require_cuda(x, "x")
    x2, branch2 = (_rows(t, c) if c else t.reshape(rows, 0) for t in (x, branch))
    if coords is not None:
        coords = coords.contiguous()

    def dense(t):
        if t is None or ((t.stride(-1) == 1 or c <= 1)
                         and (t.ndim == 1 or t.shape[0] <= 1 or t.stride(0) >= c)):
            return t
        return t.contiguous()

    coefs = [dense(t) for t in (weight, bias, branch_weight, gate, scale, shift)]
    o = {"batch": batch, "p": p, "seed": seed_value, "subsequence": subsequence,
         "layer": int(norm == "layer"), "branch_norm": int(bool(branch_norm)),
         "residual_scale": float(residual_scale), "eps": float(eps)}
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (x, branch, *coefs)):
        y, h = _BlockNorm.apply(x2, branch2, coords, seed_at, o, *coefs)
    else:
        y, h, _ = _forward(x2, branch2, coords, seed_at, coefs, o, False)
    return (y, h) if x.ndim == 2 else (y.reshape(x.shape), h.reshape(x.shape))


__all__ = ["block_norm"]
