"""Bindings of the row norms.

``row_norm`` (``sv_rownorm``): LayerNorm32 with the residual block's modulation and SiLU fused
into one pass over the rows (``src/mlx_diffuser/layers/trellis.py:16-43``,
``src/mlx_diffuser/models/trellis_slat.py:77-80``).

``rms_norm`` (``sv_rms_norm``): root-mean-square norm with the residual's addition, an 8-bit output
with one scale per row, and gradients."""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from .. import _native as N


def row_norm(
    x: torch.Tensor,
    *,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    scale: torch.Tensor | None = None,
    shift: torch.Tensor | None = None,
    coords: torch.Tensor | None = None,
    batch_size: int | None = None,
    silu: bool = False,
    eps: float = 1e-6,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``silu?( LN32(x) [* weight + bias] [* (1 + scale[b]) + shift[b]] )`` over the last axis,
    fp32 inside, one rounding to ``x.dtype``. ``weight`` / ``bias``: fp32 ``[C]``. ``scale`` /
    ``shift``: ``[B, C]`` (or ``[C]`` / ``[1, C]``, shared by every row), rows picked by
    ``coords[:, 0]`` of an ``[N, 4]`` int32 coordinate tensor."""

    N.require_cuda(x, "x")
    c = x.shape[-1]
    flat = x.reshape(-1, c).contiguous()
    n = flat.shape[0]
    if flat.dtype not in N.DTYPE_CODE:
        raise ValueError(f"row_norm: unsupported dtype {flat.dtype}")
    dev = flat.device
    if weight is not None:
        weight = weight.to(device=dev, dtype=torch.float32).contiguous()
        if weight.shape != (c,):
            raise ValueError(f"row_norm: weight must have shape ({c},)")
    if bias is not None:
        bias = bias.to(device=dev, dtype=torch.float32).contiguous()
    mods: list[torch.Tensor | None] = []
    for name, t in (("scale", scale), ("shift", shift)):
        if t is None:
            mods.append(None)
            continue
        t = t.to(device=dev, dtype=flat.dtype)
        if t.ndim == 1:
            t = t[None]
        if t.ndim != 2 or t.shape[1] != c:
            raise ValueError(f"row_norm: {name} must have shape (B, {c})")
        if t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < c):
            t = t.contiguous()
        mods.append(t)
    live = [m for m in mods if m is not None]
    b = 0
    mod_stride = 0
    if live:
        if coords is None:
            raise ValueError("row_norm: modulation needs the coordinates (batch column)")
        rows = {m.shape[0] for m in live}
        b = int(batch_size) if batch_size is not None else max(rows)
        if any(r not in (1, b) for r in rows):
            raise ValueError(f"row_norm: modulation rows {sorted(rows)} for batch {b}")
        strides = {0 if m.shape[0] == 1 else m.stride(0) for m in live}
        if len(strides) > 1:  # scale and shift laid out differently: make both dense
            mods = [None if m is None else m.expand(b, c).contiguous() for m in mods]
            strides = {c}
        mod_stride = strides.pop()
        coords = coords.to(device=dev, dtype=torch.int32).contiguous()
        if coords.shape != (n, 4):
            raise ValueError(f"row_norm: coords must have shape ({n}, 4)")
    if out is None:
        out = torch.empty_like(flat)
    rc = N.load().sv_rownorm(
        flat.data_ptr(), n, c, N.DTYPE_CODE[flat.dtype], float(eps), N.ptr(weight), N.ptr(bias),
        N.ptr(mods[0]), N.ptr(mods[1]), mod_stride, N.ptr(coords), b, int(bool(silu)),
        out.data_ptr(),
        N.status_word(dev).data_ptr(), N.stream(dev),
    )
    N.check(rc, "row_norm")
    return out.reshape(x.shape)


def _rows(t: torch.Tensor, c: int) -> torch.Tensor:
    """``t`` as [rows, c] with contiguous rows that do not overlap; a view where it can be one."""

    t = t.reshape(-1, c) if t.ndim != 2 else t
    if (t.stride(1) == 1 or c <= 1) and (t.shape[0] <= 1 or t.stride(0) >= c):
        return t
    return t.contiguous()


def _rms_forward(x, residual, weight, eps, quantize, keep_rstd):
    n, c = x.shape
    dev = x.device
    lib = N.load()
    h = x.new_empty((n, c)) if residual is not None else None
    rstd = x.new_empty((n,), dtype=torch.float32) if keep_rstd else None
    scale = x.new_empty((n,), dtype=torch.float32) if quantize else None
    out = x.new_empty((n, c), dtype=torch.float8_e4m3fn) if quantize else x.new_empty((n, c))
    code = N.DTYPE_CODE[x.dtype]
    with N.on_device(dev):
        rc = lib.sv_rms_norm(
            x.data_ptr(), max(x.stride(0), c), N.ptr(residual),
            max(residual.stride(0), c) if residual is not None else 0, n, c, code, eps,
            N.ptr(weight), N.ptr(h), N.ptr(rstd), out.data_ptr(),
            N.SV_FLOAT8_E4M3 if quantize else code, N.ptr(scale), N.status_word(dev).data_ptr(),
            N.stream(dev))
    N.check(rc, "rms_norm")
    return out, scale, h, rstd


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        w32 = None if weight is None else weight.to(torch.float32).contiguous()
        out, _, h, rstd = _rms_forward(x, residual, w32, eps, False, True)
        ctx.save_for_backward(x if h is None else h, w32, rstd)
        ctx.weight_dtype = None if weight is None else weight.dtype
        ctx.set_materialize_grads(False)
        return out if h is None else (out, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, w32, rstd = ctx.saved_tensors
        if dy is None and dh is None:
            return None, None, None, None
        need_x, need_r, need_w, _ = ctx.needs_input_grad
        if dy is None:
            dw = torch.zeros_like(w32, dtype=ctx.weight_dtype) if need_w else None
            return (dh if need_x else None), (dh if need_r else None), dw, None
        n, c = h.shape
        dev = h.device
        lib = N.load()
        dy = dy.contiguous()
        dh = None if dh is None else dh.contiguous()
        dx = h.new_empty((n, c))
        dw = h.new_empty((c,), dtype=torch.float32) if need_w else None
        with N.on_device(dev):
            nbytes = lib.sv_rms_norm_backward_workspace_bytes(c) if need_w else 0
            ws = N.workspace(nbytes, dev) if need_w else None
            rc = lib.sv_rms_norm_backward(
                h.data_ptr(), max(h.stride(0), c), dy.data_ptr(), N.ptr(dh), n, c,
                N.DTYPE_CODE[h.dtype], N.ptr(w32), rstd.data_ptr(), dx.data_ptr(), N.ptr(dw),
                N.ptr(ws), nbytes, N.status_word(dev).data_ptr(), N.stream(dev))
        N.check(rc, "rms_norm (backward)")
        if dw is not None:
            dw = dw.to(ctx.weight_dtype)
        return (dx if need_x else None), (dx if need_r else None), dw, None


def rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    *,
    residual: torch.Tensor | None = None,
    eps: float = 1e-6,
    quantize: bool = False,
):
    """``h * rsqrt(mean(h * h) + eps) * weight`` over the last axis, ``h = x + residual`` (``x``
    without one), fp32 inside.

    ``h`` is rounded to ``x.dtype`` before it is normed: it is the residual stream that goes on to
    the next block, returned beside the result. ``weight``: (C,), any float type, used in fp32.
    ``residual``: like ``x``. At most 8192 channels.

    Returns ``y`` in ``x.dtype``, or ``(y, h)`` with a residual. With ``quantize``, ``y`` is a pair
    ``(q, scale)``: ``q`` in ``torch.float8_e4m3fn`` and one fp32 scale per row (``x.shape[:-1]``),
    the row's largest magnitude over 448 (1 for a row of zeros), so that ``y = q * scale``, as
    ``linear`` takes it. Gradients for ``x``, ``residual`` and ``weight``; the 8-bit form has none.
    """

    x = N.as_tensor(x)
    if x.ndim < 1 or x.dtype not in N.DTYPE_CODE:
        raise ValueError(f"rms_norm: unsupported input, shape {tuple(x.shape)}, dtype {x.dtype}")
    c = x.shape[-1]
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"rms_norm: residual must be a {tuple(x.shape)} {x.dtype} tensor, got "
                         f"{tuple(residual.shape)} {residual.dtype}")
    if weight is not None and (weight.shape != (c,) or not weight.is_floating_point()):
        raise ValueError(f"rms_norm: weight must be a float tensor of shape ({c},)")
    for name, t in (("residual", residual), ("weight", weight)):
        if t is not None and t.device != x.device:
            raise ValueError(f"rms_norm: {name} is on {t.device}, x on {x.device}")
    if not eps >= 0:
        raise ValueError("rms_norm: eps must not be negative")
    grads = torch.is_grad_enabled() and (
        x.requires_grad or (residual is not None and residual.requires_grad)
        or (weight is not None and weight.requires_grad))
    if grads and quantize:
        raise ValueError("rms_norm: the 8-bit output has no gradients")
    N.refuse_tangents("rms_norm", x, residual, weight)
    N.require_cuda(x, "x")
    x2 = _rows(x, c) if c else x.reshape(math.prod(x.shape[:-1]), 0)
    r2 = None
    if residual is not None:
        r2 = _rows(residual, c) if c else residual.reshape(x2.shape)
    if grads:
        out = _RmsNorm.apply(x2, r2, weight, float(eps))
        if residual is None:
            return out if x.ndim == 2 else out.reshape(x.shape)
        return out if x.ndim == 2 else (out[0].reshape(x.shape), out[1].reshape(x.shape))
    w32 = None if weight is None else weight.to(torch.float32).contiguous()
    out, scale, h, _ = _rms_forward(x2, r2, w32, float(eps), bool(quantize), False)
    if x.ndim != 2:
        out = out.reshape(x.shape)
        h = None if h is None else h.reshape(x.shape)
        scale = None if scale is None else scale.reshape(x.shape[:-1])
    y = (out, scale) if quantize else out
    return y if residual is None else (y, h)


__all__ = ["rms_norm", "row_norm"]
