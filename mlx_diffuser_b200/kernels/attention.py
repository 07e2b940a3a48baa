"""Windowed attention with a learned relative position bias (``sv_window_attention*``): the kernel
calls under ``sparse_self_attention(..., position_bias=...)``."""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from .. import _native as N

MAX_DIM = 128
MAX_BUCKETS = 25
MAX_REACH = 1023


def window_plan(coords: torch.Tensor, perm: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """The window grouping's rows in window order, with coordinates and window bounds
    (``sv_window_plan``)."""

    dev = coords.device
    n = perm.numel()
    lib = N.load()
    plan = torch.empty(max(int(lib.sv_window_plan_bytes(n)), 1), dtype=torch.uint8, device=dev)
    with N.on_device(dev):
        rc = lib.sv_window_plan(coords.data_ptr(), perm.data_ptr(), offsets.data_ptr(),
                                offsets.numel() - 1, n, plan.data_ptr(),
                                N.status_word(dev).data_ptr(), N.stream(dev))
    N.check(rc, "attention plan")
    return plan


def _strides(q, k, v):
    return (ctypes.c_int64 * 6)(q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0),
                                v.stride(1))


def _forward(q, k, v, table, lut, plan, windows, scale, train):
    n, heads, dim = q.shape
    dev = q.device
    out = q.new_empty((n, heads, dim))
    stats = q.new_empty((heads, n, 2), dtype=torch.float32) if train else None
    # what rounding `out` left out: the backward pass takes dS from a difference with dout . out
    rest = torch.empty_like(out) if train and q.dtype != torch.float32 else None
    lib = N.load()
    code = N.DTYPE_CODE[q.dtype]
    with N.on_device(dev):
        nbytes = lib.sv_window_attention_workspace_bytes(n, heads, dim, code, windows)
        ws = N.workspace(nbytes, dev) if nbytes else None
        rc = lib.sv_window_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _strides(q, k, v), n, heads, dim, code,
            plan.data_ptr(), windows, table.data_ptr(), table.shape[-1], lut.data_ptr(),
            lut.numel() // 2, scale, out.data_ptr(), N.ptr(rest), N.ptr(stats), N.ptr(ws), nbytes,
            N.stream(dev))
    N.check(rc, "sparse_self_attention")
    return out, rest, stats


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, lut, plan, windows, scale):
        out, rest, stats = _forward(q, k, v, table, lut, plan, windows, scale, True)
        ctx.scale = scale
        # not a saved tensor: one laid out under inference mode could not be, and nothing changes it
        ctx.plan = plan
        ctx.save_for_backward(q, k, v, table, lut, out, rest, stats)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, table, lut, out, rest, stats = ctx.saved_tensors
        n, heads, dim = q.shape
        dev = q.device
        dout = dout.contiguous()
        dq, dk, dv = (q.new_empty((n, heads, dim)) for _ in range(3))
        dtable = torch.empty_like(table) if ctx.needs_input_grad[3] else None
        lib = N.load()
        nbytes = lib.sv_window_attention_backward_workspace_bytes(n, heads, table.shape[-1])
        with N.on_device(dev):
            ws = N.workspace(nbytes, dev)
            rc = lib.sv_window_attention_backward(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), _strides(q, k, v), out.data_ptr(),
                N.ptr(rest), dout.data_ptr(), stats.data_ptr(), n, heads, dim,
                N.DTYPE_CODE[q.dtype], ctx.plan.data_ptr(), table.data_ptr(), table.shape[-1],
                lut.data_ptr(), lut.numel() // 2, ctx.scale, dq.data_ptr(), dk.data_ptr(),
                dv.data_ptr(), N.ptr(dtable), ws.data_ptr(), nbytes, N.stream(dev))
        N.check(rc, "sparse_self_attention (backward)")
        return dq, dk, dv, dtable, None, None, None, None


def biased_window_attention(q, k, v, table, lut, plan, windows: int, scale: float) -> torch.Tensor:
    """Attention inside the plan's ``windows`` windows: ``q``, ``k``, ``v`` (N, heads, dim) of one type,
    ``table`` (heads, B, B, B) of the same type, ``lut`` int32 (2 * reach + 1,)."""

    q, k, v = (t if t.stride(2) == 1 or t.shape[2] <= 1 else t.contiguous() for t in (q, k, v))
    table, lut = table.contiguous(), lut.contiguous()
    if torch.is_grad_enabled() and (
            q.requires_grad or k.requires_grad or v.requires_grad or table.requires_grad):
        return _WindowAttention.apply(q, k, v, table, lut, plan, windows, scale)
    return _forward(q, k, v, table, lut, plan, windows, scale, False)[0]


__all__ = ["biased_window_attention", "window_plan"]
