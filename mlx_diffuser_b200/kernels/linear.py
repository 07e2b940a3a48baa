"""Linear projection of feature rows with bias, activation and residual in its epilogue
(``sv_linear_*``): ``act(x @ weight.T + bias) + residual`` in one pass, with gradients, and with
8-bit operands. ``SparseLinear`` (``src/mlx_diffuser/layers/trellis_sparse.py:13-30``) calls it when
it is given an activation or a residual."""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from .. import _native as N


def _row_major(t: torch.Tensor) -> torch.Tensor:
    """``t`` [rows, cols] as it is when its rows are contiguous and do not overlap."""

    if t.stride(1) == 1 or t.shape[1] <= 1:
        if t.shape[0] <= 1 or t.stride(0) >= t.shape[1]:
            return t
    return t.contiguous()


def _ld(t: torch.Tensor) -> int:
    """Row stride in elements (that of a lone row does not matter)."""

    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _unaligned(address: int, ld: int, t: torch.Tensor) -> bool:
    return (address | ld * t.element_size()) & 15 != 0


def _forward(x, weight, bias, residual, activation, x_scale, w_scale, out_dtype, keep_preact):
    m, k = x.shape
    n = weight.shape[0]
    dev = x.device
    out = weight.new_empty((m, n), dtype=out_dtype)
    preact = weight.new_empty((m, n), dtype=torch.float32) if keep_preact else None
    if m == 0 or n == 0:
        return out, preact
    code = N.DTYPE_CODE.get(x.dtype, N.SV_FLOAT8_E4M3)
    px, ldx, pw, ldw = x.data_ptr(), _ld(x), weight.data_ptr(), _ld(weight)
    copies = _unaligned(px, ldx, x) + 2 * _unaligned(pw, ldw, weight)
    lib = N.load()
    with N.on_device(dev):
        nbytes = lib.sv_linear_workspace_bytes(N.SV_LINEAR_FORWARD, m, k, n, code, copies)
        ws = N.workspace(nbytes, dev) if nbytes else None
        rc = lib.sv_linear_forward(
            px, ldx, pw, ldw, N.ptr(bias), N.ptr(residual),
            0 if residual is None else _ld(residual), N.ptr(x_scale), N.ptr(w_scale), m, k, n,
            code, N.DTYPE_CODE[out_dtype], N.ACTIVATION_CODE[activation], out.data_ptr(),
            N.ptr(preact), N.ptr(ws), nbytes, N.status_word(dev).data_ptr(), N.stream(dev))
    N.check(rc, "linear")
    return out, preact


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        acts = N.ACTIVATION_CODE[activation] != 0
        out, preact = _forward(x, weight, bias, residual, activation, None, None, x.dtype, acts)
        ctx.activation = activation
        ctx.save_for_backward(x, weight, preact)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x, weight, preact = ctx.saved_tensors
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        dout = dout.contiguous()
        m, k = x.shape
        n = weight.shape[0]
        dev = x.device
        code = N.DTYPE_CODE[x.dtype]
        dx = x.new_empty((m, k)) if need_x else None
        dw = x.new_empty((n, k)) if need_w else None
        db = x.new_empty((n,)) if need_b else None
        if need_x or need_w or need_b:
            px, pw, pd = x.data_ptr(), weight.data_ptr(), dout.data_ptr()
            ldx, ldw = _ld(x), _ld(weight)
            copies = (_unaligned(px, ldx, x) + 2 * _unaligned(pw, ldw, weight)
                      + 4 * (preact is not None or _unaligned(pd, n, dout)))
            lib = N.load()
            with N.on_device(dev):
                nbytes = lib.sv_linear_workspace_bytes(N.SV_LINEAR_BACKWARD, m, k, n, code, copies)
                # held over the call: another thread's launches on this stream could take it meanwhile
                ws = N.workspace(nbytes, dev)
                rc = lib.sv_linear_backward(
                    pd, N.ptr(preact), px, ldx, pw, ldw, m, k, n, code,
                    N.ACTIVATION_CODE[ctx.activation], N.ptr(dx), N.ptr(dw), N.ptr(db),
                    ws.data_ptr(), nbytes, N.status_word(dev).data_ptr(), N.stream(dev))
            N.check(rc, "linear (backward)")
        return dx, dw, db, dout if need_r else None, None


def linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    activation: str | None = None,
    residual: torch.Tensor | None = None,
    x_scale: torch.Tensor | None = None,
    weight_scale: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` over the last axis of ``x`` (..., K), fp32
    accumulation, one rounding.

    ``weight`` is (N, K), ``bias`` (N,), ``residual`` (..., N); ``activation`` is None, ``"silu"``,
    ``"gelu"`` or ``"gelu_tanh"``. float32 (exact fp32 products), float16 and bfloat16 (tensor
    cores), every tensor of one type, with gradients for all of them.

    8 bits: ``x`` and ``weight`` in ``torch.float8_e4m3fn`` stand for ``x * x_scale[..., None]`` and
    ``weight * weight_scale[:, None]`` (fp32 scales per row, as ``rms_norm(..., quantize=True)``
    gives them; None is 1). The result, the bias and the residual are bfloat16 or float16
    (``out_dtype``, by default the bias's or the residual's type, else bfloat16). No gradients.
    """

    x, weight = N.as_tensor(x), N.as_tensor(weight)
    if activation not in N.ACTIVATION_CODE:
        raise ValueError(f"linear: unknown activation {activation!r}")
    if x.ndim < 1 or weight.ndim != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"linear: weight must have shape (N, {x.shape[-1] if x.ndim else '?'}), "
                         f"got {tuple(weight.shape)}")
    n = weight.shape[0]
    e4m3 = x.dtype == torch.float8_e4m3fn
    if not e4m3 and x.dtype not in N.DTYPE_CODE:
        raise ValueError(f"linear: unsupported dtype {x.dtype}")
    if weight.dtype != x.dtype:
        raise ValueError(f"linear: x is {x.dtype} and weight {weight.dtype}")
    if e4m3:
        if out_dtype is None:
            out_dtype = next((t.dtype for t in (bias, residual) if t is not None), torch.bfloat16)
        if out_dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"linear: 8-bit operands give float16 or bfloat16, not {out_dtype}")
    else:
        if x_scale is not None or weight_scale is not None:
            raise ValueError("linear: scales go with float8_e4m3fn operands")
        if out_dtype not in (None, x.dtype):
            raise ValueError(f"linear: the result has the operands' type {x.dtype}")
        out_dtype = x.dtype
    dev = x.device
    rows = x.shape[:-1]
    for name, t, want, dtype in (
        ("weight", weight, weight.shape, x.dtype),
        ("bias", bias, (n,), out_dtype),
        ("residual", residual, (*rows, n), out_dtype),
        ("x_scale", x_scale, rows, torch.float32),
        ("weight_scale", weight_scale, (n,), torch.float32),
    ):
        if t is None:
            continue
        if t.shape != want or t.dtype != dtype:
            raise ValueError(f"linear: {name} must be a {tuple(want)} {dtype} tensor, got "
                             f"{tuple(t.shape)} {t.dtype}")
        if t.device != dev:
            raise ValueError(f"linear: {name} is on {t.device}, x on {dev}")
    grads = torch.is_grad_enabled() and (
        x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
        or (residual is not None and residual.requires_grad))
    if grads and e4m3:
        raise ValueError("linear: 8-bit operands have no gradients")
    N.refuse_tangents("linear", x, weight, bias, residual, x_scale, weight_scale)
    N.require_cuda(x, "x")
    x2 = _row_major(x if x.ndim == 2 else x.reshape(math.prod(rows), x.shape[-1]))
    w2 = _row_major(weight)
    r2 = None
    if residual is not None:
        r2 = _row_major(residual if x.ndim == 2 else residual.reshape(x2.shape[0], n))
    b2 = None if bias is None else bias.contiguous()
    if grads:
        out = _Linear.apply(x2, w2, b2, r2, activation)
    else:
        xs = None if x_scale is None else x_scale.reshape(-1).contiguous()
        ws = None if weight_scale is None else weight_scale.contiguous()
        out, _ = _forward(x2, w2, b2, r2, activation, xs, ws, out_dtype, False)
    return out if x.ndim == 2 else out.reshape(*rows, n)


__all__ = ["linear"]
