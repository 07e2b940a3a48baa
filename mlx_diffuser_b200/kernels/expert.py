"""A mixture of experts over feature rows: the router (``sv_route``) and the linear projections grouped by
expert (``sv_expert_linear``), with gradients."""

from __future__ import annotations

import dataclasses

import torch
from torch.autograd.function import once_differentiable

from .. import _native as N
from .linear import _ld, _row_major

MAX_EXPERTS = 1024
MAX_CHOICES = 32


@dataclasses.dataclass
class ExpertRoutes:
    """Where each row goes: ``route``'s result.

    ``experts`` [rows, k] int32, -1 where there is none; ``weights`` [rows, k] float32, with gradients
    to the logits. The slots ``row * k + choice`` by expert, in ``order`` [rows * k]: expert e has positions
    ``offsets[e]`` to ``offsets[e + 1]``, slots without an expert come last; ``place`` [rows, k] is a
    slot's position, or -1."""

    experts: torch.Tensor
    weights: torch.Tensor
    order: torch.Tensor
    offsets: torch.Tensor
    place: torch.Tensor

    @property
    def rows(self) -> int:
        return self.experts.shape[0]

    @property
    def choices(self) -> int:
        return self.experts.shape[1]

    @property
    def num_experts(self) -> int:
        return self.offsets.shape[0] - 1


def _route(logits, k, normalize):
    """(weights, experts, order, offsets, place)."""

    n, e = logits.shape
    dev = logits.device
    lib = N.load()
    weights = torch.empty((n, k), dtype=torch.float32, device=dev)
    experts = torch.empty((n, k), dtype=torch.int32, device=dev)
    place = torch.empty_like(experts)
    order = experts.new_empty((n * k,))
    offsets = experts.new_empty((e + 1,))
    nbytes = lib.sv_route_workspace_bytes(n, e, k)
    ws = N.workspace(nbytes, dev) if nbytes else None
    rc = N.call(dev, lib.sv_route, logits.data_ptr(), max(logits.stride(0), e), n, e, k,
                N.DTYPE_CODE[logits.dtype], normalize, experts.data_ptr(), weights.data_ptr(),
                order.data_ptr(), offsets.data_ptr(), place.data_ptr(), N.ptr(ws), nbytes,
                N.stream(dev))
    if rc:
        N.check(rc, "route")
    return weights, experts, order, offsets, place


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, normalize, found):
        weights, experts, *rest = _route(logits, k, normalize)
        found += experts, *rest
        ctx.save_for_backward(logits, experts, weights)
        ctx.normalize = normalize
        return weights

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights):
        logits, experts, weights = ctx.saved_tensors
        n, e = logits.shape
        dev = logits.device
        dweights = dweights.contiguous()
        dlogits = torch.empty((n, e), dtype=logits.dtype, device=dev)
        rc = N.call(dev, N.load().sv_route_backward, logits.data_ptr(), max(logits.stride(0), e),
                    n, e, experts.shape[1], N.DTYPE_CODE[logits.dtype], ctx.normalize,
                    experts.data_ptr(), weights.data_ptr(), dweights.data_ptr(), dlogits.data_ptr(),
                    N.stream(dev))
        if rc:
            N.check(rc, "route (backward)")
        return dlogits, None, None, None


def route(logits: torch.Tensor, k: int, *, normalize: bool = True) -> ExpertRoutes:
    """Sends each row to the ``k`` experts with the largest ``logits`` (rows, experts): float32,
    float16 or bfloat16, at most 1024 experts and 32 choices.

    Choices go by falling logit, the lower expert first among equals. An expert whose logit is -inf is
    never chosen: a row that has fewer than ``k`` others has -1 in its last choices, with weight
    0. ``weights`` are the softmax over the chosen logits, or over all of them without ``normalize``;
    their gradients reach ``logits``. As in ``torch.topk`` a NaN counts as the largest, and as in a softmax
    it makes the row's weights NaN. Nothing is read back to the host.
    """

    logits = N.as_tensor(logits)
    if logits.ndim != 2 or logits.dtype not in N.DTYPE_CODE:
        raise ValueError(f"route: logits must be a float (rows, experts) tensor, got "
                         f"{tuple(logits.shape)} {logits.dtype}")
    e = logits.shape[1]
    if not 1 <= e <= MAX_EXPERTS:
        raise ValueError(f"route: 1 to {MAX_EXPERTS} experts, got {e}")
    k = int(k)
    if not 1 <= k <= min(e, MAX_CHOICES):
        raise ValueError(f"route: 1 to {min(e, MAX_CHOICES)} choices, got {k}")
    N.refuse_tangents("route", logits)
    N.require_cuda(logits, "logits")
    logits = _row_major(logits)
    if torch.is_grad_enabled() and logits.requires_grad:
        found: list[torch.Tensor] = []
        weights = _Route.apply(logits, k, int(bool(normalize)), found)
        experts, order, offsets, place = found
    else:
        weights, experts, order, offsets, place = _route(logits, k, int(bool(normalize)))
    return ExpertRoutes(experts, weights, order, offsets, place)


def _pack(x, weight, bias, p, order, offsets, place, preact, rows, o) -> bytes:
    experts, outputs, inputs = weight.shape
    n, k = p.shape
    return N.EXPERT_ARGS.pack(
        n, x.data_ptr(), _ld(x), weight.data_ptr(), max(weight.stride(1), inputs),
        weight.stride(0) if experts > 1 else outputs * max(weight.stride(1), inputs),
        0 if bias is None else bias.data_ptr(), order.data_ptr(),
        offsets.data_ptr(), place.data_ptr(), p.data_ptr(), 0 if preact is None else preact.data_ptr(),
        0 if rows is None else rows.data_ptr(), inputs, outputs, k, experts, N.DTYPE_CODE[x.dtype],
        *o)


def _forward(x, weight, bias, p, order, offsets, place, o, keep):
    act, _, combine = o
    n, k = p.shape
    slots, outputs = n * k, weight.shape[1]
    dev = x.device
    out = x.new_empty((n if combine else slots, outputs))
    rows = preact = None
    if combine:
        rows = torch.empty((slots, outputs), dtype=torch.float32, device=dev)
    if keep and act:
        preact = torch.empty((slots, outputs), dtype=torch.float32, device=dev)
    a = _pack(x, weight, bias, p, order, offsets, place, preact, rows, o)
    lib = N.load()
    nbytes = lib.sv_expert_linear_workspace_bytes(a, N.SV_LINEAR_FORWARD, 0, 0, None)
    ws = N.workspace(nbytes, dev) if nbytes else None
    rc = N.call(dev, lib.sv_expert_linear, a, out.data_ptr(), N.ptr(ws), nbytes,
                N.status_word(dev).data_ptr(), N.stream(dev))
    if rc:
        N.check(rc, "expert_linear")
    return out, preact, rows


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, p, order, offsets, place, o):
        act, gather, combine = o
        if combine and ctx.needs_input_grad[3]:
            combine = 2  # the weights' gradients are formed from the positions' results
        out, preact, rows = _forward(x, weight, bias, p, order, offsets, place, (act, gather, combine),
                                     True)
        ctx.save_for_backward(x, weight, p, order, offsets, place, preact, rows)
        ctx.options = o
        ctx.bias_shape = None if bias is None else bias.shape
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x, weight, p, order, offsets, place, preact, rows = ctx.saved_tensors
        need_x, need_w, need_b, need_p, *_ = ctx.needs_input_grad
        o, dev = ctx.options, x.device
        dout = dout.contiguous()
        dx = x.new_empty(x.shape) if need_x else None
        dw = x.new_empty(weight.shape) if need_w else None
        db = x.new_empty(ctx.bias_shape) if need_b else None
        dp = torch.empty_like(p) if need_p else None
        a = _pack(x, weight, None, p, order, offsets, place, preact, rows, o)
        lib = N.load()
        at = dout.data_ptr()
        nbytes = lib.sv_expert_linear_workspace_bytes(a, N.SV_LINEAR_BACKWARD, need_x, need_w, at)
        ws = N.workspace(nbytes, dev)
        rc = N.call(dev, lib.sv_expert_linear_backward, a, at, N.ptr(dx), N.ptr(dw), N.ptr(db),
                    N.ptr(dp), ws.data_ptr(), nbytes, N.status_word(dev).data_ptr(), N.stream(dev))
        if rc:
            N.check(rc, "expert_linear (backward)")
        return dx, dw, db, dp, None, None, None, None


def expert_linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    routes: ExpertRoutes,
    bias: torch.Tensor | None = None,
    *,
    activation: str | None = None,
    gather: bool = False,
    combine: bool = False,
) -> torch.Tensor:
    """Each row through its experts' projections: ``act(x_p @ weight[e].T + bias[e])`` for every position
    p of expert e in ``routes.order``, fp32 accumulation.

    ``weight`` is (experts, N, K), ``bias`` (experts, N); ``activation`` as in
    :func:`~mlx_diffuser_b200.linear`. With ``gather``, ``x`` is (rows, K) and each position takes its
    row; without it, ``x`` is (rows * k, K) in the order of the experts, such as the result of a call
    without ``combine``: (rows * k, N), zeros where no expert has the position. With ``combine`` the result
    is (rows, N): ``sum_j routes.weights[:, j] * r[routes.place[:, j]]`` over the places that an expert
    has, where r, held in float32, are the positions' results. A feed-forward block of experts is

        h = expert_linear(x, up, routes, activation="gelu_tanh", gather=True)
        y = expert_linear(h, down, routes, combine=True)

    float32 (exact fp32 products), float16 and bfloat16 (tensor cores), every tensor of one type but the
    routes' float32 weights, with gradients for all of them (for the weights with ``combine``, which alone
    reads them). No size is read back to the host, whatever the experts' shares are.
    """

    x, weight = N.as_tensor(x), N.as_tensor(weight)
    if activation not in N.ACTIVATION_CODE:
        raise ValueError(f"expert_linear: unknown activation {activation!r}")
    if not isinstance(routes, ExpertRoutes):
        raise ValueError("expert_linear: routes must be an ExpertRoutes")
    shape, dtype, dev = weight.shape, x.dtype, x.device
    if x.ndim != 2 or len(shape) != 3 or shape[2] != x.shape[1]:
        raise ValueError(f"expert_linear: x must have shape (rows, K) and weight (experts, N, K), got "
                         f"{tuple(x.shape)} and {tuple(shape)}")
    if dtype not in N.DTYPE_CODE:
        raise ValueError(f"expert_linear: unsupported dtype {dtype}")
    e, outputs, inputs = shape
    p = routes.weights
    n, k = routes.experts.shape
    want_rows = n if gather else n * k
    if x.shape[0] != want_rows:
        raise ValueError(f"expert_linear: x has {x.shape[0]} rows, the routes ask for {want_rows}")
    if not 1 <= e <= MAX_EXPERTS or routes.num_experts != e:
        raise ValueError(f"expert_linear: weight has {e} experts, the routes {routes.num_experts}")
    for name, t, want, kind in (
        ("weight", weight, shape, dtype),
        ("bias", bias, (e, outputs), dtype),
        ("routes.weights", p, (n, k), torch.float32),
        ("routes.order", routes.order, (n * k,), torch.int32),
        ("routes.offsets", routes.offsets, (e + 1,), torch.int32),
        ("routes.place", routes.place, (n, k), torch.int32),
    ):
        if t is None:
            continue
        if t.shape != want or t.dtype != kind:
            raise ValueError(f"expert_linear: {name} must be a {tuple(want)} {kind} tensor, got "
                             f"{tuple(t.shape)} {t.dtype}")
        if t.device != dev:
            raise ValueError(f"expert_linear: {name} is on {t.device}, x on {dev}")
    N.refuse_tangents("expert_linear", x, weight, bias, p)
    N.require_cuda(x, "x")
    x = _row_major(x)
    if not weight.is_contiguous() and (
            not (weight.stride(2) == 1 or inputs <= 1) or weight.stride(1) < inputs
            or weight.stride(0) < outputs * inputs):
        weight = weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    order, offsets, place = routes.order.contiguous(), routes.offsets.contiguous(), routes.place.contiguous()
    # without the weighted sum the weights are not read, and nothing goes back to the router
    p = p.contiguous() if combine else p.detach() if p.requires_grad else p
    o = N.ACTIVATION_CODE[activation], int(bool(gather)), int(bool(combine))
    if torch.is_grad_enabled() and (
            x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
            or p.requires_grad):
        return _ExpertLinear.apply(x, weight, bias, N.savable(p), N.savable(order),
                                   N.savable(offsets), N.savable(place), o)
    return _forward(x, weight, bias, p, order, offsets, place, o, False)[0]


__all__ = ["ExpertRoutes", "expert_linear", "route"]
