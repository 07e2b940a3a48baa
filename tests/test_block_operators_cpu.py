"""What ``rms_norm``, ``linear`` and the biased attention refuse, and their host-side parts: no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from mlx_diffuser_b200 import _native as N
from mlx_diffuser_b200 import (
    SparseTensor,
    linear,
    position_buckets,
    rms_norm,
    sparse_self_attention,
)
from mlx_diffuser_b200.layers.resblock import SparseLinear


def test_rms_norm_refusals():
    x = torch.zeros((4, 8))
    with pytest.raises(ValueError, match="unsupported input"):
        rms_norm(x.to(torch.float64))
    with pytest.raises(ValueError, match="unsupported input"):
        rms_norm(torch.tensor(1.0))
    with pytest.raises(ValueError, match="residual must be"):
        rms_norm(x, residual=x[:2])
    with pytest.raises(ValueError, match="residual must be"):
        rms_norm(x, residual=x.half())
    with pytest.raises(ValueError, match="weight must be"):
        rms_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="weight must be"):
        rms_norm(x, torch.ones(8, dtype=torch.int32))
    for eps in (-1e-6, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            rms_norm(x, eps=eps)
    with pytest.raises(ValueError, match="no gradients"):
        rms_norm(x.clone().requires_grad_(True), quantize=True)
    with pytest.raises(ValueError, match="weight is on"):
        rms_norm(x, torch.ones(8, device="meta"))
    with pytest.raises(RuntimeError, match="CUDA device"):
        rms_norm(x)


def test_linear_refusals():
    x, w = torch.zeros((4, 8)), torch.zeros((6, 8))
    e = torch.float8_e4m3fn
    with pytest.raises(ValueError, match="unknown activation"):
        linear(x, w, activation="relu")
    for bad in (torch.zeros((6, 7)), torch.zeros(8), torch.zeros((1, 6, 8))):
        with pytest.raises(ValueError, match="weight must have shape"):
            linear(x, bad)
    with pytest.raises(ValueError, match="unsupported dtype"):
        linear(x.double(), w.double())
    with pytest.raises(ValueError, match="x is torch.float32"):
        linear(x, w.half())
    with pytest.raises(ValueError, match="operands' type"):
        linear(x, w, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="scales go with"):
        linear(x, w, x_scale=torch.ones(4))
    with pytest.raises(ValueError, match="bias must be"):
        linear(x, w, torch.zeros(8))
    with pytest.raises(ValueError, match="bias must be"):
        linear(x, w, torch.zeros(6, dtype=torch.float16))
    with pytest.raises(ValueError, match="residual must be"):
        linear(x, w, residual=torch.zeros((4, 8)))
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        linear(x.to(e), w.to(e), out_dtype=torch.float32)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        linear(x.to(e), w.to(e), torch.zeros(6))
    with pytest.raises(ValueError, match="x_scale must be"):
        linear(x.to(e), w.to(e), x_scale=torch.ones((4, 1)))
    with pytest.raises(ValueError, match="weight_scale must be"):
        linear(x.to(e), w.to(e), weight_scale=torch.ones(6, dtype=torch.float16))
    with pytest.raises(ValueError, match="no gradients"):
        linear(x.to(e), w.to(e), torch.zeros(6, dtype=torch.bfloat16, requires_grad=True))
    with pytest.raises(ValueError, match="bias is on"):
        linear(x, w, torch.zeros(6, device="meta"))
    with pytest.raises(RuntimeError, match="CUDA device"):
        linear(x, w)
    with pytest.raises(RuntimeError, match="CUDA device"):
        SparseLinear(8, 6).project(x, activation="silu")
    assert SparseLinear(8, 6).project(x).shape == (4, 6)  # the plain projection as before


def test_biased_attention_refusals():
    coords = torch.zeros((5, 4), dtype=torch.int32)
    x = SparseTensor(torch.zeros((5, 1)), coords)
    q = torch.zeros((5, 2, 16))
    table, lut = torch.zeros((2, 3, 3, 3)), position_buckets(1, 1)

    def run(q=q, k=q, v=q, table=table, lut=lut):
        return sparse_self_attention(x, q, k, v, position_bias=table, position_buckets=lut)

    with pytest.raises(ValueError, match="share shape"):
        run(k=q[:4])
    with pytest.raises(ValueError, match="go together"):
        run(lut=None)
    with pytest.raises(ValueError, match="go together"):
        run(table=None)
    with pytest.raises(ValueError, match="share a dtype"):
        run(table=table.half())
    with pytest.raises(ValueError, match="share a dtype"):
        run(v=q.half())
    with pytest.raises(ValueError, match="share a dtype"):
        run(q=q[:, 0], k=q[:, 0], v=q[:, 0])
    with pytest.raises(ValueError, match="unsupported feature dtype"):
        run(q.double(), q.double(), q.double(), table.double())
    for bad in (torch.zeros((3, 3, 3, 3)), torch.zeros((2, 3, 3)), torch.zeros((2, 3, 5, 3))):
        with pytest.raises(ValueError, match="position_bias must have shape"):
            run(table=bad)
    for bad in (lut.long(), lut[:2], lut[None], lut[:0]):
        with pytest.raises(ValueError, match="position_buckets must be"):
            run(lut=bad)
    wide = torch.zeros((5, 2, 129))
    with pytest.raises(ValueError, match="head_dim"):
        run(wide, wide, wide)
    with pytest.raises(ValueError, match="head_dim"):
        run(table=torch.zeros((2, 26, 26, 26)))
    with pytest.raises(ValueError, match="reach"):
        run(lut=torch.zeros(2 * 1024 + 1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA device"):
        run()


def test_position_buckets():
    assert position_buckets(0, 0).tolist() == [0]
    assert position_buckets(3, 3).tolist() == list(range(7))
    assert position_buckets(3, 9).tolist() == list(range(7))
    # near 1 exactly, then one bucket up to the reach
    assert position_buckets(4, 2).tolist() == [0, 0, 0, 1, 2, 3, 4, 4, 4]
    # three logarithmic steps from 2 to 16: up to 4, 8 and 16
    half = [0, 1, 2, 3, 3, 4, 4, 4, 4, *[5] * 8]
    want = [5 - a for a in half[:0:-1]] + [5 + a for a in half]
    assert position_buckets(16, 5, exact=2).tolist() == want
    for reach, side in ((7, 7), (31, 8), (1023, 12), (15, 1), (2, 1)):
        lut = position_buckets(reach, side)
        assert lut.dtype == torch.int32 and lut.shape == (2 * reach + 1,)
        assert (lut[1:] - lut[:-1]).min() >= 0 and lut[0] == 0 and lut[-1] == 2 * side
        assert torch.equal(lut, 2 * side - lut.flip(0))
    for bad in ((-1, 1), (4, 0), (0, 3), (4, -2)):
        with pytest.raises(ValueError, match="position_buckets"):
            position_buckets(*bad)
    for exact in (0, 3):
        with pytest.raises(ValueError, match="exact"):
            position_buckets(8, 2, exact=exact)


def test_c_entry_points_check_before_any_launch():
    lib = N.load()
    p = 256  # an aligned address that nothing reads: every call below ends before a launch
    assert lib.sv_rms_norm(None, 0, None, 0, 0, 8, 2, 1e-6, None, None, None, None, 2, None,
                           None, None) == N.SV_OK
    assert lib.sv_rms_norm(p, 8, None, 0, 4, 8, 7, 1e-6, None, None, None, p, 2, None,
                           None, None) == N.SV_ERR_BAD_DTYPE
    assert lib.sv_rms_norm(p, 8, None, 0, 4, 8, 2, 1e-6, None, None, None, p, 0, None,
                           None, None) == N.SV_ERR_BAD_DTYPE
    assert lib.sv_rms_norm(p, 8, None, 0, 4, 8, 2, 1e-6, None, None, None, p, 3, None,
                           None, None) == N.SV_ERR_INVALID_ARGUMENT  # e4m3 without a scale
    assert lib.sv_rms_norm(p, 7, None, 0, 4, 8, 2, 1e-6, None, None, None, p, 2, None,
                           None, None) == N.SV_ERR_INVALID_ARGUMENT
    assert lib.sv_rms_norm(p, 9000, None, 0, 4, 8193, 2, 1e-6, None, None, None, p, 2, None,
                           None, None) == N.SV_ERR_UNSUPPORTED
    assert lib.sv_rms_norm(p, 8, None, 0, 4, 8, 2, -1.0, None, None, None, p, 2, None,
                           None, None) == N.SV_ERR_INVALID_ARGUMENT
    assert lib.sv_rms_norm_backward_workspace_bytes(1024) > 0
    assert lib.sv_rms_norm_backward(p, 8, p, None, 4, 8, 2, None, p, p, p, None, 0,
                                    None, None) == N.SV_ERR_WORKSPACE

    def forward(m=20, k=64, n=64, dtype=2, out=2, act=0, ldx=64, ldw=64, x=p, ws=None, nbytes=0):
        return lib.sv_linear_forward(x, ldx, p, ldw, None, None, 0, None, None, m, k, n, dtype, out,
                                     act, p, None, ws, nbytes, None, None)

    assert forward(m=0, x=None) == N.SV_OK
    assert forward(dtype=9) == N.SV_ERR_BAD_DTYPE
    assert forward(out=1) == N.SV_ERR_BAD_DTYPE
    assert forward(dtype=3, out=0) == N.SV_ERR_BAD_DTYPE
    assert forward(act=4) == N.SV_ERR_INVALID_ARGUMENT
    assert forward(ldx=63) == N.SV_ERR_INVALID_ARGUMENT
    assert forward(x=None) == N.SV_ERR_INVALID_ARGUMENT
    assert forward(m=-1) == N.SV_ERR_INVALID_ARGUMENT
    assert forward(m=2**31) == N.SV_ERR_UNSUPPORTED
    # an operand that TMA cannot read needs its padded copy
    assert lib.sv_linear_workspace_bytes(N.SV_LINEAR_FORWARD, 20, 63, 64, 2, 3) >= 84 * 128
    assert forward(k=63, ldx=63, ldw=63) == N.SV_ERR_WORKSPACE
    def backward(m=4, k=8, n=8, dtype=2, act=1, z=p, ldx=8, ldw=8, dx=p, dw=p, db=p, ws=None,
                 nbytes=0):
        return lib.sv_linear_backward(p, z, p, ldx, p, ldw, m, k, n, dtype, act, dx, dw, db, ws,
                                      nbytes, None, None)

    assert backward() == N.SV_ERR_WORKSPACE
    need = lib.sv_linear_workspace_bytes(N.SV_LINEAR_BACKWARD, 4, 8, 8, 2, 4)
    assert need >= 4 * 16 + 4 * 8
    assert backward(ws=p, nbytes=need - 1) == N.SV_ERR_WORKSPACE
    assert backward(z=None) == N.SV_ERR_INVALID_ARGUMENT
    assert backward(dx=None, dw=None, db=None) == N.SV_OK
    assert backward(n=0, dx=None) == backward(m=0, dw=None, db=None) == N.SV_OK
    assert backward(ldw=7) == backward(ldx=7) == N.SV_ERR_INVALID_ARGUMENT
    assert backward(act=4) == N.SV_ERR_INVALID_ARGUMENT
    assert backward(dtype=5) == backward(dtype=3) == N.SV_ERR_BAD_DTYPE
    assert backward(k=-1) == N.SV_ERR_INVALID_ARGUMENT
    assert backward(k=2**31) == N.SV_ERR_UNSUPPORTED

    six = (ctypes.c_int64 * 6)(*[64] * 6)

    def attend(n=4, heads=2, dim=16, dtype=2, buckets=3, reach=1, q=p):
        return lib.sv_window_attention(q, p, p, six, n, heads, dim, dtype, p, 1, p, buckets, p,
                                       reach, 0.25, p, None, None, None, 0, None)

    assert attend(n=0, q=None) == N.SV_OK
    assert attend(dtype=3) == N.SV_ERR_BAD_DTYPE
    assert attend(q=None) == N.SV_ERR_INVALID_ARGUMENT
    assert attend(buckets=0) == N.SV_ERR_INVALID_ARGUMENT
    for bad in ({"dim": 129}, {"buckets": 26}, {"reach": 1024}, {"n": 2**25 + 1},
                {"heads": 65536}):
        assert attend(**bad) == N.SV_ERR_UNSUPPORTED
    assert lib.sv_window_plan_bytes(10) >= 10 * 32 and lib.sv_window_plan_bytes(0) == 0
    assert lib.sv_window_plan(None, None, None, 0, 0, None, None, None) == N.SV_OK
    assert lib.sv_window_plan(p, p, p, 0, 5, p, None, None) == N.SV_ERR_INVALID_ARGUMENT
    nbytes = lib.sv_window_attention_backward_workspace_bytes(100, 2, 3)
    assert nbytes >= 2 * 27 * 8 + 2 * 100 * 4
    assert lib.sv_window_attention_backward(p, p, p, six, p, None, p, p, 100, 2, 16, 2, p, p, 3, p,
                                            1, 0.25, p, p, p, p, p, nbytes - 1,
                                            None) == N.SV_ERR_WORKSPACE
