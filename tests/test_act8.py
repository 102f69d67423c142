"""8-bit activation checkpoints on the CPU: refusals, sizes, and the oracle's own properties."""
import math

import pytest
import torch

import operator_oracle as Q

A = 1 << 20


def refuse(pkg, text, call, *args, **kwargs):
    with pytest.raises(pkg.RlcuError) as e:
        call(*args, **kwargs)
    assert e.value.code == pkg.ERR_INVALID and text in str(e.value), str(e.value)


def test_sizes(pkg):
    assert [pkg.act8_blocks(c) for c in (0, 1, 127, 128, 129, 4096)] == [0, 1, 1, 1, 2, 32]
    assert pkg.act8_rmsnorm_grad_workspace(0, 4096) == 0
    assert pkg.act8_rmsnorm_grad_workspace(1, 4096) >= 4 * 4096
    assert pkg.act8_rmsnorm_grad_workspace(1 << 20, 4096) <= 16 << 20


def test_store_and_load_refusals(pkg):
    B, C = A + (1 << 16), A + (2 << 16)
    store = lambda x=A, dt=pkg.F16, rows=2, cols=8, codes=B, scales=C, **k: pkg.act8_store(x, dt, rows, cols, codes, scales, **k)  # noqa: E731
    load = lambda x=A, dt=pkg.F16, rows=2, cols=8, codes=B, scales=C, **k: pkg.act8_load(codes, scales, rows, cols, x, dt, **k)  # noqa: E731
    for f in (store, load):
        refuse(pkg, "dtype", f, dt=9)
        refuse(pkg, "null", f, x=None)
        refuse(pkg, "null", f, codes=None)
        refuse(pkg, "null", f, scales=None)
        refuse(pkg, "stride", f, x_stride=7)
        refuse(pkg, "stride", f, code_stride=7)
        refuse(pkg, "stride", f, rows=1 << 30, x_stride=1 << 40)
        refuse(pkg, "rows", f, rows=1 << 31)
        refuse(pkg, "rows", f, cols=1 << 31)
        refuse(pkg, "aligned", f, x=A + 1)
        refuse(pkg, "overlap", f, codes=A + 8)
        f(x=None, codes=None, scales=None, rows=0)
        f(x=None, codes=None, scales=None, cols=0)


def test_rmsnorm_refusals(pkg):
    B, C, D = A + (1 << 16), A + (2 << 16), A + (3 << 16)

    def forward(rows=2, cols=8, w=C, wd=pkg.F32, eps=1e-6, y=D, dt=pkg.F16, **k):
        pkg.act8_rmsnorm(A, B, rows, cols, w, wd, eps, y, dt, **k)

    def backward(rows=2, cols=8, w=C, wd=pkg.F32, eps=1e-6, dy=D, dt=pkg.F16, dx=D + 4096, dw=A, ws=D + 8192, n=1 << 20, **k):
        pkg.act8_rmsnorm_grad(A, B, rows, cols, w, wd, eps, dy, dt, dx, dw, ws, n, **k)

    for f in (forward, backward):
        refuse(pkg, "dtype", f, dt=5)
        refuse(pkg, "dtype", f, wd=5)
        refuse(pkg, "weight", f, w=None)
        refuse(pkg, "weight", f, w=C + 2)
        for eps in (-1.0, math.inf, math.nan):
            refuse(pkg, "eps", f, eps=eps)
        refuse(pkg, "stride", f, code_stride=3)
    refuse(pkg, "null", forward, y=None)
    refuse(pkg, "overlap", forward, y=A)
    refuse(pkg, "stride", forward, y_stride=3)
    refuse(pkg, "null", backward, dy=None)
    refuse(pkg, "null", backward, dx=None)
    refuse(pkg, "overlap", backward, dx=D + 2)
    refuse(pkg, "overlap", backward, dx=A)
    refuse(pkg, "overlap", backward, dresidual=D + 4096 + 8)
    refuse(pkg, "stride", backward, dresidual=D, dresidual_stride=2)
    refuse(pkg, "flags", backward, flags=2)
    refuse(pkg, "workspace", backward, ws=None)
    refuse(pkg, "workspace", backward, ws=D + 8192 + 4)
    refuse(pkg, "workspace", backward, n=pkg.act8_rmsnorm_grad_workspace(2, 8) - 1)


def test_rmsnorm_refuses_vectors_that_are_not_aligned(pkg):
    B, C, D = A + (1 << 16), A + (2 << 16), A + (3 << 16)
    refuse(pkg, "rstd", pkg.act8_rmsnorm, A, B, 2, 8, C, pkg.F32, 1e-6, D, pkg.F16, A + 2)
    refuse(pkg, "dweight", pkg.act8_rmsnorm_grad, A, B, 2, 8, C, pkg.F32, 1e-6, D, pkg.F16, D + 4096, C + 6, D + 8192, 1 << 20)


def test_oracle_rounding_is_at_most_half_a_step():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(40, 300, generator=g) * torch.exp(3 * torch.randn(40, 300, generator=g))
    codes, scales = Q.act8_encode(x)
    v = Q.act8_decode(codes, scales)
    s = torch.exp2(scales.to(Q.F64) - 127).repeat_interleave(128, 1)[:, :300]
    assert ((v - x).abs() <= torch.maximum(x.to(Q.F64).abs() * 2.0 ** -4, s * 2.0 ** -10)).all()
    assert (v.abs() <= 448 * s).all()


def test_oracle_rmsnorm_gradient_is_autograds():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 37, generator=g, dtype=Q.F64, requires_grad=True)
    w = torch.randn(37, generator=g, dtype=Q.F64, requires_grad=True)
    dy = torch.randn(5, 37, generator=g, dtype=Q.F64)
    y, _ = Q.rmsnorm(x, w, 1e-6)
    y.backward(dy)
    dx, dw = Q.rmsnorm_grad(x.detach(), w.detach(), 1e-6, dy)
    assert (dx - x.grad).abs().max() < 1e-12 and (dw - w.grad).abs().max() < 1e-12
