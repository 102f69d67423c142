"""8-bit checkpoints on the CPU: refusals beyond those of test_act8.py."""
import pytest
import torch

A, ROOM = 1 << 20, 1 << 16


def refuse(pkg, text, call, *args, **kwargs):
    with pytest.raises(pkg.RlcuError) as e:
        call(*args, **kwargs)
    assert e.value.code == pkg.ERR_INVALID and text in str(e.value), str(e.value)


def taken(pkg, call, *args, **kwargs):
    """The arguments pass; without a GPU the call ends there."""
    if torch.cuda.is_available():
        return
    with pytest.raises(pkg.RlcuError) as e:
        call(*args, **kwargs)
    assert e.value.code == pkg.ERR_CUDA, str(e.value)


def places(n):
    return [A + k * ROOM for k in range(n)]


def test_scales_over_values_or_codes_are_refused(pkg):
    x, codes, scales = places(3)
    rows, cols = 3, 300                               # 9 scales; FP16 rows of 600 bytes, codes of 300 in 512

    def store(scales=scales):
        pkg.act8_store(x, pkg.F16, rows, cols, codes, scales, 320, 512)

    def load(scales=scales):
        pkg.act8_load(codes, scales, rows, cols, x, pkg.F16, 512, 320)

    for f in (store, load):
        for at in (x, x - 8, x + 599, x + 632, x + 2 * 640 + 599):
            refuse(pkg, "overlap", f, scales=at)
        taken(pkg, f, scales=x + 600)                 # 40 bytes lie between two rows
        taken(pkg, f, scales=x + 631)
    for at in (codes, codes - 8, codes + 299, codes + 504, codes + 2 * 512 + 299):
        refuse(pkg, "overlap", store, scales=at)
    taken(pkg, store, scales=codes + 300)


def test_norms_that_write_over_what_they_read_are_refused(pkg):
    codes, scales, w, y, rstd = places(5)

    def forward(scales=scales, w=w, rstd=rstd):
        pkg.act8_rmsnorm(codes, scales, 4, 128, w, pkg.F32, 1e-6, y, pkg.BF16, rstd)

    for name, size in (("scales", 4), ("w", 512), ("rstd", 16)):
        for at in (y, y + 1020, y - size + 4):
            refuse(pkg, "overlap", forward, **{name: at})
    for at in (codes, codes + 508, scales, w + 508, w - 12):
        refuse(pkg, "overlap", forward, rstd=at)


def test_norm_gradients_that_write_over_what_they_read_are_refused(pkg):
    codes, scales, w, dy, dres, dx, dw, ws = places(8)
    need = pkg.act8_rmsnorm_grad_workspace(4, 128)

    def backward(scales=scales, w=w, dw=dw, ws=ws):
        pkg.act8_rmsnorm_grad(codes, scales, 4, 128, w, pkg.F32, 1e-6, dy, pkg.F16, dx, dw, ws, need, dres)

    for name, size in (("scales", 4), ("w", 512), ("dw", 512), ("ws", need)):
        for at in (dx, dx + 1008, dx - size + 16 & ~15 if size > 16 else dx):
            refuse(pkg, "overlap", backward, **{name: at})
    for at in (codes, codes + 496, scales, w, w + 496, dy, dy + 1008, dres, dres + 1008):
        refuse(pkg, "overlap", backward, dw=at)
        refuse(pkg, "overlap", backward, ws=at)
    refuse(pkg, "overlap", backward, dw=ws)
    refuse(pkg, "overlap", backward, dw=ws + need - 4)
    taken(pkg, backward, dw=ws + need)
    taken(pkg, backward, dw=None, ws=dx)              # without dweight there is no workspace


def test_matrices_beside_each_other_in_one_buffer(pkg):
    """dx beside dy, codes beside values: rows of one buffer, each with its part of them."""
    x, scales, w, dw, ws = places(5)
    need = pkg.act8_rmsnorm_grad_workspace(5, 16)

    def backward(dx, dres=None):
        pkg.act8_rmsnorm_grad(x + ROOM // 2, scales, 5, 16, w, pkg.F32, 1e-6, x, pkg.F16, dx, dw, ws, need, dres, dy_stride=64, dresidual_stride=64,
                              dx_stride=64)

    def store(codes):
        pkg.act8_store(x, pkg.F16, 5, 16, codes, scales, 64, 128)

    for shift in range(-6 * 128, 6 * 128 + 1, 2):
        meets = any(abs(shift + 128 * k) < 32 for k in range(-4, 5))
        if shift and meets:
            refuse(pkg, "overlap", backward, x + shift)
            refuse(pkg, "overlap", backward, x + 64 * 128, x + 64 * 128 + shift)
        else:
            taken(pkg, backward, x + shift)
            taken(pkg, backward, x + 64 * 128, x + 64 * 128 + shift)
        if any(-16 < shift + 128 * k < 32 for k in range(-4, 5)):
            refuse(pkg, "overlap", store, x + shift)
        else:
            taken(pkg, store, x + shift)
