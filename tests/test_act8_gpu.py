"""GPU tests of 8-bit activation checkpoints and the RMSNorm that reads them, against the 64-bit oracle."""
import math

import pytest
import torch

import operator_oracle as Q

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def device():
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    torch.cuda.set_device(0)


def activations(rows, cols, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    size = torch.exp(torch.randn(cols, generator=g))
    return (torch.randn(rows, cols, generator=g) * size).to(Q.DTYPES[dtype])


def store(pkg, x, pad=0, offset=0, cpad=0, coffset=0):
    """(codes, scales) on the device, guards checked."""
    rows, cols = x.shape
    xb = Q.Rows(x, pad, offset)
    cb = Q.Rows(torch.full((rows, cols), 0x33, dtype=torch.uint8), cpad, coffset)
    sb = Q.Rows(torch.full((rows, pkg.act8_blocks(cols)), 0x33, dtype=torch.uint8), 0, 3)
    dt = {torch.float16: pkg.F16, torch.bfloat16: pkg.BF16, torch.float32: pkg.F32}[x.dtype]
    pkg.act8_store(xb.ptr, dt, rows, cols, cb.ptr, sb.ptr, xb.stride, cb.stride)
    torch.cuda.synchronize()
    assert xb.guards_intact() and cb.guards_intact() and sb.guards_intact()
    assert torch.equal(xb.get().view(xb.word), x.view(xb.word))
    return cb, sb


def load(pkg, cb, sb, dtype, pad=0, offset=0):
    ob = Q.Rows(torch.full((cb.rows, cb.cols), 3.0, dtype=Q.DTYPES[dtype]), pad, offset)
    pkg.act8_load(cb.ptr, sb.ptr, cb.rows, cb.cols, ob.ptr, Q.kind(pkg, dtype), cb.stride, ob.stride)
    torch.cuda.synchronize()
    assert ob.guards_intact()
    return ob.get()


def check_round_trip(pkg, x, out=None, pad=0, offset=0, cpad=0, coffset=0, opad=0, ooffset=0):
    codes, scales = Q.act8_encode(x)
    cb, sb = store(pkg, x, pad, offset, cpad, coffset)
    assert torch.equal(sb.get(), scales)
    got, want = cb.get(), codes.view(torch.uint8)
    nan = torch.isnan(codes.float())
    assert torch.equal(got[~nan], want[~nan])
    assert bool(((got[nan] & 0x7F) == 0x7F).all())
    name = out or {v: k for k, v in Q.DTYPES.items()}[x.dtype]
    most = float(torch.finfo(Q.DTYPES[name]).max)
    values = Q.act8_decode(codes, scales).clamp(-most, most).to(Q.DTYPES[name])     # NaN passes the clamp
    back = load(pkg, cb, sb, name, opad, ooffset)
    assert torch.equal(torch.isnan(back), nan)
    assert torch.equal(back[~nan].view(torch.int16 if back.element_size() == 2 else torch.int32),
                       values[~nan].view(torch.int16 if back.element_size() == 2 else torch.int32))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 127), (2, 128), (3, 129), (5, 255), (7, 1000), (33, 1024), (2, 4104), (300, 264), (1, 20001)])
def test_round_trip_sizes(pkg, dtype, rows, cols):
    check_round_trip(pkg, activations(rows, cols, dtype, rows + cols))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("pad,offset,cpad,coffset,opad,ooffset", [(1, 0, 0, 0, 0, 0), (0, 1, 0, 0, 0, 1), (8, 0, 8, 0, 8, 0), (0, 0, 3, 1, 0, 0),
                                                                 (24, 8, 8, 8, 0, 0), (0, 0, 0, 0, 5, 2), (4, 4, 0, 4, 4, 4)])
def test_round_trip_strides_and_offsets(pkg, dtype, pad, offset, cpad, coffset, opad, ooffset):
    for cols in (1, 200, 1024):
        check_round_trip(pkg, activations(9, cols, dtype, cols), None, pad, offset, cpad, coffset, opad, ooffset)


@pytest.mark.parametrize("source", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
def test_round_trip_between_types(pkg, source, out):
    check_round_trip(pkg, activations(20, 500, source, 3), out)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_round_trip_special_values(pkg, dtype):
    """Blocks of zeros, one value, the scale's border, ties, the type's largest and smallest values, inf and NaN."""
    t = Q.DTYPES[dtype]
    x = torch.zeros(16, 256, dtype=t)
    info = torch.finfo(t)
    x[0, 5] = 448.0
    x[1, 5] = float(torch.nextafter(torch.tensor(448.0, dtype=t), torch.tensor(1e4, dtype=t)))
    x[2, :128] = torch.arange(128).to(t) * 0.25
    x[3, 0] = info.max
    x[4, 0] = info.tiny
    x[5, 0] = info.tiny * 2.0 ** -3 if dtype != "f16" else 2.0 ** -24
    x[6, 3], x[6, 4], x[6, 5] = math.inf, -math.inf, 1.5
    x[7, 200], x[7, 201] = math.nan, -2.0
    x[8, :] = math.inf
    x[9, :] = -0.0
    x[10, :128] = torch.linspace(-448, 448, 128).to(t)
    x[11, 0], x[11, 1] = 448.0, 2.0 ** -9 * 0.5        # half of the smallest code: a tie to zero
    x[12, 0], x[12, 1], x[12, 2] = 448.0, 2.0 ** -9 * 1.5, 2.0 ** -6
    x[13, 0] = -info.max
    x[14, 0], x[14, 1] = 256.0, 17.0                   # 17 lies between 16 and 18
    x[15, 0], x[15, 1] = 256.0, 19.0
    check_round_trip(pkg, x)
    if dtype == "f32":
        check_round_trip(pkg, x, "f16")
        check_round_trip(pkg, x, "bf16")


def test_rows_past_32_bits(pkg):
    """Codes and values whose offsets pass 2^32."""
    rows, cols, stride = 3, 300, (1 << 31) + 64
    x = activations(rows, cols, "f16", 1)
    big, codes = torch.empty(rows * stride, dtype=torch.float16, device="cuda"), torch.empty(rows * stride, dtype=torch.uint8, device="cuda")
    scales = torch.empty(rows, 3, dtype=torch.uint8, device="cuda")
    for r in range(rows):
        big[r * stride:r * stride + cols] = x[r].cuda()
    pkg.act8_store(big.data_ptr(), pkg.F16, rows, cols, codes.data_ptr(), scales.data_ptr(), stride, stride)
    big.zero_()
    pkg.act8_load(codes.data_ptr(), scales.data_ptr(), rows, cols, big.data_ptr(), pkg.F16, stride, stride)
    w, y = torch.ones(cols, device="cuda"), torch.empty(rows * stride, dtype=torch.float16, device="cuda")
    pkg.act8_rmsnorm(codes.data_ptr(), scales.data_ptr(), rows, cols, w.data_ptr(), pkg.F32, 1e-6, y.data_ptr(), pkg.F16, None, stride, stride)
    torch.cuda.synchronize()
    cb, sb = store(pkg, x)
    assert torch.equal(torch.stack([big[r * stride:r * stride + cols] for r in range(rows)]).cpu(), load(pkg, cb, sb, "f16"))
    ref = torch.empty(rows, cols, dtype=torch.float16, device="cuda")
    pkg.act8_rmsnorm(cb.ptr, sb.ptr, rows, cols, w.data_ptr(), pkg.F32, 1e-6, ref.data_ptr(), pkg.F16)
    torch.cuda.synchronize()
    want, _ = Q.rmsnorm(Q.act8_decode(*Q.act8_encode(x)), torch.ones(cols), 1e-6)
    got = torch.stack([y[r * stride:r * stride + cols] for r in range(rows)]).cpu()
    for v in (got, ref.cpu()):
        assert ((v.to(Q.F64) - want).abs() <= want.abs() * (2.0 ** -20 + 2.0 ** -11) + 2.0 ** -25).all()


# ---- RMSNorm ------------------------------------------------------------------------

def norm_case(rows, cols, dtype, seed, wname="f32"):
    x = activations(rows, cols, dtype, seed)
    g = torch.Generator().manual_seed(seed + 77)
    w = (1 + 0.3 * torch.randn(cols, generator=g)).to(Q.DTYPES[wname])
    dy = (torch.randn(rows, cols, generator=g) * 0.1).to(Q.DTYPES[dtype])
    dres = (torch.randn(rows, cols, generator=g) * 0.1).to(Q.DTYPES[dtype])
    return x, w, dy, dres


def held(pkg, x, cpad=0, coffset=0):
    codes, scales = Q.act8_encode(x)
    cb, sb = Q.Rows(codes.view(torch.uint8), cpad, coffset), Q.Rows(scales)
    return cb, sb, Q.act8_decode(codes, scales)


def sum_error(n):
    """A sum of n squares or products in FP32, 32 or more partial sums: (n / 32 + 16) roundings of 2^-24 each."""
    return (n / 32 + 16) * 2.0 ** -24


def check_norm(pkg, rows, cols, dtype, seed=0, wname="f32", eps=1e-6, cpad=0, coffset=0, ypad=0, yoffset=0):
    x, w, _, _ = norm_case(rows, cols, dtype, seed, wname)
    cb, sb, v = held(pkg, x, cpad, coffset)
    yb, wb = Q.Rows(torch.full_like(x, 3.0), ypad, yoffset), w.cuda()
    rstd = torch.full((rows,), 7.0, device="cuda")
    pkg.act8_rmsnorm(cb.ptr, sb.ptr, rows, cols, wb.data_ptr(), Q.kind(pkg, wname), eps, yb.ptr, Q.kind(pkg, dtype), rstd.data_ptr(), cb.stride, yb.stride)
    torch.cuda.synchronize()
    assert yb.guards_intact() and cb.guards_intact()
    want, want_r = Q.rmsnorm(v, w, float(torch.tensor(eps, dtype=torch.float32)))
    rel = sum_error(cols) / 2 + 2.0 ** -21
    assert ((rstd.cpu().to(Q.F64) - want_r).abs() <= want_r * rel).all()
    assert ((yb.get().to(Q.F64) - want).abs() <= want.abs() * rel * 1.01 + Q.rounding(want * (1 + rel), x.dtype)).all()


def check_norm_grad(pkg, rows, cols, dtype, seed=0, wname="f32", eps=1e-6, residual=True, cpad=0, coffset=0, pad=0, offset=0, dpad=0, doffset=0,
                    dw=True, accumulate=False, in_place=None):
    x, w, dy, dres = norm_case(rows, cols, dtype, seed, wname)
    cb, sb, v = held(pkg, x, cpad, coffset)
    db, rb = Q.Rows(dy, pad, offset), Q.Rows(dres, dpad, doffset) if residual else None
    ob = {"dy": db, "dres": rb, None: Q.Rows(torch.full_like(x, 3.0), dpad, doffset)}[in_place]
    wb, dwb = w.cuda(), torch.full((cols,), 0.25, device="cuda")
    need = pkg.act8_rmsnorm_grad_workspace(rows, cols)
    ws = torch.full((need + 64,), 0x5A, dtype=torch.uint8, device="cuda")
    pkg.act8_rmsnorm_grad(cb.ptr, sb.ptr, rows, cols, wb.data_ptr(), Q.kind(pkg, wname), eps, db.ptr, Q.kind(pkg, dtype), ob.ptr,
                          dwb.data_ptr() if dw else None, ws.data_ptr() if dw else None, need if dw else 0, rb.ptr if residual else None, cb.stride,
                          db.stride, rb.stride if residual else 0, ob.stride, pkg.ACT8_ACCUMULATE if accumulate else 0)
    torch.cuda.synchronize()
    assert ob.guards_intact() and db.guards_intact() and cb.guards_intact()
    if dw:
        assert bool((ws[need:] == 0x5A).all())
    eps = float(torch.tensor(eps, dtype=torch.float32))
    want, want_w = Q.rmsnorm_grad(v, w, eps, dy, dres if residual else None)
    rstd = 1 / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    g = (dy.to(Q.F64) * w.to(Q.F64)).abs()
    # the two terms of dx are off by the relative error of their factors; the mean of g x by that of a sum of their sizes
    rel = sum_error(cols) * 1.5 + 2.0 ** -20
    parts = rstd * (g + v.abs() * rstd ** 2 * (g * v.abs()).mean(1, keepdim=True)) + (dres.to(Q.F64).abs() if residual else 0)
    assert ((ob.get().to(Q.F64) - want).abs() <= parts * rel * 1.01 + Q.rounding(want.abs() + parts * rel, x.dtype)).all()
    if dw:
        size = (dy.to(Q.F64) * v * rstd).abs().sum(0)
        base = 0.25 if accumulate else 0.0
        tol = size * ((rows / 32 + 330) * 2.0 ** -24 + sum_error(cols) + 2.0 ** -20) + (want_w.abs() + base) * 2.0 ** -23
        assert ((dwb.cpu().to(Q.F64) - want_w - base).abs() <= tol).all()
    else:
        assert bool((dwb == 0.25).all())


WIDTHS = [1, 7, 64, 128, 130, 1000, 1024, 1001, 2048, 4096, 5120, 8192, 8200, 20000]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("cols", WIDTHS)
def test_norm_widths(pkg, dtype, cols):
    for rows in (1, 5):
        check_norm(pkg, rows, cols, dtype, cols)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("cols", WIDTHS)
def test_norm_grad_widths(pkg, dtype, cols):
    for rows, residual in ((1, True), (6, False)):
        check_norm_grad(pkg, rows, cols, dtype, cols, residual=residual)


@pytest.mark.parametrize("rows,cols", [(1000, 128), (2500, 256), (700, 1024), (400, 2048), (150, 4096), (3000, 40)])
def test_norm_many_rows(pkg, rows, cols):
    check_norm(pkg, rows, cols, "bf16", rows)
    check_norm_grad(pkg, rows, cols, "bf16", rows)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(5000, 77), (1300, 500), (700, 513), (650, 1001), (400, 1501), (310, 4001), (300, 6001), (160, 8191)])
def test_norm_many_rows_that_start_anywhere(pkg, rows, cols, dtype):
    """More rows than CTAs, at each width that has threads of its own: the row ahead, and the sums over a CTA's rows."""
    check_norm(pkg, rows, cols, dtype, rows)
    check_norm_grad(pkg, rows, cols, dtype, rows, residual=dtype == "bf16")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("cpad,coffset,pad,offset,dpad,doffset", [(0, 0, 3, 1, 0, 0), (1, 1, 0, 0, 0, 0), (16, 0, 8, 0, 16, 0), (8, 8, 8, 8, 8, 8), (0, 0, 0, 0, 1, 3), (0, 4, 4, 4, 4, 4)])
def test_norm_strides_and_offsets(pkg, dtype, cpad, coffset, pad, offset, dpad, doffset):
    for cols in (24, 640, 1024):
        check_norm(pkg, 11, cols, dtype, 1, cpad=cpad, coffset=coffset, ypad=dpad, yoffset=doffset)
        check_norm_grad(pkg, 11, cols, dtype, 1, cpad=cpad, coffset=coffset, pad=pad, offset=offset, dpad=dpad, doffset=doffset)


@pytest.mark.parametrize("wname", ["f16", "bf16", "f32"])
def test_norm_weight_types(pkg, wname):
    for cols in (300, 1024):
        check_norm(pkg, 5, cols, "bf16", 2, wname)
        check_norm_grad(pkg, 5, cols, "bf16", 2, wname)


@pytest.mark.parametrize("in_place", ["dy", "dres"])
@pytest.mark.parametrize("cols", [77, 1024, 4096])
def test_norm_grad_in_place(pkg, in_place, cols):
    check_norm_grad(pkg, 40, cols, "f16", 3, in_place=in_place)


def test_norm_grad_accumulates_and_can_leave_the_weight_out(pkg):
    for cols in (90, 1024):
        check_norm_grad(pkg, 50, cols, "bf16", 4, accumulate=True)
        check_norm_grad(pkg, 50, cols, "bf16", 4, dw=False)


def test_norm_of_zero_rows_and_zero_values(pkg):
    """No rows: dweight is zero, or stays when it accumulates.  Rows of zeros: finite with eps, as the formula is."""
    dw = torch.full((64,), 5.0, device="cuda")
    w = torch.ones(64, device="cuda")
    pkg.act8_rmsnorm_grad(None, None, 0, 64, w.data_ptr(), pkg.F32, 1e-6, None, pkg.F16, None, dw.data_ptr(), None, 0, flags=pkg.ACT8_ACCUMULATE)
    torch.cuda.synchronize()
    assert bool((dw == 5).all())
    pkg.act8_rmsnorm_grad(None, None, 0, 64, w.data_ptr(), pkg.F32, 1e-6, None, pkg.F16, None, dw.data_ptr(), None, 0)
    torch.cuda.synchronize()
    assert bool((dw == 0).all())
    x = torch.zeros(3, 64, dtype=torch.float16)
    cb, sb = store(pkg, x)
    y, rstd = torch.empty(3, 64, dtype=torch.float16, device="cuda"), torch.empty(3, device="cuda")
    pkg.act8_rmsnorm(cb.ptr, sb.ptr, 3, 64, w.data_ptr(), pkg.F32, 1e-6, y.data_ptr(), pkg.F16, rstd.data_ptr())
    torch.cuda.synchronize()
    assert bool((y == 0).all()) and ((rstd.cpu() - 1000).abs() < 1e-2).all()


def test_norm_nan_stays_in_its_row(pkg):
    x, w, dy, _ = norm_case(6, 1024, "f16", 5)
    x[2, 100] = math.inf
    cb, sb = store(pkg, x)
    dyb, wb, dx, dw = dy.cuda(), w.cuda(), torch.empty(6, 1024, dtype=torch.float16, device="cuda"), torch.empty(1024, device="cuda")
    ws = torch.empty(pkg.act8_rmsnorm_grad_workspace(6, 1024), dtype=torch.uint8, device="cuda")
    pkg.act8_rmsnorm_grad(cb.ptr, sb.ptr, 6, 1024, wb.data_ptr(), pkg.F32, 1e-6, dyb.data_ptr(), pkg.F16, dx.data_ptr(), dw.data_ptr(), ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    bad = torch.isnan(dx)
    assert bool(bad[2].all()) and not bool(bad[[0, 1, 3, 4, 5]].any()) and bool(torch.isnan(dw).all())


def test_norm_grad_is_the_difference_quotient(pkg):
    """Differences of the forward call's own output over the weight, which it is linear in: exact but for the two
    outputs' errors (2^-20 relative) over the step."""
    rows, cols = 3, 40
    x, w, dy, _ = norm_case(rows, cols, "f32", 6)
    cb, sb, _ = held(pkg, x)
    wb, dyb = w.cuda(), dy.cuda()
    dx, dw = torch.empty(rows, cols, device="cuda"), torch.empty(cols, device="cuda")
    ws = torch.empty(pkg.act8_rmsnorm_grad_workspace(rows, cols), dtype=torch.uint8, device="cuda")
    pkg.act8_rmsnorm_grad(cb.ptr, sb.ptr, rows, cols, wb.data_ptr(), pkg.F32, 1e-6, dyb.data_ptr(), pkg.F32, dx.data_ptr(), dw.data_ptr(), ws.data_ptr(), ws.numel())

    def loss(weight):
        y = torch.empty(rows, cols, device="cuda")
        pkg.act8_rmsnorm(cb.ptr, sb.ptr, rows, cols, weight.data_ptr(), pkg.F32, 1e-6, y.data_ptr(), pkg.F32)
        return (y.double() * dyb.double())

    for j in range(cols):
        up, down = wb.clone(), wb.clone()
        up[j] += 0.5
        down[j] -= 0.5
        a, b = loss(up), loss(down)
        step = float(up[j]) - float(down[j])
        tol = float((a.abs() + b.abs())[:, j].sum()) * 2.0 ** -19 / step
        assert abs(float((a - b).sum()) / step - float(dw[j])) <= tol + abs(float(dw[j])) * 2.0 ** -20


def test_two_streams_and_a_graph(pkg):
    """Two backward calls at once with a workspace each, then one of them captured and replayed."""
    rows, cols = 600, 1024
    sets = []
    for k in range(2):
        x, w, dy, _ = norm_case(rows, cols, "bf16", k)
        cb, sb, _ = held(pkg, x)
        sets.append(dict(cb=cb, sb=sb, w=w.cuda(), dy=dy.cuda(), ws=torch.empty(pkg.act8_rmsnorm_grad_workspace(rows, cols), dtype=torch.uint8, device="cuda")))

    def call(s, dx, dw, stream):
        pkg.act8_rmsnorm_grad(s["cb"].ptr, s["sb"].ptr, rows, cols, s["w"].data_ptr(), pkg.F32, 1e-6, s["dy"].data_ptr(), pkg.BF16, dx.data_ptr(),
                              dw.data_ptr(), s["ws"].data_ptr(), s["ws"].numel(), stream=stream)

    out = [[(torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda"), torch.empty(cols, device="cuda")) for _ in range(2)] for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for k in range(2):
        call(sets[k], *out[0][k], None)
    torch.cuda.synchronize()
    for _ in range(4):
        for k in range(2):
            call(sets[k], *out[1][k], streams[k].cuda_stream)
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(p, q) for p, q in zip(out[0][k], out[1][k]))
    dx, dw = torch.empty_like(out[0][0][0]), torch.empty(cols, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(sets[0], dx, dw, torch.cuda.current_stream().cuda_stream)
    sets[0]["dy"].mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(dw, 2 * out[0][0][1]) and torch.equal(dx, 2 * out[0][0][0])
