"""GPU tests of the losses against the 64-bit oracle: element types, vocabularies from one entry up, odd sizes,
strides and offsets, masked logits, rows that take no part, in-place gradients, streams, graphs, and a run of
loss -> gradient statistics -> optimizer step."""
import ctypes as C
import math

import pytest
import torch

import operator_oracle as Q

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def device():
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    torch.cuda.set_device(0)


def scaler_of(pkg, scale):
    host = pkg.ScalerState(scale, 0, 0, 0, 1000, 0.9, 0.999, 0.0)
    return torch.frombuffer(bytearray(bytes(host)), dtype=torch.uint8).cuda()


def gaussian(rows, cols, dtype, seed, size=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, cols, generator=g) * size).to(Q.DTYPES[dtype])


def targets_of(rows, vocab, seed, ignored=0.2):
    g = torch.Generator().manual_seed(seed + 1)
    y = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32)
    skip = torch.rand(rows, generator=g) < ignored
    return torch.where(skip, torch.full_like(y, -100), y)


def run_logprob(pkg, z, y, it, coef=None, scaler=None, pad=0, offset=0, gpad=0, goffset=0, stream=None):
    """(logp, lse, grad or None); guards checked."""
    rows, vocab = z.shape
    zb, yb = Q.Rows(z, pad, offset), y.cuda()
    logp, lse = torch.full((rows,), 7.0, device="cuda"), torch.full((rows,), 7.0, device="cuda")
    dt = {torch.float16: pkg.F16, torch.bfloat16: pkg.BF16, torch.float32: pkg.F32}[z.dtype]
    pkg.token_logprob(zb.ptr, dt, rows, vocab, yb.data_ptr(), logp.data_ptr(), lse.data_ptr(), zb.stride, it, stream)
    grad = None
    if coef is not None:
        gb = Q.Rows(torch.full_like(z, 3.0), gpad, goffset)
        co = coef.cuda()
        pkg.token_logprob_grad(zb.ptr, dt, rows, vocab, yb.data_ptr(), lse.data_ptr(), co.data_ptr(), gb.ptr, zb.stride, gb.stride,
                               it, scaler.data_ptr() if scaler is not None else None, stream)
        torch.cuda.synchronize()
        assert gb.guards_intact()
        grad = gb.get()
    torch.cuda.synchronize()
    assert zb.guards_intact()
    assert torch.equal(zb.get().view(zb.word), z.view(zb.word))
    return logp.cpu(), lse.cpu(), grad


def close(got, want, tol, what):
    got, want = got.to(Q.F64), want.to(Q.F64)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{what}: infinities differ"
    off = (got - want).abs()[fine]
    tol = torch.broadcast_to(torch.as_tensor(tol, dtype=Q.F64), want.shape)[fine]
    assert bool((off <= tol).all()), f"{what}: off by {float((off - tol).max()):.3g} more than {float(tol[(off - tol).argmax()]):.3g}"


def check_logprob(pkg, z, y, it=1.0, scale=None, seed=0, **where):
    rows, vocab = z.shape
    g = torch.Generator().manual_seed(seed + 5)
    coef = torch.randn(rows, generator=g)
    if rows > 3:
        coef[1] = 0.0
    scaler = scaler_of(pkg, scale) if scale else None
    logp, lse, grad = run_logprob(pkg, z, y, it, coef, scaler, **where)
    it = float(torch.tensor(it, dtype=torch.float32))
    want, want_lse, p, takes = Q.logprob(z, y, it)
    e = Q.logprob_error(z, y, it)
    close(logp, want, e + want.abs().nan_to_num(0, 0, 0) * 2.0 ** -22, "logp")
    close(lse, want_lse, e + want_lse.abs().nan_to_num(0, 0, 0) * 2.0 ** -22, "lse")
    factor = it * (scale or 1.0)
    want_grad = Q.logits_grad(p, y, takes, coef, factor)
    # a probability carries the error of the FP32 lse it is taken from and its own; 1 - p the same in absolute terms
    size = (coef.to(Q.F64).abs() * factor)[:, None]
    rel = (2 * e + want_lse.abs().nan_to_num(0, 0, 0) * 2.0 ** -22)[:, None]
    hot = torch.zeros_like(p)
    inside = torch.nonzero(takes)[:, 0]
    hot[inside, y.long()[inside]] = 1.0
    # exponentials below 2^-126 are flushed to zero; they are then divided by a sum of at least 1/2
    tol = size * 2.0 ** -125 + size * (p.nan_to_num(0) + hot * 2.0 ** -20) * rel + want_grad.abs().nan_to_num(0) * 2.0 ** -22 + hot * size * 2.0 ** -23
    tol = torch.where(takes[:, None], tol, torch.zeros_like(tol))
    close(grad, want_grad, tol * 1.01 + Q.rounding(want_grad.nan_to_num(0), z.dtype), "grad")
    dead = ~takes | (coef == 0)
    assert bool((grad[dead] == 0).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 7), (4, 8), (2, 129), (7, 1000), (3, 4099), (5, 32000), (2, 50001), (1, 151936), (3, 262145)])
def test_logprob_sizes(pkg, dtype, rows, vocab):
    check_logprob(pkg, gaussian(rows, vocab, dtype, rows + vocab), targets_of(rows, vocab, vocab), seed=vocab)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("pad,offset,gpad,goffset", [(3, 0, 3, 0), (0, 1, 0, 1), (5, 3, 5, 3), (8, 0, 0, 0), (1, 2, 4, 5), (0, 0, 1, 0), (16, 0, 16, 8)])
def test_logprob_strides_and_offsets(pkg, dtype, pad, offset, gpad, goffset):
    for vocab in (1, 5, 1003, 40007):
        check_logprob(pkg, gaussian(6, vocab, dtype, 3), targets_of(6, vocab, 3), pad=pad, offset=offset, gpad=gpad, goffset=goffset)


@pytest.mark.parametrize("dtype,it", [("f16", 0.5), ("bf16", 1.7), ("f32", 1.0 / 0.7), ("f32", 10.0)])
def test_logprob_temperature_and_loss_scale(pkg, dtype, it):
    check_logprob(pkg, gaussian(9, 3001, dtype, 8), targets_of(9, 3001, 8), it=it, scale=256.0)


@pytest.mark.parametrize("rows,vocab", [(700, 1536), (1200, 33), (160, 32000), (75, 151936)])
def test_logprob_many_rows(pkg, rows, vocab):
    check_logprob(pkg, gaussian(rows, vocab, "bf16", rows), targets_of(rows, vocab, rows))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("vocab", [40, 5003, 70000])
def test_logprob_masked_logits(pkg, dtype, vocab):
    z = gaussian(12, vocab, dtype, 4)
    low = torch.finfo(z.dtype).min
    y = torch.zeros(12, dtype=torch.int32) + 3
    z[0, 10:] = -math.inf                         # a masked tail
    z[1, :] = -math.inf
    z[1, 3] = 1.0                                 # one token left: logp 0
    z[2, :] = -math.inf
    z[2, 4] = 1.0                                 # one token left, and it is not the target
    z[3, :] = -math.inf                           # nothing left
    z[4, 20:] = low                               # masked with the type's lowest value
    z[5, :] = low
    z[6, 5] = math.nan
    z[7, 7] = math.inf
    z[8, :] = math.nan
    y[8] = -1                                     # a row of NaN that takes no part
    z[9, :] = -40.0
    z[9, 9] = 40.0                                # a confident row
    z[10, 3] = 30.0                               # ... whose target it is
    y[11] = vocab                                 # a target behind the vocabulary takes no part
    if dtype == "f16":                            # FP16's lowest value is a logit like any other
        z[5, 3] = 0.0
    check_logprob(pkg, z, y)


@pytest.mark.parametrize("rows,vocab,dtype", [(6000, 600, "f16"), (9001, 515, "f32"), (2500, 9000, "bf16"), (1500, 16411, "f16"), (260, 151936, "bf16")])
def test_rows_by_the_thousand(pkg, rows, vocab, dtype):
    """More rows than fit the GPU at once: CTAs and clusters take over row after row, each exactly once."""
    z, y = gaussian(rows, vocab, dtype, rows), targets_of(rows, vocab, rows)
    check_logprob(pkg, z, y)
    check_policy(pkg, z, y, scale=64.0)
    pkg.losses_check()


def test_logprob_huge_logits_do_not_vanish(pkg):
    z = torch.full((2, 64), 3.0e38, dtype=torch.float32)
    logp, _, _ = run_logprob(pkg, z, torch.tensor([0, 1], dtype=torch.int32), 1.0)
    assert bool(torch.isnan(logp).all())          # their product with log2 e is beyond FP32: said, not hidden


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("vocab", [11, 5001, 151936])
def test_gradient_in_place(pkg, dtype, vocab):
    z, y = gaussian(5, vocab, dtype, 1), targets_of(5, vocab, 1)
    coef = torch.linspace(-1, 1, 5)
    _, _, apart = run_logprob(pkg, z, y, 1.0, coef)
    zb, yb, co = Q.Rows(z), y.cuda(), coef.cuda()
    logp, lse = torch.empty(5, device="cuda"), torch.empty(5, device="cuda")
    dt = Q.kind(pkg, dtype)
    pkg.token_logprob(zb.ptr, dt, 5, vocab, yb.data_ptr(), logp.data_ptr(), lse.data_ptr())
    pkg.token_logprob_grad(zb.ptr, dt, 5, vocab, yb.data_ptr(), lse.data_ptr(), co.data_ptr(), zb.ptr)
    torch.cuda.synchronize()
    assert torch.equal(zb.get(), apart) and zb.guards_intact()


def test_gradient_is_the_difference_quotient(pkg):
    """Central differences of the kernel's own log-probability, step 1/16: off by at most h^2/6 times the third
    derivative (under 1/6 for a softmax) plus the two values' errors over the step."""
    vocab, h = 23, 1 / 16
    z, y = gaussian(1, vocab, "f32", 2), torch.tensor([4], dtype=torch.int32)
    _, _, grad = run_logprob(pkg, z, y, 1.0, torch.ones(1))
    up = z.repeat(vocab, 1) + h * torch.eye(vocab)
    down = z.repeat(vocab, 1) - h * torch.eye(vocab)
    ys = y.repeat(vocab)
    a, b = run_logprob(pkg, up, ys, 1.0)[0], run_logprob(pkg, down, ys, 1.0)[0]
    e = float(Q.logprob_error(up, ys, 1.0).max()) + 2.0 ** -20
    assert ((a - b) / (2 * h) - grad[0]).abs().max() <= h * h / 36 + e / h


def test_rows_past_32_bits(pkg):
    """Rows whose element offsets pass 2^32, logits and gradient."""
    vocab, stride, rows = 1000, (1 << 31) + 40, 3
    z, y = gaussian(rows, vocab, "f16", 3), torch.tensor([5, 999, 0], dtype=torch.int32)
    big = torch.empty(rows * stride, dtype=torch.float16, device="cuda")
    out = torch.empty(rows * stride, dtype=torch.float16, device="cuda")
    for r in range(rows):
        big[r * stride:r * stride + vocab] = z[r].cuda()
    logp, lse, co, yb = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.ones(rows, device="cuda"), y.cuda()
    pkg.token_logprob(big.data_ptr(), pkg.F16, rows, vocab, yb.data_ptr(), logp.data_ptr(), lse.data_ptr(), stride)
    pkg.token_logprob_grad(big.data_ptr(), pkg.F16, rows, vocab, yb.data_ptr(), lse.data_ptr(), co.data_ptr(), out.data_ptr(), stride, stride)
    torch.cuda.synchronize()
    want = run_logprob(pkg, z, y, 1.0, torch.ones(rows))
    assert torch.equal(logp.cpu(), want[0])
    got = torch.stack([out[r * stride:r * stride + vocab] for r in range(rows)]).cpu()
    assert torch.equal(got, want[2])


# ---- policy loss ------------------------------------------------------------------

def off_the_borders(delta, clip_low, clip_high, dual):
    """Log ratios are kept 1e-3 away from where a clip begins: which side such a token falls on is a matter of its last
    bits, and the gradient jumps there."""
    for border in [math.log(b) for b in (1 - clip_low, 1 + clip_high, dual) if 0 < b < math.inf]:
        delta = torch.where((delta - border).abs() < 1e-3, torch.full_like(delta, border - 5e-3), delta)
    return delta


def policy_case(z, y, it, seed, clip, old=True, ref=True, ignored=0.2):
    rows = z.shape[0]
    g = torch.Generator().manual_seed(seed + 9)
    logp, _, _, takes = Q.logprob(z, y, it)
    delta = off_the_borders(torch.randn(rows, generator=g) * 0.6, *clip)
    a, w = torch.randn(rows, generator=g), torch.rand(rows, generator=g) + 0.1
    w[torch.rand(rows, generator=g) < ignored] = 0.0
    old = (logp - delta).float() if old else None
    ref = (logp + torch.randn(rows, generator=g) * 0.5).float() if ref else None
    return a, w, old, ref


def stat_of(kind, buffer):
    return kind.from_buffer_copy(buffer.cpu().numpy().tobytes())


def check_policy(pkg, z, y, clip=(0.2, 0.28, 3.0), kl=0.1, kl_kind=3, it=1.0, scale=None, seed=0, on_policy=False, pad=0, offset=0,
                 gpad=0, goffset=0, stream=None):
    rows, vocab = z.shape
    it32 = float(torch.tensor(it, dtype=torch.float32))
    a, w, old, ref = policy_case(z, y, it32, seed, clip, not on_policy, kl != 0)
    hp = pkg.policy_hparams(*clip, kl, kl_kind)
    zb, gb = Q.Rows(z, pad, offset), Q.Rows(torch.full_like(z, 3.0), gpad, goffset)
    on = lambda t: None if t is None else t.cuda()  # noqa: E731
    yb, ab, wb, ob, rb = on(y), on(a), on(w), on(old), on(ref)
    logp, coef = torch.full((rows,), 7.0, device="cuda"), torch.full((rows,), 7.0, device="cuda")
    stat, stat2 = (torch.full((8,), 0x7FC00000, dtype=torch.int32, device="cuda") for _ in range(2))
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    scaler = scaler_of(pkg, scale) if scale else None
    dt = {torch.float16: pkg.F16, torch.bfloat16: pkg.BF16, torch.float32: pkg.F32}[z.dtype]
    pkg.policy_loss(zb.ptr, dt, rows, vocab, at(yb), at(ab), at(wb), hp, at(logp), gb.ptr, at(stat), at(ob), at(rb), zb.stride, gb.stride,
                    it, at(scaler), stream=stream)
    # the loss alone, on the log-probabilities of the first call
    valid = ((yb >= 0) & (yb < vocab)).float() * wb
    pkg.policy_loss_logp(at(logp), rows, at(ab), at(valid), hp, at(stat2), at(coef), at(ob), at(rb), stream=stream)
    torch.cuda.synchronize()
    assert zb.guards_intact() and gb.guards_intact()
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
    clip32, kl32 = [f32(c) for c in clip], f32(kl)
    want, _, p, takes = Q.logprob(z, y, it32, w != 0)
    e = Q.logprob_error(z, y, it32) + want.abs() * 2.0 ** -22
    close(logp.cpu(), want, e, "logp")
    per = Q.policy(want, old, ref, a, w, takes, *clip32, kl32, kl_kind)
    ce = Q.policy_error(e, old, ref, want, a, w, takes, kl32)
    close(coef.cpu(), per[2], ce, "coef")
    for s in (stat_of(pkg.PolicyStat, stat), stat_of(pkg.PolicyStat, stat2)):
        assert s.tokens == int(takes.sum()) and s.clipped == int(per[3].sum())
        wd = w.to(Q.F64) * takes
        wl, wk = wd * per[0], wd * per[1]
        # l and k are off by no more than coef (their slope) times the log-probability's error, and a few roundings
        tol = float(ce.sum()) + float(wl.abs().sum() + wk.abs().sum()) * 2.0 ** -20
        k_tol = float((wd * (torch.exp((ref.to(Q.F64) - want) * takes) + 1 + (ref.to(Q.F64) - want).abs()) * (e + 2.0 ** -20)).sum()) if kl else 0.0
        assert abs(s.policy - float(wl.sum())) <= tol, (s.policy, float(wl.sum()))
        assert abs(s.kl - float(wk.sum())) <= k_tol + tol, (s.kl, float(wk.sum()))
        assert abs(s.loss - float((wl + kl32 * wk).sum())) <= tol + k_tol
        assert abs(s.weight - float(wd.sum())) <= float(wd.sum()) * 2.0 ** -22
    factor = it32 * (scale or 1.0)
    want_grad = Q.logits_grad(p, y, takes, per[2], factor)
    hot = torch.zeros_like(p)
    inside = torch.nonzero(takes)[:, 0]
    hot[inside, y.long()[inside]] = 1.0
    share = (hot - p).abs()
    # the row's factor is off by ce; a probability by 2e of itself, which is what 1 - p is off by in absolute terms
    # exponentials below 2^-126 are flushed to zero; they are then divided by a sum of at least 1/2
    tol = factor * ((per[2].abs() + ce)[:, None] * 2.0 ** -125 + ce[:, None] * share + (per[2].abs() + ce)[:, None] * p * (2 * e)[:, None]) + want_grad.abs() * 2.0 ** -21
    tol = torch.where(takes[:, None], tol, torch.zeros_like(tol))
    close(gb.get(), want_grad, tol * 1.01 + Q.rounding(want_grad, z.dtype), "grad")
    assert bool((gb.get()[~takes] == 0).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (6, 5), (9, 1000), (40, 4097), (3, 32000), (33, 50001), (6, 151936), (300, 20000), (2, 262145), (1, 700001)])
def test_policy_sizes(pkg, dtype, rows, vocab):
    check_policy(pkg, gaussian(rows, vocab, dtype, rows + vocab), targets_of(rows, vocab, vocab), seed=rows, scale=1024.0)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("pad,offset,gpad,goffset", [(3, 0, 3, 0), (0, 1, 0, 1), (8, 0, 0, 0), (1, 2, 4, 5), (16, 0, 16, 8)])
def test_policy_strides_and_offsets(pkg, dtype, pad, offset, gpad, goffset):
    for vocab in (3, 1003, 40007):
        check_policy(pkg, gaussian(6, vocab, dtype, 3), targets_of(6, vocab, 3), pad=pad, offset=offset, gpad=gpad, goffset=goffset)


@pytest.mark.parametrize("kl,kl_kind", [(0.0, 3), (0.1, 1), (0.1, 2), (0.04, 3), (-0.1, 3)])
@pytest.mark.parametrize("clip", [(0.2, 0.2, 0.0), (0.2, 0.28, 3.0), (1.0, math.inf, 0.0)])
@pytest.mark.parametrize("on_policy", [False, True])
def test_policy_terms(pkg, kl, kl_kind, clip, on_policy):
    check_policy(pkg, gaussian(300, 97, "f32", 4), targets_of(300, 97, 4), clip, kl, kl_kind, it=1.3, on_policy=on_policy)


@pytest.mark.parametrize("tokens", [1, 31, 1024, 1025, 5000, 100003])
def test_policy_loss_of_many_tokens_accumulates_and_repeats(pkg, tokens):
    """The record over micro-batches is the record over the whole, and the same call gives the same bits."""
    g = torch.Generator().manual_seed(tokens)
    logp = -torch.rand(tokens, generator=g) * 3
    delta = off_the_borders(torch.randn(tokens, generator=g) * 0.3, 0.2, 0.28, 3.0)
    old, ref = logp - delta, logp + torch.randn(tokens, generator=g) * 0.2
    a, w = torch.randn(tokens, generator=g), (torch.rand(tokens, generator=g) < 0.7).float() / tokens
    hp = pkg.policy_hparams(0.2, 0.28, 3.0, 0.1)
    d = [t.cuda() for t in (logp, old, ref, a, w)]
    whole, again, parts = (torch.zeros(8, dtype=torch.int32, device="cuda") for _ in range(3))
    coef, coef2 = (torch.full((tokens,), 9.0, device="cuda") for _ in range(2))

    def call(lo, hi, stat, out, flags):
        p = [t.data_ptr() + 4 * lo for t in d]
        pkg.policy_loss_logp(p[0], hi - lo, p[3], p[4], hp, stat.data_ptr(), out.data_ptr() + 4 * lo, p[1], p[2], flags)

    call(0, tokens, whole, coef, 0)
    call(0, tokens, again, coef2, 0)
    cuts = [0, tokens // 3, tokens // 2, tokens]
    out = torch.empty(tokens, device="cuda")
    for lo, hi in zip(cuts, cuts[1:]):
        call(lo, hi, parts, out, pkg.LOSS_ACCUMULATE)
    torch.cuda.synchronize()
    assert torch.equal(whole, again) and torch.equal(coef, coef2) and torch.equal(coef, out)
    x, y = stat_of(pkg.PolicyStat, whole), stat_of(pkg.PolicyStat, parts)
    assert (x.tokens, x.clipped, x.ratio_max) == (y.tokens, y.clipped, y.ratio_max)
    per = Q.policy(logp, old, ref, a, w, w != 0, 0.2, float(torch.tensor(0.28)), 3.0, float(torch.tensor(0.1)), 3)
    wl = w.to(Q.F64) * per[0]
    e = Q.policy_error(torch.zeros(tokens, dtype=Q.F64), old, ref, logp, a, w, w != 0, 0.1)
    close(coef.cpu(), per[2], e, "coef")
    tol = float(e.sum()) + float(wl.abs().sum()) * 2.0 ** -20
    assert x.tokens == int((w != 0).sum()) and x.clipped == int(per[3].sum())
    assert abs(x.policy - float(wl.sum())) <= tol and abs(y.policy - float(wl.sum())) <= tol
    # coef in the place of the log-probabilities
    call(0, tokens, again, d[0], 0)
    torch.cuda.synchronize()
    assert torch.equal(d[0], coef)


def test_policy_places_without_weight_hold_anything(pkg):
    z, y = gaussian(6, 500, "f16", 1), torch.tensor([1, 2, 3, 4, 5, 6], dtype=torch.int32)
    z[2] = math.nan
    a, w = torch.ones(6), torch.tensor([1.0, 1, 0, 1, 0, 1])
    a[2], a[4] = math.nan, math.inf
    old = torch.full((6,), -6.0)
    old[4] = math.nan
    hp = pkg.policy_hparams()
    d = [t.cuda() for t in (z, y, a, w, old)]
    logp, grad, stat = torch.full((6,), 5.0, device="cuda"), torch.full((6, 500), 5.0, device="cuda", dtype=torch.float16), torch.zeros(8, dtype=torch.int32, device="cuda")
    pkg.policy_loss(d[0].data_ptr(), pkg.F16, 6, 500, d[1].data_ptr(), d[2].data_ptr(), d[3].data_ptr(), hp, logp.data_ptr(),
                    grad.data_ptr(), stat.data_ptr(), d[4].data_ptr())
    torch.cuda.synchronize()
    s = stat_of(pkg.PolicyStat, stat)
    assert s.tokens == 4 and math.isfinite(s.loss) and s.weight == 4.0
    assert bool((grad[[2, 4]] == 0).all()) and bool(torch.isfinite(grad).all()) and bool((logp[[2, 4]] == 0).all())


def test_policy_empty_calls(pkg):
    stat = torch.full((8,), 77, dtype=torch.int32, device="cuda")
    hp = pkg.policy_hparams()
    pkg.policy_loss_logp(None, 0, None, None, hp, stat.data_ptr())
    torch.cuda.synchronize()
    assert bool((stat == 0).all())
    pkg.policy_loss(None, pkg.F16, 0, 8, None, None, None, hp, None, None, stat.data_ptr())
    torch.cuda.synchronize()
    assert bool((stat == 0).all())


def test_policy_loss_alone_leaves_no_gradient(pkg):
    z, y = gaussian(8, 700, "bf16", 2), targets_of(8, 700, 2)
    a, w = torch.ones(8).cuda(), torch.full((8,), 0.125).cuda()
    hp, zb, yb = pkg.policy_hparams(), z.cuda(), y.cuda()
    got = []
    for with_grad in (True, False):
        logp, stat, grad = torch.empty(8, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda"), torch.empty_like(zb)
        pkg.policy_loss(zb.data_ptr(), pkg.BF16, 8, 700, yb.data_ptr(), a.data_ptr(), w.data_ptr(), hp, logp.data_ptr(),
                        grad.data_ptr() if with_grad else None, stat.data_ptr())
        torch.cuda.synchronize()
        got.append((logp, stat))
    x, s = got[0], got[1]
    # the two calls may take different kernels: log-probabilities agree to their error, the counts exactly
    e = Q.logprob_error(z, y, 1.0) + 2.0 ** -19
    close(x[0].cpu(), s[0].cpu(), 2 * e, "logp")
    assert torch.equal(x[1][4:6], s[1][4:6])


@pytest.mark.parametrize("dtype,vocab", [("f16", 151936), ("bf16", 5001), ("f32", 32000)])
def test_policy_in_place_and_repeatable(pkg, dtype, vocab):
    rows = 9
    z, y = gaussian(rows, vocab, dtype, 6), targets_of(rows, vocab, 6)
    a, w = torch.linspace(-1, 1, rows).cuda(), torch.full((rows,), 0.1).cuda()
    hp, yb, dt = pkg.policy_hparams(), y.cuda(), Q.kind(pkg, dtype)
    outs = []
    for k in range(3):
        zb = z.cuda()
        g = zb if k == 2 else torch.empty_like(zb)
        logp, stat = torch.empty(rows, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
        pkg.policy_loss(zb.data_ptr(), dt, rows, vocab, yb.data_ptr(), a.data_ptr(), w.data_ptr(), hp, logp.data_ptr(), g.data_ptr(), stat.data_ptr())
        torch.cuda.synchronize()
        outs.append((g, logp, stat))
    for o in outs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(outs[0], o))


# ---- preference loss ----------------------------------------------------------------

def check_preference(pkg, offsets, tokens, seed=0, beta=0.1, margin=0.0, smoothing=0.0, kind=0, mean=False, ref=True, mask=True, weights=False):
    g = torch.Generator().manual_seed(seed)
    pairs = (len(offsets) - 1) // 2
    logp = -torch.rand(tokens, generator=g) * 2
    rf = logp + torch.randn(tokens, generator=g) * 0.3 if ref else None
    mk = (torch.rand(tokens, generator=g) < 0.7).to(torch.uint8) * 3 if mask else None
    pw = torch.rand(pairs, generator=g) if weights else None
    lp, rr = logp.clone(), rf.clone() if ref else None
    if mask:                                     # what a masked place holds does not matter
        lp[mk == 0] = math.nan
        if ref:
            rr[mk == 0] = math.inf
    on = lambda t: None if t is None else t.cuda()  # noqa: E731
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    db = [on(t) for t in (lp, rr, mk, torch.tensor(offsets, dtype=torch.int32), pw)]
    coef, rewards = torch.full((tokens,), 7.0, device="cuda"), torch.full((2 * pairs,), 7.0, device="cuda")
    stat = torch.full((8,), 0x7FC00000, dtype=torch.int32, device="cuda")
    hp = pkg.preference_hparams(beta, margin, smoothing, kind, mean)
    pkg.preference_loss(at(db[0]), tokens, at(db[3]), pairs, hp, at(stat), at(coef), at(rewards), at(db[1]), at(db[2]), at(db[4]))
    torch.cuda.synchronize()
    s = stat_of(pkg.PreferenceStat, stat)
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
    loss, total, correct, want, rew = Q.preference(logp, rf, mk, offsets, pairs, f32(beta), f32(margin), f32(smoothing), kind, mean, pw)
    # a term logp - ref is rounded once (2^-24 of it), sums are in 64 bits; h is off by e, the loss and the slope of a
    # pair by their own slopes times e, results are rounded once
    terms = (logp.abs() + (rf.abs() if ref else 0)).to(Q.F64)
    sums = torch.tensor([float(terms[int(lo):int(hi)].sum()) for lo, hi in zip(offsets, offsets[1:])], dtype=Q.F64)
    if mean:
        n = torch.tensor([float((mk[int(lo):int(hi)] != 0).sum()) if mask else float(hi - lo) for lo, hi in zip(offsets, offsets[1:])], dtype=Q.F64)
        sums = sums / n.clamp(min=1)
    e = float(beta * sums.max()) * 2.0 ** -22 if pairs else 0.0
    steep = 2 / beta ** 2 * (1 + float(rew.abs().max()) if pairs else 1) if kind == 2 else 1.0
    big = float(pw.sum()) if weights else 1.0
    assert s.pairs == pairs and s.correct == correct
    assert abs(s.loss - loss) <= big * steep * e + abs(loss) * 2.0 ** -22 + 2.0 ** -40
    assert abs(s.margin - total) <= big * e + abs(total) * 2.0 ** -22
    close(rewards.cpu(), rew, rew.abs() * 2.0 ** -23 + e, "rewards")
    top = float(pw.max()) if weights else 1.0 / max(1, pairs)
    close(coef.cpu(), want, want.abs() * 2.0 ** -22 + beta * top * steep * e, "coef")
    assert bool((coef.cpu()[want == 0] == 0).all())


@pytest.mark.parametrize("offsets,tokens", [([0, 1, 2], 2), ([0, 0, 0], 1), ([0, 0, 5], 5), ([2, 9, 20], 31), ([0, 5, 5, 5, 9, 1500, 1501], 1600),
                                            ([0, 40, 100, 2000, 4100, 4100, 4200], 4200)])
@pytest.mark.parametrize("mask,ref", [(True, True), (False, False)])
def test_preference_sizes(pkg, offsets, tokens, mask, ref):
    check_preference(pkg, offsets, tokens, tokens, mask=mask, ref=ref)


@pytest.mark.parametrize("kind,smoothing,margin", [(0, 0.0, 0.0), (0, 0.2, 0.3), (1, 0.0, 0.1), (2, 0.0, 0.0), (2, 0.0, 0.2)])
@pytest.mark.parametrize("mean,weights", [(False, False), (True, True)])
def test_preference_kinds(pkg, kind, smoothing, margin, mean, weights):
    g = torch.Generator().manual_seed(kind)
    cuts = torch.randint(0, 3000, (39,), generator=g).sort().values.tolist()
    check_preference(pkg, [0] + cuts + [3000], 3010, kind, 0.25, margin, smoothing, kind, mean, weights=weights)


@pytest.mark.parametrize("pairs,tokens", [(150, 9000), (1, 70000), (3, 40000), (1000, 3000), (40, 100000)])
def test_preference_large_batches(pkg, pairs, tokens):
    g = torch.Generator().manual_seed(pairs)
    cuts = torch.randint(0, tokens + 1, (2 * pairs - 1,), generator=g).sort().values.tolist()
    check_preference(pkg, [0] + cuts + [tokens], tokens, pairs, beta=0.05)


def test_preference_offsets_out_of_range_are_held_inside(pkg):
    """Entries outside [0, tokens], and ones that fall, select nothing outside the buffers."""
    tokens = 100
    for bad, good in (([-50, 40, 4000], [0, 40, 100]), ([0, 200, 300], [0, 100, 100]), ([0, 60, 30], [0, 60, 60])):
        got = []
        for offsets in (bad, good):
            lp = -(torch.arange(tokens) % 7).float().cuda()
            coef, stat = torch.full((tokens,), 7.0, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
            ob = torch.tensor(offsets, dtype=torch.int32).cuda()
            pkg.preference_loss(lp.data_ptr(), tokens, ob.data_ptr(), 1, pkg.preference_hparams(0.1), stat.data_ptr(), coef.data_ptr())
            torch.cuda.synchronize()
            got.append((coef, stat))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_preference_record_accumulates(pkg):
    lp = -torch.rand(60, generator=torch.Generator().manual_seed(1)).cuda()
    w = torch.full((3,), 1 / 3).cuda()
    hp = pkg.preference_hparams(0.5)
    offsets = torch.tensor([0, 10, 20, 30, 40, 50, 60], dtype=torch.int32).cuda()
    whole, parts = torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
    pkg.preference_loss(lp.data_ptr(), 60, offsets.data_ptr(), 3, hp, whole.data_ptr(), pair_weight=w.data_ptr())
    for k in range(3):
        pkg.preference_loss(lp.data_ptr(), 60, offsets.data_ptr() + 8 * k, 1, hp, parts.data_ptr(), pair_weight=w.data_ptr() + 4 * k, flags=pkg.LOSS_ACCUMULATE)
    torch.cuda.synchronize()
    a, b = stat_of(pkg.PreferenceStat, whole), stat_of(pkg.PreferenceStat, parts)
    assert (a.pairs, a.correct) == (b.pairs, b.correct) and abs(a.loss - b.loss) <= 3 * 2.0 ** -24 * 3


@pytest.mark.parametrize("length", [3, 700])
def test_preference_coefficients_in_the_buffer_of_the_log_probabilities(pkg, length):
    """100 pairs of `length` tokens and 50 tokens of no sequence at either end: the same bits as in a buffer of their own."""
    pairs = 100
    offsets = torch.arange(2 * pairs + 1, dtype=torch.int32, device="cuda") * length + 50
    tokens = 2 * pairs * length + 100
    g = torch.Generator().manual_seed(length)
    logp, ref = ((-torch.rand(tokens, generator=g) * 2).cuda() for _ in range(2))
    results = []
    for coef in (torch.full_like(logp, 7.0), logp):
        stat, rewards = torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(2 * pairs, device="cuda")
        pkg.preference_loss(logp.data_ptr(), tokens, offsets.data_ptr(), pairs, pkg.preference_hparams(0.1), stat.data_ptr(), coef.data_ptr(),
                            rewards.data_ptr(), ref.data_ptr())
        torch.cuda.synchronize()
        results.append((coef, stat, rewards))
    assert all(torch.equal(x, y) for x, y in zip(*results))


def test_preference_without_pairs(pkg):
    coef, stat = torch.full((9,), 7.0, device="cuda"), torch.full((8,), 7, dtype=torch.int32, device="cuda")
    lp, ob = torch.zeros(9, device="cuda"), torch.tensor([4], dtype=torch.int32, device="cuda")
    pkg.preference_loss(lp.data_ptr(), 9, ob.data_ptr(), 0, pkg.preference_hparams(0.1), stat.data_ptr(), coef.data_ptr())
    torch.cuda.synchronize()
    assert bool((coef == 0).all()) and bool((stat == 0).all())


# ---- streams, graphs, and the step they belong to ---------------------------------

def test_two_streams_at_once(pkg):
    """Calls on different buffers may overlap: nothing is shared between them."""
    z = [gaussian(64, 20000, "bf16", k).cuda() for k in range(2)]
    y = [targets_of(64, 20000, k).cuda() for k in range(2)]
    a, w = torch.ones(64, device="cuda"), torch.full((64,), 1 / 64, device="cuda")
    hp = pkg.policy_hparams()
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = {}
    for many in (False, True):
        bufs = [(torch.empty(64, device="cuda"), torch.empty_like(z[k]), torch.zeros(8, dtype=torch.int32, device="cuda")) for k in range(2)]
        torch.cuda.synchronize()
        for _ in range(5 if many else 1):
            for k in range(2):
                lp, g, st = bufs[k]
                pkg.policy_loss(z[k].data_ptr(), pkg.BF16, 64, 20000, y[k].data_ptr(), a.data_ptr(), w.data_ptr(), hp, lp.data_ptr(), g.data_ptr(),
                                st.data_ptr(), stream=streams[k].cuda_stream if many else None)
        torch.cuda.synchronize()
        out[many] = bufs
    for k in range(2):
        assert all(torch.equal(p, q) for p, q in zip(out[False][k], out[True][k]))


def test_captured_graph_follows_its_inputs(pkg):
    """The preference step (log-probabilities, loss, gradient) captured once and replayed on other contents."""
    rows, vocab = 40, 3000
    z, y = torch.empty(rows, vocab, dtype=torch.float16, device="cuda"), torch.empty(rows, dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 10, 20, 25, 38], dtype=torch.int32, device="cuda")
    logp, lse, coef, grad = (torch.empty(rows, device="cuda") for _ in range(3)), None, None, torch.empty_like(z)
    logp, lse, coef = logp
    stat, hp, scaler = torch.zeros(8, dtype=torch.int32, device="cuda"), pkg.preference_hparams(0.1), scaler_of(pkg, 512.0)

    def step(stream):
        pkg.token_logprob(z.data_ptr(), pkg.F16, rows, vocab, y.data_ptr(), logp.data_ptr(), lse.data_ptr(), stream=stream)
        pkg.preference_loss(logp.data_ptr(), rows, offsets.data_ptr(), 2, hp, stat.data_ptr(), coef.data_ptr(), stream=stream)
        pkg.token_logprob_grad(z.data_ptr(), pkg.F16, rows, vocab, y.data_ptr(), lse.data_ptr(), coef.data_ptr(), grad.data_ptr(),
                               scaler=scaler.data_ptr(), stream=stream)

    z.copy_(gaussian(rows, vocab, "f16", 0))
    y.copy_(targets_of(rows, vocab, 0))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream().cuda_stream)
    for seed in (1, 2):
        z.copy_(gaussian(rows, vocab, "f16", seed))
        y.copy_(targets_of(rows, vocab, seed))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in (logp, stat, coef, grad)]
        step(None)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(kept, (logp, stat, coef, grad)))
        assert float(grad.float().abs().sum()) > 0


def test_bounded_waits_report_and_recover(pkg):
    pkg.losses_check()
    assert pkg.losses_selftest_wait() == pkg.ERR_TIMEOUT
    pkg.losses_check()                                   # cleared, and the device is usable
    check_policy(pkg, gaussian(20, 151936, "bf16", 5), targets_of(20, 151936, 5))
    pkg.losses_check()


def test_captured_policy_loss_follows_its_inputs(pkg):
    """The fused call (rows taken over by clusters, the record from a dependent launch) captured once, replayed on other
    contents, twice in a row."""
    rows, vocab = 300, 32000
    z, y = torch.empty(rows, vocab, dtype=torch.bfloat16, device="cuda"), torch.empty(rows, dtype=torch.int32, device="cuda")
    a, w = torch.randn(rows, device="cuda"), torch.full((rows,), 1 / rows, device="cuda")
    logp, grad, stat = torch.empty(rows, device="cuda"), torch.empty_like(z), torch.zeros(8, dtype=torch.int32, device="cuda")
    hp = pkg.policy_hparams()

    def call(stream):
        pkg.policy_loss(z.data_ptr(), pkg.BF16, rows, vocab, y.data_ptr(), a.data_ptr(), w.data_ptr(), hp, logp.data_ptr(), grad.data_ptr(),
                        stat.data_ptr(), stream=stream)

    z.copy_(gaussian(rows, vocab, "bf16", 0))
    y.copy_(targets_of(rows, vocab, 0))
    call(None)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(torch.cuda.current_stream().cuda_stream)
    for seed in (1, 2):
        z.copy_(gaussian(rows, vocab, "bf16", seed))
        y.copy_(targets_of(rows, vocab, seed))
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in (logp, stat, grad)]
        for t in (logp, grad):
            t.fill_(7)
        call(None)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(kept, (logp, stat, grad)))


def test_policy_loss_reads_what_ran_before_it(pkg):
    """Calls in a row on one stream, each on what the last one wrote: no launch may run ahead of the kernels it reads from."""
    rows, vocab = 64, 4096
    z0 = gaussian(rows, vocab, "f32", 3).cuda()
    y, a, w = targets_of(rows, vocab, 3, 0.0).cuda(), torch.ones(rows, device="cuda"), torch.ones(rows, device="cuda")
    hp = pkg.policy_hparams(1.0, math.inf)
    results = []
    for wait in (True, False):
        z, logp, coef = z0.clone(), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        stat, stat2 = (torch.zeros(8, dtype=torch.int32, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        for _ in range(30):
            pkg.policy_loss(z.data_ptr(), pkg.F32, rows, vocab, y.data_ptr(), a.data_ptr(), w.data_ptr(), hp, logp.data_ptr(), z.data_ptr(), stat.data_ptr())
            if wait:
                torch.cuda.synchronize()
            pkg.policy_loss_logp(logp.data_ptr(), rows, a.data_ptr(), w.data_ptr(), hp, stat2.data_ptr(), coef.data_ptr())
            z.mul_(3.0).add_(z0)
        torch.cuda.synchronize()
        results.append((z, logp, coef, stat, stat2))
    assert all(torch.equal(p, q) for p, q in zip(*results))


def test_logprob_without_lse(pkg):
    z, y = gaussian(20, 5001, "bf16", 8).cuda(), targets_of(20, 5001, 8).cuda()
    a, b, lse = torch.empty(20, device="cuda"), torch.empty(20, device="cuda"), torch.empty(20, device="cuda")
    pkg.token_logprob(z.data_ptr(), pkg.BF16, 20, 5001, y.data_ptr(), a.data_ptr())
    pkg.token_logprob(z.data_ptr(), pkg.BF16, 20, 5001, y.data_ptr(), b.data_ptr(), lse.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(a, b)


def test_policy_loss_in_chunks_accumulates(pkg):
    """The fused call on chunks of a batch, as the output projection hands them over: gradients and log-probabilities are those
    of the whole, bit for bit where the chunks take the same kernel, and the record adds up."""
    rows, vocab, chunk = 512, 6000, 128
    z, y = gaussian(rows, vocab, "f16", 9).cuda(), targets_of(rows, vocab, 9).cuda()
    g = torch.Generator().manual_seed(9)
    a, w = torch.randn(rows, generator=g).cuda(), (torch.rand(rows, generator=g) / rows).cuda()
    hp = pkg.policy_hparams()
    out = []
    for step in (rows, chunk):
        logp, grad, stat = torch.empty(rows, device="cuda"), torch.empty_like(z), torch.zeros(8, dtype=torch.int32, device="cuda")
        for r in range(0, rows, step):
            pkg.policy_loss(z[r:].data_ptr(), pkg.F16, step, vocab, y[r:].data_ptr(), a[r:].data_ptr(), w[r:].data_ptr(), hp, logp[r:].data_ptr(),
                            grad[r:].data_ptr(), stat.data_ptr(), flags=pkg.LOSS_ACCUMULATE if r else 0)
        torch.cuda.synchronize()
        out.append((logp, grad, stat_of(pkg.PolicyStat, stat)))
    e = Q.logprob_error(z.cpu(), y.cpu(), 1.0) + 2.0 ** -19
    close(out[1][0].cpu(), out[0][0].cpu(), 2 * e, "logp")
    x, s = out[0][2], out[1][2]
    assert (x.tokens, x.clipped) == (s.tokens, s.clipped)
    size = float((w * a.abs()).sum())
    assert abs(x.loss - s.loss) <= size * 8 * 2.0 ** -24 + float((w.cpu() * a.cpu().abs() * 2 * e).sum())
    assert abs(x.weight - s.weight) <= x.weight * 8 * 2.0 ** -24
