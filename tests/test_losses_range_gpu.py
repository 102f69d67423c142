"""GPU tests of the losses on logits of any size: masks of every usual constant over whole stretches of a row, rows of
nothing but one mask, logits so large that FP32 no longer tells neighbours of their exponent apart."""
import math

import pytest
import torch

import operator_oracle as Q
from test_losses_gpu import check_policy, close, gaussian, run_logprob

pytestmark = pytest.mark.gpu

MASKS = [-1e9, -1e10, -1e12, -1e20, -1e25, -9e29, -1e30, -1e35]


def policy(pkg, z, y, it):
    """(logp, gradient) of the policy loss with weights and advantages of 1."""
    rows, vocab = z.shape
    zb, yb, one = z.cuda(), y.cuda(), torch.ones(rows, device="cuda")
    logp, grad, stat = torch.empty(rows, device="cuda"), torch.empty_like(zb), torch.zeros(8, dtype=torch.int32, device="cuda")
    dt = {torch.float16: pkg.F16, torch.bfloat16: pkg.BF16, torch.float32: pkg.F32}[z.dtype]
    pkg.policy_loss(zb.data_ptr(), dt, rows, vocab, yb.data_ptr(), one.data_ptr(), one.data_ptr(), pkg.policy_hparams(), logp.data_ptr(),
                    grad.data_ptr(), stat.data_ptr(), inv_temperature=it)
    torch.cuda.synchronize()
    return logp.cpu(), grad.cpu()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [40, 5003, 151936])
def test_masked_stretches_are_as_minus_infinity(pkg, dtype, vocab):
    """A logit below the others by 2^8 and more adds nothing to an FP32 sum: the same bits as with -inf, whatever the mask,
    wherever it lies and however many of a thread's entries it covers."""
    for it in (1.0, 0.7, 1 / 0.6):
        for lo, hi in ((vocab // 4, vocab), (0, vocab * 3 // 4), (vocab // 3, vocab // 2)):
            keep = gaussian(len(MASKS) + 1, vocab, dtype, vocab)
            z, plain = keep.clone(), keep.clone()
            plain[:, lo:hi] = -math.inf
            for r, m in enumerate(MASKS):
                z[r, lo:hi] = m
            z[-1, lo:hi] = -1e15
            z[-1, lo:(lo + hi) // 2] = -1e10           # two masks in one row
            y = torch.full((len(z),), 0 if lo else vocab - 1, dtype=torch.int32)
            coef = torch.linspace(-1, 1, len(z))
            for got, want in zip(run_logprob(pkg, z, y, it, coef), run_logprob(pkg, plain, y, it, coef)):
                assert bool(torch.isfinite(want).all()) and torch.equal(got, want)
            for got, want in zip(policy(pkg, z, y, it), policy(pkg, plain, y, it)):
                assert bool(torch.isfinite(want).all()) and torch.equal(got, want)


@pytest.mark.parametrize("vocab", [40, 5003, 70000])
def test_masked_stretches_of_f16_under_a_low_temperature(pkg, vocab):
    it = 1e5                                           # (a gradient of 1 times that is beyond FP16: inf, the same on both sides)
    z, plain = (gaussian(4, vocab, "f16", vocab, 1e-4) for _ in range(2))
    z[:, vocab // 4:] = -65504.0                       # times 1e5 log2 e: -9.5e9
    plain[:, vocab // 4:] = -math.inf
    y = torch.tensor([0, 1, 2, 3], dtype=torch.int32)
    coef = torch.ones(4)
    for got, want in zip(run_logprob(pkg, z, y, it, coef), run_logprob(pkg, plain, y, it, coef)):
        assert not bool(torch.isnan(want).any()) and torch.equal(got, want)
    for got, want in zip(policy(pkg, z, y, it), policy(pkg, plain, y, it)):
        assert not bool(torch.isnan(want).any()) and torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [40, 5003, 70000, 262145])
@pytest.mark.parametrize("it", [1.0, 0.7, 1 / 0.6])
def test_rows_of_one_value_are_uniform(pkg, dtype, vocab, it):
    """All logits alike, of any size: log p = -log(vocab).  c = it * log2 e cancels, so the error is that of a row without
    spread."""
    values = [0.0, -3.0, 1e4, -1e4, 1e7, -1e7, 1e8, -1e8, -1e9, 1e9, -1e10, 1e10, 1e15, -1e20, 1e20, -9e29, 1e30, 1e37]
    z = torch.tensor(values).to(Q.DTYPES[dtype])[:, None].expand(len(values), vocab).contiguous()
    y = torch.arange(len(values), dtype=torch.int32) * (vocab - 1) // (len(values) - 1)
    logp, lse, _ = run_logprob(pkg, z, y, it)
    it32 = float(torch.tensor(it, dtype=torch.float32))
    want = torch.full((len(values),), -math.log(vocab), dtype=Q.F64)
    e = Q.logprob_error(z, y, it32)
    close(logp, want, e + want.abs() * 2.0 ** -22, "logp")
    want_lse = z[:, 0].double() * it32 - want
    close(lse, want_lse, e + want_lse.abs() * 2.0 ** -22, "lse")
    # the 64-bit oracle forms log p as a difference, which holds while doubles are fine enough for it (1e9: to 2^-23)
    small = z[:, 0].double().abs() <= 1.1e9
    check_policy(pkg, z[small], y[small], it=it, scale=64.0)
    logp, grad = policy(pkg, z, y, it)
    close(logp, want, e + want.abs() * 2.0 ** -22, "logp")
    p = torch.full(z.shape, 1.0 / vocab, dtype=Q.F64)
    want_grad = Q.logits_grad(p, y, torch.ones(len(z), dtype=torch.bool), -torch.ones(len(z)), it32)      # coef = -1 on policy
    hot = (want_grad < 0).double()
    close(grad, want_grad, want_grad.abs() * (2 * float(e.max()) + 2.0 ** -21) + hot * it32 * 2.0 ** -23 + Q.rounding(want_grad, z.dtype), "grad")


@pytest.mark.parametrize("vocab", [40, 5003, 70000])
@pytest.mark.parametrize("it", [0.5, 0.6, 0.69, 1.0])
def test_neighbours_of_large_logits_are_told_apart(pkg, vocab, it):
    """Steps of FP32 around 1e10 are 1024: among such logits the largest share the probability, and the next below has
    log p = -1024 it - log(count)."""
    it32 = float(torch.tensor(it, dtype=torch.float32))
    for top in (1e10, -1e10):
        for share in (1, 7, vocab // 2):
            z = torch.full((2, vocab), top - 1024.0)
            g = torch.Generator().manual_seed(share)
            at = torch.randperm(vocab, generator=g)[:share]
            z[:, at] = top
            other = int((~torch.isin(torch.arange(vocab), at)).nonzero()[0])
            y = torch.tensor([int(at[0]), other], dtype=torch.int32)
            logp, grad = policy(pkg, z, y, it)
            alone, lse, _ = run_logprob(pkg, z, y, it)
            want = torch.tensor([-math.log(share), -1024.0 * it32 - math.log(share)], dtype=Q.F64)
            e = (vocab / 128 + 24) * 2.0 ** -24 + 2.0 ** -21
            for got in (logp, alone):
                close(got, want, e + want.abs() * 2.0 ** -22, "logp")
            close(lse, torch.full((2,), top * it32 + math.log(share), dtype=Q.F64), abs(top) * it32 * 2.0 ** -22, "lse")
            p = torch.zeros(2, vocab, dtype=Q.F64)
            p[:, at] = 1.0 / share
            # advantage and weight 1, on policy: coef = -1
            want_grad = Q.logits_grad(p, y, torch.ones(2, dtype=torch.bool), -torch.ones(2), it32)
            close(grad, want_grad, want_grad.abs() * (2 * e + 2.0 ** -21) + it32 * 2.0 ** -23, "grad")


def test_a_masked_target_is_far_away(pkg):
    z = gaussian(3, 5003, "f32", 3)
    z[:, 100:3000] = -1e12
    y = torch.tensor([100, 2999, 50], dtype=torch.int32)
    logp, lse, _ = run_logprob(pkg, z, y, 1.0)
    want = Q.logprob(z, y)
    close(logp, want[0], want[0].abs() * 2.0 ** -22 + 2.0 ** -18, "logp")
    logp, grad = policy(pkg, z, y, 1.0)
    close(logp, want[0], want[0].abs() * 2.0 ** -22 + 2.0 ** -18, "logp")
    assert bool(torch.isfinite(grad).all())


def test_a_gradient_from_an_unusable_log_sum_exp_is_not_made_up(pkg):
    """FP32 holds -1e9 to 64: of such a log-sum-exp no probability can be told, and the row says so."""
    for vocab in (40, 5003):
        z = gaussian(3, vocab, "f32", 1)
        z[1] = -1e9
        y = torch.tensor([0, 1, 2], dtype=torch.int32)
        _, lse, grad = run_logprob(pkg, z, y, 1.0, torch.ones(3))
        assert float(lse[1]) == -1e9
        assert bool(torch.isnan(grad[1]).all()) and bool(torch.isfinite(grad[[0, 2]]).all())


@pytest.mark.parametrize("it", [1.0, 1e-25])
@pytest.mark.parametrize("vocab", [40, 5003])
def test_rows_of_nothing_but_absent_logits(pkg, it, vocab):
    z = torch.full((4, vocab), -math.inf)
    z[1] = -2e30
    z[2] = torch.finfo(torch.float32).min
    z[3, 1::2] = -1e31
    y = torch.tensor([0, 1, 2, 3], dtype=torch.int32)
    logp, lse, grad = run_logprob(pkg, z, y, it, torch.ones(4))
    other, fused = policy(pkg, z, y, it)
    for t in (logp, lse, other):
        assert bool((t == -math.inf).all())
    rest = torch.ones(4, vocab, dtype=torch.bool)
    rest[torch.arange(4), y.long()] = False
    for t, at_target in ((grad, it), (fused, -it)):
        assert bool((t[rest] == 0).all()) and bool((t[~rest] == torch.tensor(at_target)).all())


def test_rows_looked_at_again_in_graphs_and_on_two_streams(pkg):
    """A third of the rows are nothing but one mask; the calls are captured on two streams, replayed together on other
    contents, and give what calls one after the other give."""
    rows, vocab = 1100, 4096
    sets = []
    for k in range(2):
        z = torch.empty(rows, vocab, dtype=torch.bfloat16, device="cuda")
        y = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(k), dtype=torch.int32).cuda()
        one = torch.ones(rows, device="cuda")
        sets.append((z, y, one, torch.empty(rows, device="cuda"), torch.empty_like(z), torch.zeros(8, dtype=torch.int32, device="cuda")))
    hp = pkg.policy_hparams()

    def fill(seed):
        for k, s in enumerate(sets):
            s[0].copy_(gaussian(rows, vocab, "bf16", seed + 10 * k))
            s[0][k::3] = -1e12
            s[0][k + 1, 7:] = -1e20

    def call(s, stream):
        z, y, one, logp, grad, stat = s
        pkg.policy_loss(z.data_ptr(), pkg.BF16, rows, vocab, y.data_ptr(), one.data_ptr(), one.data_ptr(), hp, logp.data_ptr(), grad.data_ptr(),
                        stat.data_ptr(), stream=stream)

    fill(0)
    graphs, streams = [], [torch.cuda.Stream() for _ in sets]
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call(s, torch.cuda.current_stream().cuda_stream)
    fill(1)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    kept = [[t.clone() for t in s[3:]] for s in sets]
    for s, old in zip(sets, kept):
        for t in s[3:]:
            t.zero_()
        call(s, None)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(old, s[3:]))
    for k, (logp, grad, _) in enumerate(kept):
        assert ((logp[k::3].double() + math.log(vocab)).abs() <= 2.0 ** -17).all() and bool(torch.isfinite(grad).all())
    pkg.losses_check()
