"""GPU tests of the loss kernels' bounded waits that give up: they are told to give up at once, report it, and wait on, so
that nothing is left on its way.  What such a call leaves must not look like a result."""
import math

import pytest
import torch

import operator_oracle as Q
from test_losses_gpu import gaussian, stat_of, targets_of

pytestmark = pytest.mark.gpu


@pytest.fixture
def impatient(pkg):
    """Sets the number of tries for the waits of later calls; put back, and the condition cleared, at the end."""
    before = pkg.losses_selftest_tries(0)
    pkg.losses_selftest_tries(before)
    yield pkg.losses_selftest_tries
    pkg.losses_selftest_tries(before)
    try:
        pkg.losses_check()
    except pkg.RlcuError:
        pass


class Call:
    def __init__(self, pkg, rows, vocab, dtype, in_place=False, with_grad=True):
        self.pkg, self.rows, self.vocab = pkg, rows, vocab
        self.kind, self.in_place, self.with_grad = Q.kind(pkg, dtype), in_place, with_grad
        self.source = gaussian(rows, vocab, dtype, rows).cuda()
        self.y = targets_of(rows, vocab, rows).cuda()
        self.a = torch.linspace(-1, 1, rows).cuda()
        self.w = torch.full((rows,), 1 / rows).cuda()
        self.hp = pkg.policy_hparams()

    def __call__(self):
        z = self.source.clone()
        grad = z if self.in_place else torch.full_like(z, 7.0)
        logp, stat = torch.full((self.rows,), 7.0, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
        self.pkg.policy_loss(z.data_ptr(), self.kind, self.rows, self.vocab, self.y.data_ptr(), self.a.data_ptr(), self.w.data_ptr(), self.hp,
                             logp.data_ptr(), grad.data_ptr() if self.with_grad else None, stat.data_ptr())
        torch.cuda.synchronize()
        return logp.cpu(), grad.cpu(), stat_of(self.pkg.PolicyStat, stat)


def same(x, y):
    return torch.equal(x[0], y[0]) and torch.equal(x[1], y[1]) and bytes(x[2]) == bytes(y[2])


def spoilt(got, good, with_grad=True):
    logp, grad, s = got
    assert bool(torch.isnan(logp).all()) and all(math.isnan(v) for v in (s.loss, s.policy, s.weight))
    if with_grad:
        assert bool(torch.isnan(grad[:, 0]).all()) and torch.equal(grad[:, 1:], good[1][:, 1:])


@pytest.mark.parametrize("rows,vocab,dtype", [(20, 151936, "bf16"), (3, 32000, "f32"), (700, 4097, "f16"), (1500, 16411, "f16"), (1, 70000, "f32")])
@pytest.mark.parametrize("in_place", [False, True])
def test_a_policy_loss_whose_waits_gave_up_is_spoilt_and_the_next_one_is_not(pkg, impatient, rows, vocab, dtype, in_place):
    call = Call(pkg, rows, vocab, dtype, in_place)
    good = call()
    pkg.losses_check()
    assert math.isfinite(good[2].loss)
    before = impatient(0)
    got = call()
    impatient(before)
    spoilt(got, good)
    spoilt(call(), good)                              # nobody has asked yet
    with pytest.raises(pkg.RlcuError) as e:
        pkg.losses_check()
    assert e.value.code == pkg.ERR_TIMEOUT
    pkg.losses_check()
    assert same(call(), good)


def test_the_loss_alone_and_the_other_kernels_are_spoilt_too(pkg, impatient):
    few, alone = Call(pkg, 12, 40, "f32"), Call(pkg, 6, 70000, "bf16", with_grad=False)
    good = few(), alone()
    before = impatient(0)
    got = alone()
    impatient(before)
    spoilt(got, good[1], with_grad=False)
    spoilt(few(), good[0])
    with pytest.raises(pkg.RlcuError):
        pkg.losses_check()
    assert same(few(), good[0]) and same(alone(), good[1])


def test_log_probabilities_after_a_wait_taken_up_again(pkg, impatient):
    z, y = gaussian(5, 151936, "f16", 1).cuda(), targets_of(5, 151936, 1).cuda()
    results = []
    before = impatient(0)
    for tries in (before, 0):
        impatient(tries)
        logp, lse = torch.full((5,), 7.0, device="cuda"), torch.full((5,), 7.0, device="cuda")
        pkg.token_logprob(z.data_ptr(), pkg.F16, 5, 151936, y.data_ptr(), logp.data_ptr(), lse.data_ptr())
        torch.cuda.synchronize()
        results.append((logp, lse))
        if tries:
            pkg.losses_check()
    assert all(torch.equal(p, q) for p, q in zip(*results))
    with pytest.raises(pkg.RlcuError) as e:
        pkg.losses_check()
    assert e.value.code == pkg.ERR_TIMEOUT


def test_the_vector_loss_has_no_such_waits(pkg, impatient):
    logp, a, w = torch.full((50,), -1.0, device="cuda"), torch.ones(50, device="cuda"), torch.full((50,), 0.02, device="cuda")
    call = Call(pkg, 20, 151936, "bf16")
    before = impatient(0)
    call()
    impatient(before)
    stat = torch.zeros(8, dtype=torch.int32, device="cuda")
    pkg.policy_loss_logp(logp.data_ptr(), 50, a.data_ptr(), w.data_ptr(), pkg.policy_hparams(), stat.data_ptr())
    torch.cuda.synchronize()
    assert abs(stat_of(pkg.PolicyStat, stat).loss + 1.0) < 1e-5
