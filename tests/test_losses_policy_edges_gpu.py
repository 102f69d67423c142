"""GPU tests of the policy loss at the ends of its terms' ranges."""
import math

import pytest
import torch

from test_losses_gpu import stat_of

pytestmark = pytest.mark.gpu


def losses(pkg, logp, old, a, w, hp, ref=None):
    """(coef, record) of the call on log-probabilities, and (gradient, record) of the fused one on logits that have them:
    two entries, log p and log(1 - p)."""
    n = len(logp)
    on = [torch.tensor(v, dtype=torch.float32).cuda() for v in (logp, old, a, w)]
    rf = torch.tensor(ref, dtype=torch.float32).cuda() if ref else None
    coef, stat = torch.full((n,), 7.0, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
    pkg.policy_loss_logp(on[0].data_ptr(), n, on[2].data_ptr(), on[3].data_ptr(), hp, stat.data_ptr(), coef.data_ptr(), on[1].data_ptr(),
                         rf.data_ptr() if ref else None)
    z = torch.stack([on[0], torch.log1p(-torch.exp(on[0]))], 1).contiguous()
    y, out, grad, stat2 = torch.zeros(n, dtype=torch.int32).cuda(), torch.empty(n).cuda(), torch.full((n, 2), 7.0).cuda(), torch.zeros_like(stat)
    pkg.policy_loss(z.data_ptr(), pkg.F32, n, 2, y.data_ptr(), on[2].data_ptr(), on[3].data_ptr(), hp, out.data_ptr(), grad.data_ptr(), stat2.data_ptr(),
                    on[1].data_ptr(), rf.data_ptr() if ref else None)
    torch.cuda.synchronize()
    return coef.cpu(), stat_of(pkg.PolicyStat, stat), grad.cpu(), stat_of(pkg.PolicyStat, stat2)


@pytest.mark.parametrize("clip", [(0.2, 0.28, 0.0), (0.2, 0.28, 3.0), (1.0, math.inf, 0.0)])
@pytest.mark.parametrize("zero", [0.0, -0.0])
def test_tokens_without_advantage_whose_ratio_is_beyond_fp32(pkg, clip, zero):
    """exp(99) times 0 is 0, like exp(80) times 0: neither loss nor gradient."""
    coef, s, grad, s2 = losses(pkg, [-1.0, -1.0, -1.0], [-100.0, -81.0, -1.25], [zero, zero, 1.0], [0.5, 0.5, 1.0], pkg.policy_hparams(*clip))
    cut = 1.28 < math.exp(0.25) and clip[1] < 1.0
    r = 1.28 if cut else math.exp(0.25)
    for rec in (s, s2):
        assert abs(rec.loss + r) <= r * 2.0 ** -20 and rec.tokens == 3 and rec.clipped == cut and rec.ratio_max == math.inf
    assert bool((coef[:2] == 0).all()) and abs(float(coef[2]) + (0 if cut else r)) <= r * 2.0 ** -20
    assert bool((grad[:2] == 0).all()) and bool(torch.isfinite(grad).all())


def test_a_ratio_that_is_not_a_number_still_shows(pkg):
    for old in (-math.inf, math.nan):
        coef, s, grad, s2 = losses(pkg, [-1.0, -1.0], [old, -1.0], [0.0, 0.0], [0.5, 0.5], pkg.policy_hparams())
        assert math.isnan(float(coef[0])) and float(coef[1]) == 0 and math.isnan(s.loss) and math.isnan(s2.loss)
        assert bool(torch.isnan(grad[0]).all()) and bool((grad[1] == 0).all())


def test_a_positive_advantage_is_clipped_at_any_ratio(pkg):
    coef, s, grad, s2 = losses(pkg, [-1.0, -1.0], [-100.0, -math.inf], [2.0, 2.0], [0.5, 0.5], pkg.policy_hparams(0.2, 0.25))
    for rec in (s, s2):
        assert rec.loss == -2.5 and rec.clipped == 2
    assert bool((coef == 0).all()) and bool((grad == 0).all())
