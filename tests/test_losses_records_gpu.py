"""GPU tests of the records of the losses where a cluster has CTAs with little or no work: the ones that are done at once
hand their sums to a first CTA that must have started."""
import pytest
import torch

import operator_oracle as Q
from test_losses_gpu import check_preference, off_the_borders, stat_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1025, 1500, 2048, 3000, 4097, 9000])
def test_policy_records_of_clusters_with_idle_ctas(pkg, tokens):
    g = torch.Generator().manual_seed(tokens)
    logp = -torch.rand(tokens, generator=g) * 3
    old = logp - off_the_borders(torch.randn(tokens, generator=g) * 0.3, 0.2, 0.2, 0.0)
    a, w = torch.randn(tokens, generator=g), torch.rand(tokens, generator=g)
    hp = pkg.policy_hparams(0.2, 0.2)
    d = [t.cuda() for t in (logp, a, w, old)]
    per = Q.policy(logp, old, None, a, w, w != 0, float(torch.tensor(0.2)), float(torch.tensor(0.2)), 0.0, 0.0, 3)
    wl = w.to(Q.F64) * per[0]
    e = Q.policy_error(torch.zeros(tokens, dtype=Q.F64), old, None, logp, a, w, w != 0, 0.0)
    records = torch.full((200, 8), 0x7FC00000, dtype=torch.int32, device="cuda")
    for k in range(200):
        pkg.policy_loss_logp(d[0].data_ptr(), tokens, d[1].data_ptr(), d[2].data_ptr(), hp, records[k].data_ptr(), None, d[3].data_ptr())
    torch.cuda.synchronize()
    assert bool((records == records[0]).all())
    s = stat_of(pkg.PolicyStat, records[0])
    assert (s.tokens, s.clipped) == (tokens, int(per[3].sum()))
    assert abs(s.loss - float(wl.sum())) <= float(e.sum()) + float(wl.abs().sum()) * 2.0 ** -20


@pytest.mark.parametrize("pairs,tokens", [(3, 40000), (5, 40000), (9, 70000), (3, 9000)])
def test_preference_records_of_clusters_with_idle_ctas(pkg, pairs, tokens):
    """More CTAs than pairs (their number is a power of two), without coefficients to write."""
    g = torch.Generator().manual_seed(pairs)
    cuts = torch.randint(0, tokens + 1, (2 * pairs - 1,), generator=g).sort().values.tolist()
    offsets = [0] + cuts + [tokens]
    check_preference(pkg, offsets, tokens, pairs, mask=False)
    logp, ob = -torch.rand(tokens, generator=g).cuda(), torch.tensor(offsets, dtype=torch.int32).cuda()
    records = torch.full((200, 8), 0x7FC00000, dtype=torch.int32, device="cuda")
    hp = pkg.preference_hparams(0.1)
    for k in range(200):
        pkg.preference_loss(logp.data_ptr(), tokens, ob.data_ptr(), pairs, hp, records[k].data_ptr())
    torch.cuda.synchronize()
    assert bool((records == records[0]).all())
    beta = float(torch.tensor(0.1))
    sums = torch.stack([logp.cpu().to(Q.F64)[lo:hi].sum() for lo, hi in zip(offsets, offsets[1:])]).view(pairs, 2)
    h = beta * (sums[:, 0] - sums[:, 1])
    loss, margin = float(torch.nn.functional.softplus(-h, threshold=1e9).mean()), float(h.mean())
    s = stat_of(pkg.PreferenceStat, records[0])
    assert (s.pairs, s.correct) == (pairs, int((sums[:, 0] > sums[:, 1]).sum()))
    assert abs(s.loss - loss) <= abs(loss) * 2.0 ** -20 and abs(s.margin - margin) <= abs(margin) * 2.0 ** -20


@pytest.mark.parametrize("kind,smoothing", [(0, 0.0), (0, 0.1), (1, 0.0)])
def test_preference_pairs_of_infinite_margin(pkg, kind, smoothing):
    """A token the policy gives no probability (log p = -inf) in a rejected sequence settles its pair: loss 0 and gradient 0,
    unless labels are smoothed; in a chosen one the loss is infinite and its slope the steepest."""
    inf, e = float("inf"), float(torch.tensor(smoothing))
    hp = pkg.preference_hparams(0.25, 0.0, smoothing, kind)
    cases = (([-1.0, -2.0, -0.5, -inf], inf, inf if smoothing else 0.0, e, 1),
             ([-2.5, -inf, -1.5, -1.0], -inf, inf, -(1 - e) if kind == 0 else -1.0, 0))
    for logp, margin, loss, slope, correct in cases:
        lp, ob = torch.tensor(logp).cuda(), torch.tensor([0, 2, 4], dtype=torch.int32).cuda()
        coef, stat = torch.full((4,), 7.0, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
        pkg.preference_loss(lp.data_ptr(), 4, ob.data_ptr(), 1, hp, stat.data_ptr(), coef.data_ptr())
        torch.cuda.synchronize()
        s = stat_of(pkg.PreferenceStat, stat)
        assert (s.loss, s.margin, s.correct) == (loss, margin, correct)
        want = torch.tensor([0.25 * slope] * 2 + [-0.25 * slope] * 2)
        assert (coef.cpu() - want).abs().max() <= 2.0 ** -26          # one rounding of a quarter


@pytest.mark.parametrize("kind", [0, 1, 2])
def test_preference_pairs_of_weight_zero_hold_anything(pkg, kind):
    """Pairs that pad a batch: the same record and coefficients as the batch without them, and 0 at their tokens."""
    g = torch.Generator().manual_seed(kind)
    logp = -torch.rand(60, generator=g)
    w = torch.tensor([0.25, 0.0, 0.5, 0.0, 0.25])
    offsets = torch.arange(11, dtype=torch.int32) * 6
    bad = logp.clone()
    bad[12:24] = float("nan")
    bad[40] = -float("inf")
    results = []
    for lp, pairs in ((bad, [0, 1, 2, 3, 4]), (torch.cat([logp[0:12], logp[24:36], logp[48:60]]), [0, 2, 4])):
        d = [lp.cuda(), offsets[:2 * len(pairs) + 1].cuda(), w[pairs].cuda()]
        coef, stat = torch.full((lp.numel(),), 7.0, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
        pkg.preference_loss(d[0].data_ptr(), lp.numel(), d[1].data_ptr(), len(pairs), pkg.preference_hparams(0.3, kind=kind), stat.data_ptr(),
                            coef.data_ptr(), pair_weight=d[2].data_ptr())
        torch.cuda.synchronize()
        results.append((coef.cpu(), stat_of(pkg.PreferenceStat, stat)))
    (coef, s), (short, t) = results
    assert (s.loss, s.margin, s.pairs, t.pairs) == (t.loss, t.margin, 5, 3)
    assert bool((coef[12:24] == 0).all()) and bool((coef[36:48] == 0).all())
    assert torch.equal(torch.cat([coef[0:12], coef[24:36], coef[48:60]]), short)
