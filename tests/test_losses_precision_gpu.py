"""GPU tests of the gradient of log-probabilities for confident targets among logits with a large common offset."""
import pytest
import torch

import operator_oracle as Q

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,offset,gap", [("f32", 1e4, 12.0), ("f32", -3e4, 15.0), ("f32", 5e5, 14.0), ("f32", 20.0, 16.0), ("bf16", 512.0, 16.0),
                                              ("f16", 1e4, 16.0)])
@pytest.mark.parametrize("vocab,gpad", [(40, 0), (5003, 0), (5003, 1), (70000, 0)])
def test_the_target_entry_of_a_confident_row(pkg, dtype, offset, gap, vocab, gpad):
    """1 - p is a few 1e-6 to 1e-2 here, below what an FP32 log-sum-exp of this size can tell."""
    rows, step = 6, {"f32": 2.0 ** -4, "bf16": 4.0, "f16": 8.0}[dtype]
    g = torch.Generator().manual_seed(vocab)
    z = offset - gap - step * torch.randint(0, 4, (rows, vocab), generator=g)
    y = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32)
    z[torch.arange(rows), y.long()] = offset
    z = z.to(Q.DTYPES[dtype])
    assert bool((z.double().gather(1, y.long()[:, None]) == offset).all())
    coef = torch.linspace(-1, 1, rows)
    want, want_lse, p, takes = Q.logprob(z, y)
    e = Q.logprob_error(z, y, 1.0)
    # the oracle in 64 bits: log p from the other tokens' share, whose sum has no offset
    rest = torch.exp(z.double() - offset).sum(1) - 1.0
    want = -torch.log1p(rest)
    zb, yb, cb = z.cuda(), y.cuda(), coef.cuda()
    gb = Q.Rows(torch.full_like(z, 3.0), gpad)
    logp, lse = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    kind = Q.kind(pkg, dtype)
    pkg.token_logprob(zb.data_ptr(), kind, rows, vocab, yb.data_ptr(), logp.data_ptr(), lse.data_ptr())
    pkg.token_logprob_grad(zb.data_ptr(), kind, rows, vocab, yb.data_ptr(), lse.data_ptr(), cb.data_ptr(), gb.ptr, 0, gb.stride, logp=logp.data_ptr())
    torch.cuda.synchronize()
    got = gb.get().double()
    # log p is off by e in absolute terms (e counts the spread of the logits, not their offset) and so is 1 - p
    assert ((logp.cpu().double() - want).abs() <= e + want.abs() * 2.0 ** -22).all()
    at = got[torch.arange(rows), y.long()]
    share = -torch.expm1(want)
    tol = coef.double().abs() * (e + share * 2.0 ** -21)
    assert ((at - coef.double() * share).abs() <= tol + Q.rounding(coef.double() * share + tol, z.dtype)).all()
    # the others: relative to themselves
    p = torch.exp(z.double() - offset + want[:, None])
    grad = Q.logits_grad(p, y, takes, coef)
    rel = (want_lse.abs() * 2.0 ** -22 + 2 * e + 2.0 ** -20)[:, None]
    off = (got - grad).abs() - grad.abs() * rel * 1.5 - Q.rounding(grad, z.dtype) * 1.01
    off[torch.arange(rows), y.long()] = 0.0
    assert bool((off <= 2.0 ** -125).all())


@pytest.mark.parametrize("vocab", [40, 5003])
def test_rows_without_part_and_empty_rows_with_log_probabilities_given(pkg, vocab):
    z = torch.zeros(4, vocab)
    z[1] = -float("inf")
    z[2] = -1e9
    y, coef = torch.tensor([-1, 3, 4, 5], dtype=torch.int32), torch.tensor([1.0, 1.0, 1.0, 0.0])
    zb, yb, cb, grad = z.cuda(), y.cuda(), coef.cuda(), torch.full_like(z, 7.0).cuda()
    logp, lse = torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
    pkg.token_logprob(zb.data_ptr(), pkg.F32, 4, vocab, yb.data_ptr(), logp.data_ptr(), lse.data_ptr())
    pkg.token_logprob_grad(zb.data_ptr(), pkg.F32, 4, vocab, yb.data_ptr(), lse.data_ptr(), cb.data_ptr(), grad.data_ptr(), logp=logp.data_ptr())
    torch.cuda.synchronize()
    hot = torch.zeros(vocab)
    hot[3] = 1.0
    got = grad.cpu()
    assert bool((got[0] == 0).all()) and torch.equal(got[1].abs(), hot) and bool(torch.isnan(got[2]).all()) and bool((got[3] == 0).all())
