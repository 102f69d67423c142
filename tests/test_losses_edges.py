"""Losses on the CPU: refusals and host-side settings beyond those of test_losses.py."""
import pytest
import torch


def test_tries_of_the_waits_are_bounded_and_put_back(pkg):
    before = pkg.losses_selftest_tries(5)
    assert before > 5
    assert pkg.losses_selftest_tries(0xFFFFFFFF) == 5
    assert pkg.losses_selftest_tries(before) == before          # no more than the number they start with


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


def test_log_probabilities_over_what_the_call_reads_are_refused(pkg):
    z, y, logp, lse = places(4)
    rows, vocab, stride = 5, 8, 24                    # FP16 rows of 16 bytes, 48 apart

    def call(logp=logp, lse=lse, targets=y):
        pkg.token_logprob(z, pkg.F16, rows, vocab, targets, logp, lse, row_stride=stride)

    for name in ("logp", "lse"):
        for at in (y, y + 16, y - 16, z, z + 12, z - 16, z + 4 * 48, z + 4 * 48 + 12, z + 32):
            refuse(pkg, "overlap", call, **{name: at})
    refuse(pkg, "overlap", call, lse=logp)
    refuse(pkg, "overlap", call, lse=logp + 16)
    # 20 bytes that fill the 32 between two rows up to the next one's start are not the logits'
    taken(pkg, call, logp=z + 28)
    taken(pkg, call, logp=z + 16)


def test_a_gradient_over_vectors_of_its_call_is_refused(pkg):
    z, y, lse, coef, scaler, g = places(6)

    def call(targets=y, lse=lse, coef=coef, scaler=scaler):
        pkg.token_logprob_grad(z, pkg.F32, 3, 16, targets, lse, coef, g, grad_stride=32, scaler=scaler)

    for name in ("targets", "lse", "coef", "scaler"):
        for at in (g, g - 8, g + 60, g + 128 + 4, g + 2 * 128 + 60, g + 120):
            refuse(pkg, "overlap", call, **{name: at})


def test_policy_losses_that_write_over_what_they_read_are_refused(pkg):
    z, y, old, ref, adv, w, logp, scaler, g, stat = places(10)
    ok = pkg.policy_hparams(0.2, 0.28, 3.0, 0.1)

    def call(targets=y, old=old, ref=ref, adv=adv, w=w, logp=logp, scaler=scaler, g=g, stat=stat):
        pkg.policy_loss(z, pkg.BF16, 4, 8, targets, adv, w, ok, logp, g, stat, old_logp=old, ref_logp=ref, scaler=scaler)

    for name in ("targets", "old", "ref", "adv", "w", "logp", "scaler"):
        for at in (g, g + 60, g - 12, stat, stat + 16, stat - 12):
            refuse(pkg, "overlap", call, **{name: at})
    for at in (y, y + 12, z, z + 60, scaler + 16, stat):
        refuse(pkg, "overlap", call, logp=at)
    for at in (z, z + 48, g + 48, g - 16):
        refuse(pkg, "overlap", call, stat=at)
        if at < g - 16:
            refuse(pkg, "overlap", call, stat=at, g=None)
    refuse(pkg, "overlap", call, logp=z + 4, g=None)
    for name in ("old", "ref", "adv", "w"):
        refuse(pkg, "overlap", pkg.policy_loss_logp, logp, 6, adv if name != "adv" else stat, w if name != "w" else stat + 16, ok, stat,
               old_logp=old if name != "old" else stat - 16, ref_logp=ref if name != "ref" else stat + 28)
    refuse(pkg, "overlap", pkg.policy_loss_logp, stat - 20, 6, adv, w, ok, stat, ref_logp=ref)
    refuse(pkg, "overlap", pkg.policy_loss_logp, logp, 6, adv, w, ok, stat, coef=stat + 4, ref_logp=ref)


def test_preference_losses_that_write_over_what_they_read_are_refused(pkg):
    logp, ref, mask, offsets, weight, coef, rewards, stat = places(8)

    def call(logp=logp, ref=ref, mask=mask, offsets=offsets, weight=weight, coef=coef, rewards=rewards, stat=stat):
        pkg.preference_loss(logp, 40, offsets, 3, pkg.preference_hparams(0.1), stat, coef, rewards, ref, mask, weight)

    for name, size in (("logp", 160), ("ref", 160), ("mask", 40), ("offsets", 28), ("weight", 12)):
        for out, room in ((rewards, 24), (stat, 32)) + (((coef, 160),) if name in ("mask", "offsets", "weight") else ()):
            for at in (out, out + room - 4, out - size + 4):
                refuse(pkg, "overlap", call, **{name: at})
    for at in (coef, coef + 156, stat + 28, stat - 20):
        refuse(pkg, "overlap", call, rewards=at)
    for at in (coef, coef + 144):
        refuse(pkg, "overlap", call, stat=at)


def brute(p, p_row, q, q_row, stride, rows):
    """Whether two matrices share a byte, row by row."""
    return any(p + i * stride < q + j * stride + q_row and q + j * stride < p + i * stride + p_row for i in range(rows) for j in range(rows))


def test_a_gradient_beside_its_logits_in_one_buffer(pkg):
    """Every place of a gradient around logits of the same stride: refused where a row of one meets a row of the other,
    taken elsewhere (in the same place: in place)."""
    z, y, lse, coef = places(4)
    rows, vocab, stride = 4, 6, 20                    # FP16
    for shift in range(-5 * stride, 5 * stride + 1):
        def call():
            pkg.token_logprob_grad(z, pkg.F16, rows, vocab, y, lse, coef, z + 2 * shift, row_stride=stride, grad_stride=stride)

        if shift and brute(z, 12, z + 2 * shift, 12, 40, rows):
            refuse(pkg, "overlap", call)
        else:
            taken(pkg, call)


def test_log_probabilities_given_to_the_gradient_are_checked(pkg):
    z, y, lse, coef, g, logp = places(6)

    def call(logp):
        pkg.token_logprob_grad(z, pkg.F16, 3, 16, y, lse, coef, g, logp=logp)

    refuse(pkg, "aligned", call, logp + 2)
    for at in (g, g + 92, g - 8):
        refuse(pkg, "overlap", call, at)
    taken(pkg, call, logp)
    taken(pkg, call, None)
