"""Losses on the CPU: what the entry points refuse (nothing is launched), and the oracle against torch's autograd."""
import math

import pytest
import torch

import operator_oracle as Q

A = 1 << 20           # an address that is never read: every call here is refused before it could be


def refuse(pkg, text, call, *args, **kwargs):
    with pytest.raises(pkg.RlcuError) as e:
        call(*args, **kwargs)
    assert e.value.code == pkg.ERR_INVALID and text in str(e.value), str(e.value)


def test_logprob_refusals(pkg):
    f = pkg.token_logprob
    refuse(pkg, "dtype", f, A, 7, 1, 8, A, A)
    refuse(pkg, "vocab", f, A, pkg.F16, 1, 0, A, A)
    refuse(pkg, "vocab", f, A, pkg.F16, 1, 1 << 31, A, A)
    refuse(pkg, "stride", f, A, pkg.F16, 1, 8, A, A, row_stride=7)
    refuse(pkg, "stride", f, A, pkg.F16, 1 << 30, 8, A, A, row_stride=1 << 40)
    refuse(pkg, "rows", f, A, pkg.F16, 1 << 31, 8, A, A)
    for t in (0.0, -1.0, math.inf, math.nan, 2e6):
        refuse(pkg, "inv_temperature", f, A, pkg.F16, 1, 8, A, A, inv_temperature=t)
    refuse(pkg, "null", f, None, pkg.F16, 1, 8, A, A)
    refuse(pkg, "null", f, A, pkg.F16, 1, 8, None, A)
    refuse(pkg, "null", f, A, pkg.F16, 1, 8, A, None)
    refuse(pkg, "aligned", f, A + 1, pkg.F16, 1, 8, A, A)
    refuse(pkg, "aligned", f, A + 2, pkg.F32, 1, 8, A, A)
    f(None, pkg.F16, 0, 8, None, None)                       # no rows: nothing to do


def test_logprob_grad_refusals(pkg):
    f = pkg.token_logprob_grad
    B = A + (1 << 16)
    refuse(pkg, "null", f, A, pkg.F16, 1, 8, A, None, A, B)
    refuse(pkg, "null", f, A, pkg.F16, 1, 8, A, A, None, B)
    refuse(pkg, "null", f, A, pkg.F16, 1, 8, A, A, A, None)
    refuse(pkg, "stride", f, A, pkg.F16, 1, 8, A, A, A, B, grad_stride=5)
    refuse(pkg, "aligned", f, A, pkg.F32, 1, 8, A, A, A, B + 2)
    refuse(pkg, "overlap", f, A, pkg.F16, 2, 8, A, A, A, A + 16)
    refuse(pkg, "overlap", f, A, pkg.F16, 2, 8, A, A, A, A, grad_stride=16)
    refuse(pkg, "overlap", f, A, pkg.F16, 1, 8, A, A, A, A + 14)
    f(None, pkg.F16, 0, 8, None, None, None, None)


def test_policy_refusals(pkg):
    ok = pkg.policy_hparams(0.2, 0.28, 3.0, 0.1)

    def vector(hp=ok, logp=A, tokens=4, adv=A, w=A, stat=A, ref=A, flags=0):
        pkg.policy_loss_logp(logp, tokens, adv, w, hp, stat, ref_logp=ref, flags=flags)

    for bad in ((-0.1, 0.2), (1.5, 0.2), (0.2, -0.1), (math.nan, 0.2), (0.2, math.nan)):
        refuse(pkg, "clip", vector, hp=pkg.policy_hparams(*bad))
    for c in (1.0, 0.5, -2.0, math.inf, math.nan):
        refuse(pkg, "dual_clip", vector, hp=pkg.policy_hparams(0.2, 0.2, c))
    refuse(pkg, "kl_coef", vector, hp=pkg.policy_hparams(kl_coef=math.nan))
    refuse(pkg, "kl_kind", vector, hp=pkg.policy_hparams(kl_coef=0.1, kl_kind=4))
    refuse(pkg, "ref_logp", vector, ref=None)
    refuse(pkg, "flags", vector, flags=2)
    refuse(pkg, "null", vector, adv=None)
    refuse(pkg, "null", vector, w=None)
    refuse(pkg, "null", vector, logp=None)
    refuse(pkg, "record", vector, stat=None)
    refuse(pkg, "record", vector, stat=A + 8)
    refuse(pkg, "tokens", vector, tokens=1 << 31)
    B = A + (1 << 16)
    refuse(pkg, "null logp", pkg.policy_loss, A, pkg.F16, 1, 8, A, A, A, ok, None, B, A, ref_logp=A)
    refuse(pkg, "overlap", pkg.policy_loss, A, pkg.F16, 2, 8, A, A, A, ok, A, A + 4, A, ref_logp=A)
    refuse(pkg, "vocab", pkg.policy_loss, A, pkg.F16, 2, 0, A, A, A, ok, A, B, A, ref_logp=A)


def test_preference_refusals(pkg):
    def call(hp, stat=A, offsets=A, logp=A, tokens=4, pairs=1, flags=0):
        pkg.preference_loss(logp, tokens, offsets, pairs, hp, stat, flags=flags)

    ok = pkg.preference_hparams(0.1)
    for beta in (0.0, -1.0, math.inf, math.nan):
        refuse(pkg, "beta", call, pkg.preference_hparams(beta))
    refuse(pkg, "margin", call, pkg.preference_hparams(0.1, margin=math.inf))
    refuse(pkg, "kind", call, pkg.preference_hparams(0.1, kind=3))
    for e in (-0.1, 0.6, math.nan):
        refuse(pkg, "label_smoothing", call, pkg.preference_hparams(0.1, label_smoothing=e))
    refuse(pkg, "label_smoothing", call, pkg.preference_hparams(0.1, label_smoothing=0.1, kind=pkg.PREF_IPO))
    bad = pkg.preference_hparams(0.1)
    bad.length_mean = 2
    refuse(pkg, "length_mean", call, bad)
    refuse(pkg, "record", call, ok, stat=None)
    refuse(pkg, "offsets", call, ok, offsets=None)
    refuse(pkg, "logp", call, ok, logp=None)
    refuse(pkg, "tokens", call, ok, tokens=1 << 31)
    refuse(pkg, "pairs", call, ok, pairs=1 << 31)
    refuse(pkg, "flags", call, ok, flags=4)


@pytest.mark.parametrize("kl_kind", [1, 2, 3])
@pytest.mark.parametrize("dual", [0.0, 3.0])
def test_oracle_policy_gradient_is_autograds(kl_kind, dual):
    g = torch.Generator().manual_seed(kl_kind)
    n = 200
    z = torch.randn(n, 11, generator=g, dtype=Q.F64)
    y = torch.randint(0, 11, (n,), generator=g)
    a, w = torch.randn(n, generator=g, dtype=Q.F64), torch.rand(n, generator=g, dtype=Q.F64)
    z.requires_grad_()
    logp = z.log_softmax(1).gather(1, y[:, None])[:, 0]
    old = (logp + torch.randn(n, generator=g, dtype=Q.F64) * 0.8).detach()
    ref = (logp + torch.randn(n, generator=g, dtype=Q.F64) * 0.5).detach()
    r, d = (logp - old).exp(), logp - ref
    best = torch.minimum(r * a, r.clamp(0.8, 1.28) * a)
    if dual:
        best = torch.where(a < 0, torch.maximum(best, dual * a), best)
    k = {1: d, 2: d * d / 2, 3: (-d).exp() + d - 1}[kl_kind]
    loss = (w * (0.1 * k - best)).sum()
    loss.backward()
    l, kk, coef, _ = Q.policy(logp.detach(), old, ref, a, w, torch.ones(n, dtype=torch.bool), 0.2, 0.28, dual, 0.1, kl_kind)
    assert abs(float((w * (l + 0.1 * kk)).sum().detach()) - float(loss.detach())) < 1e-12 * n
    _, _, p, takes = Q.logprob(z.detach(), y)
    assert (Q.logits_grad(p, y, takes, coef) - z.grad).abs().max() < 1e-12


@pytest.mark.parametrize("kind,mean,smoothing", [(0, False, 0.0), (0, True, 0.1), (1, False, 0.0), (2, True, 0.0)])
def test_oracle_preference_gradient_is_autograds(kind, mean, smoothing):
    g = torch.Generator().manual_seed(kind)
    offsets = [0, 3, 3, 9, 14, 20, 30]
    logp = torch.randn(31, generator=g, dtype=Q.F64, requires_grad=True)
    ref = torch.randn(31, generator=g, dtype=Q.F64)
    mask = (torch.rand(31, generator=g) < 0.8).to(torch.uint8)
    total = 0.0
    for i in range(3):
        s = []
        for q in (2 * i, 2 * i + 1):
            m = mask[offsets[q]:offsets[q + 1]].to(Q.F64)
            v = ((logp - ref)[offsets[q]:offsets[q + 1]] * m).sum()
            s.append(v / m.sum().clamp(min=1) if mean else v)
        h = 0.3 * (s[0] - s[1]) - 0.05
        if kind == 0:
            total = total - (1 - smoothing) * torch.nn.functional.logsigmoid(h) - smoothing * torch.nn.functional.logsigmoid(-h)
        elif kind == 1:
            total = total + (1 - h).clamp(min=0)
        else:
            total = total + (h / 0.3 - 0.5 / 0.3) ** 2
    (total / 3).backward()
    loss, _, _, coef, _ = Q.preference(logp.detach(), ref, mask, offsets, 3, 0.3, 0.05, smoothing, kind, mean)
    assert abs(loss - float(total) / 3) < 1e-12 and (coef - logp.grad).abs().max() < 1e-12


def test_headers_are_plain_c(tmp_path):
    """The three headers compile as C with nothing but each other."""
    import os
    import shutil
    import subprocess
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "headers.c"
    src.write_text("#include \"rlcu_act8.h\"\n#include \"rlcu_losses.h\"\n#include \"rlcu_adamw.h\"\n"
                   "typedef char a[sizeof(rlcu_policy_stat) == 32 && sizeof(rlcu_preference_stat) == 32 ? 1 : -1];\n"
                   "int main(void) { return RLCU_ACT8_BLOCK == 128 ? 0 : 1; }\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-Werror", "-pedantic", "-I", os.path.join(root, "include"), "-c", str(src),
                    "-o", str(tmp_path / "headers.o")], check=True)


def test_vectors_that_overlap_or_are_not_aligned_are_refused(pkg):
    """The log-probabilities a policy loss writes would be read as the old ones; odd addresses would fault the GPU."""
    B, D = A + (1 << 16), A + (2 << 16)
    ok = pkg.policy_hparams(0.2, 0.28, 3.0, 0.1)

    def policy(old=B, ref=B, adv=B, w=B, logp=D, targets=B, scaler=None):
        pkg.policy_loss(A, pkg.F16, 2, 8, targets, adv, w, ok, logp, None, A, old_logp=old, ref_logp=ref, scaler=scaler)

    for name in ("old", "ref", "adv", "w"):
        refuse(pkg, "overlap", policy, **{name: D})
        refuse(pkg, "overlap", policy, **{name: D + 4})
        refuse(pkg, "aligned", policy, **{name: B + 2})
    for name in ("logp", "targets", "scaler"):
        refuse(pkg, "aligned", policy, **{name: B + 1})

    def vector(coef=D, logp=B, ref=B, adv=B, w=B, old=B):
        pkg.policy_loss_logp(logp, 4, adv, w, ok, A, coef=coef, old_logp=old, ref_logp=ref)

    for name in ("logp", "ref", "adv", "w", "old"):
        refuse(pkg, "overlap", vector, **{name: D + 4})
        refuse(pkg, "aligned", vector, **{name: B + 3})
    refuse(pkg, "aligned", vector, coef=D + 2)

    def preference(coef=D, logp=B, ref=B, offsets=B, weight=B, rewards=B):
        pkg.preference_loss(logp, 4, offsets, 1, pkg.preference_hparams(0.1), A, coef=coef, rewards=rewards, ref_logp=ref, pair_weight=weight)

    for name in ("logp", "ref"):
        refuse(pkg, "overlap", preference, **{name: D - 8})
    for name in ("coef", "logp", "ref", "offsets", "weight", "rewards"):
        refuse(pkg, "aligned", preference, **{name: B + 2})
    refuse(pkg, "aligned", pkg.token_logprob, A, pkg.F16, 1, 8, B + 2, B)
    refuse(pkg, "aligned", pkg.token_logprob, A, pkg.F16, 1, 8, B, B + 2)
    refuse(pkg, "aligned", pkg.token_logprob_grad, A, pkg.F16, 1, 8, B, B + 1, B, D)
