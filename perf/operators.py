"""What is measured of the training-step operators: token log-probabilities of logits, the clipped policy
loss, the preference loss, 8-bit activation checkpoints and the RMSNorm that reads them.

``listed()`` gives the cases, ``prepare`` what a trainer has in hand before the call, ``run`` one pass: with
``own`` false in elementary torch operations, with ``own`` true through this repository's package.  ``exact``
computes the same from the definitions in 64 bits.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZES = {"f16": 2, "bf16": 2, "f32": 4}
BLOCK = 128                     # columns that share one scale of an 8-bit checkpoint
EPS = 1e-6                      # of the RMSNorm
CLIP_LOW, CLIP_HIGH = 0.2, 0.28
DUAL_CLIP = 3.0
BETA = 0.1                      # of the preference loss
SMOOTH = 0.05


# ---------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------

def listed():
    return [
        # scoring rollouts with the reference model: 2048 tokens of the 151936-entry vocabulary, forward only
        {"name": "logprob-2048x151936-bf16", "op": "logprob", "rows": 2048, "vocab": 151936, "dtype": "bf16", "grad": False, "skip": 0.1},
        # a preference or SFT micro-batch whose vocabulary is odd, FP32 logits, forward and gradient
        {"name": "logprob-grad-1000x50001-f32", "op": "logprob", "rows": 1000, "vocab": 50001, "dtype": "f32", "grad": True, "skip": 0.1},
        # the trainer's 256-row chunk of the output projection, FP16 with a loss scale
        {"name": "policy-256x151936-f16", "op": "policy", "rows": 256, "vocab": 151936, "dtype": "f16", "kl": 0.04, "off_policy": True, "skip": 0.1},
        # a whole micro-batch at once
        {"name": "policy-4096x151936-bf16", "op": "policy", "rows": 4096, "vocab": 151936, "dtype": "bf16", "kl": 0.04, "off_policy": True, "skip": 0.1},
        # the loss alone, from log-probabilities that are there already
        {"name": "policy-logp-16384", "op": "policy_logp", "rows": 16384, "kl": 0.04, "off_policy": True, "skip": 0.3},
        # one pair of short answers: latency
        {"name": "preference-1x200", "op": "preference", "pairs": 1, "length": 200, "mask": True, "ref": True, "kind": "sigmoid", "mean": False},
        # a large ragged batch of pairs
        {"name": "preference-128x2048", "op": "preference", "pairs": 128, "length": 2048, "mask": True, "ref": True, "kind": "sigmoid", "mean": False},
        # checkpoint of a few tokens, there and back: latency
        {"name": "act8-3x1024-f16", "op": "act8", "rows": 3, "cols": 1024, "dtype": "f16"},
        # checkpoint of one layer's input of a long micro-batch, there and back
        {"name": "act8-16384x4096-bf16", "op": "act8", "rows": 16384, "cols": 4096, "dtype": "bf16"},
        # first step of a layer's recomputation
        {"name": "norm-8192x1024-f16", "op": "norm", "rows": 8192, "cols": 1024, "dtype": "f16", "grad": False, "residual": False},
        # last step of a layer's backward pass, joined with the residual's gradient
        {"name": "norm-grad-16384x4096-bf16", "op": "norm", "rows": 16384, "cols": 4096, "dtype": "bf16", "grad": True, "residual": True},
        # few rows, a width that fills neither blocks nor vectors
        {"name": "norm-grad-77x1001-f32", "op": "norm", "rows": 77, "cols": 1001, "dtype": "f32", "grad": True, "residual": False},
    ]


def _spread(rng, low, high):
    """A whole number, uniform over its logarithm."""
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["logprob", "policy", "policy_logp", "preference", "act8", "norm"])
    dtype = rng.choice(["f16", "bf16", "f32"])
    if op in ("logprob", "policy"):
        vocab = rng.choice([_spread(rng, 500, 151936), 8 * _spread(rng, 2000, 18992)])
        rows = _spread(rng, 1, min(4096, 4096 * 151936 // vocab // SIZES[dtype] * 2))
        case = {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "skip": rng.choice([0.0, 0.1, 0.5])}
        if op == "logprob":
            return {**case, "grad": rng.random() < 0.6}
        return {**case, "kl": rng.choice([0.0, 0.04, 0.1]), "off_policy": rng.random() < 0.8}
    if op == "policy_logp":
        return {"op": op, "rows": _spread(rng, 1, 65536), "kl": rng.choice([0.0, 0.04, 0.1]), "off_policy": True, "skip": rng.choice([0.0, 0.3])}
    if op == "preference":
        length = _spread(rng, 1, 4096)
        return {"op": op, "pairs": _spread(rng, 1, min(256, 2 * 128 * 2048 // length)), "length": length, "mask": rng.random() < 0.7,
                "ref": rng.random() < 0.8, "kind": rng.choice(["sigmoid", "sigmoid", "hinge", "ipo"]), "mean": rng.random() < 0.3}
    cols = rng.choice([_spread(rng, 1, 8192), 128 * _spread(rng, 1, 64)])
    rows = _spread(rng, 1, min(32768, 16384 * 4096 // cols // SIZES[dtype] * 2))
    case = {"op": op, "rows": rows, "cols": cols, "dtype": dtype}
    if op == "norm":
        grad = rng.random() < 0.6
        case.update(grad=grad, residual=grad and rng.random() < 0.5)
    return case


def work(case):
    op = case["op"]
    if op in ("logprob", "policy"):
        n, size = case["rows"] * case["vocab"], SIZES[case["dtype"]]
        read = n * (1 - case["skip"]) * size           # rows that take no part are not read
        wrote = n * size if op == "policy" or case["grad"] else 0
        flops = n * (1 - case["skip"]) * (4 + (4 if wrote else 0))
        return {"bytes": read + wrote + 28 * case["rows"], "flops": flops}
    if op == "policy_logp":
        return {"bytes": case["rows"] * 4 * (4 + bool(case["kl"])), "flops": 20 * case["rows"]}
    if op == "preference":
        tokens = case["pairs"] * case["length"]        # of both sequences of every pair
        return {"bytes": tokens * (8 + 4 * case["ref"] + case["mask"]) + 28 * case["pairs"], "flops": 4 * tokens + 40 * case["pairs"]}
    n, size = case["rows"] * case["cols"], SIZES[case["dtype"]]
    held = n + case["rows"] * -(-case["cols"] // BLOCK)
    if op == "act8":
        return {"bytes": 2 * (n * size + held), "flops": 4 * n}
    if not case["grad"]:
        return {"bytes": held + n * size + 4 * case["rows"] + 4 * case["cols"], "flops": 5 * n}
    return {"bytes": held + n * size * (2 + case["residual"]) + 8 * case["cols"], "flops": 12 * n}


# ---------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _scaler(scale):
    """A loss-scale record (scale, growth_tracker, step, skipped, growth_interval, beta1, beta2, grad_mul) on the device."""
    s = torch.zeros(8, dtype=torch.float32, device="cuda")
    s[0], s[5], s[6] = scale, 0.9, 0.999
    s.view(torch.int32)[4] = 1000
    return s


def _off_the_borders(delta):
    """Log ratios within 1e-4 of a clip border are moved away from it: which branch such a token takes is decided by
    the last bits of its log-probability, and the gradient jumps there."""
    for border in (math.log1p(-CLIP_LOW), math.log1p(CLIP_HIGH), math.log(DUAL_CLIP)):
        near = (delta - border).abs() < 1e-4
        delta = torch.where(near, torch.full_like(delta, border - 3e-4), delta)
    return delta


def _policy_inputs(s, case, g, logp):
    rows = case["rows"]
    s["advantage"] = torch.randn(rows, device="cuda", generator=g)
    taking = torch.rand(rows, device="cuda", generator=g) >= case["skip"]
    s["weight"] = taking.float() / max(1, int(taking.sum()))
    delta = _off_the_borders(torch.randn(rows, device="cuda", generator=g) * 0.25)
    s["old"] = (logp - delta) if case["off_policy"] else None
    s["ref"] = (logp + torch.randn(rows, device="cuda", generator=g) * 0.3) if case["kl"] else None
    s["stat"] = torch.zeros(8, dtype=torch.int32, device="cuda")


def _offsets(pairs, length, seed):
    """2*pairs sequences packed into pairs*length tokens, cut at random places: ragged, a few of them empty."""
    g = torch.Generator().manual_seed(seed)
    cuts = torch.randint(0, pairs * length + 1, (2 * pairs - 1,), generator=g).sort().values
    return torch.cat([torch.zeros(1, dtype=torch.int64), cuts, torch.tensor([pairs * length])]).to(torch.int32)


def prepare(case, seed):
    g, op = _generator(seed), case["op"]
    s = {"case": case}
    if op in ("logprob", "policy"):
        rows, vocab, dt = case["rows"], case["vocab"], DTYPES[case["dtype"]]
        z = torch.randn(rows, vocab, device="cuda", generator=g, dtype=dt).mul_(2)
        y = torch.randint(0, vocab, (rows,), device="cuda", generator=g, dtype=torch.int32)
        # a sampled token is a likely one
        z[torch.arange(rows, device="cuda"), y.long()] += (4 + 12 * torch.rand(rows, device="cuda", generator=g)).to(dt)
        s.update(logits=z, temperature=1.0, scaler=_scaler(65536.0 if case["dtype"] == "f16" else 1.0),
                 logp=torch.empty(rows, device="cuda"), lse=torch.empty(rows, device="cuda"))
        if op == "logprob":
            skip = torch.rand(rows, device="cuda", generator=g) < case["skip"]
            s["targets"] = torch.where(skip, torch.full_like(y, -100), y)
            s["coef"] = torch.randn(rows, device="cuda", generator=g) / rows
            s["grad"] = torch.empty_like(z) if case["grad"] else None
        else:
            s["targets"] = y
            logp = torch.cat([c.float().log_softmax(1).gather(1, i.long()[:, None])[:, 0] for c, i in zip(z.split(256), y.split(256))])
            _policy_inputs(s, case, g, logp)
            s["grad"] = torch.empty_like(z)
    elif op == "policy_logp":
        s["logp"] = torch.rand(case["rows"], device="cuda", generator=g).clamp_(min=1e-4).log_() * 0.7
        s["coef"] = torch.empty(case["rows"], device="cuda")
        _policy_inputs(s, case, g, s["logp"])
    elif op == "preference":
        tokens = case["pairs"] * case["length"] + 5    # a few rows of padding behind the last sequence
        s.update(tokens=tokens, offsets=_offsets(case["pairs"], case["length"], seed).cuda(),
                 logp=-torch.rand(tokens, device="cuda", generator=g) * 2, coef=torch.empty(tokens, device="cuda"),
                 rewards=torch.empty(2 * case["pairs"], device="cuda"), stat=torch.zeros(8, dtype=torch.int32, device="cuda"))
        s["ref"] = s["logp"] + torch.randn(tokens, device="cuda", generator=g) * 0.05 if case["ref"] else None
        s["mask"] = (torch.rand(tokens, device="cuda", generator=g) < 0.8).to(torch.uint8) if case["mask"] else None
    else:
        rows, cols, dt = case["rows"], case["cols"], DTYPES[case["dtype"]]
        # activations of a residual stream: channels of different size, a few of them far larger
        size = torch.exp(0.5 * torch.randn(cols, device="cuda", generator=g))
        size = torch.where(torch.rand(cols, device="cuda", generator=g) < 0.004, size * 40, size)
        x = torch.randn(rows, cols, device="cuda", generator=g).mul_(size).to(dt)
        blocks, stride = -(-cols // BLOCK), -(-cols // 16) * 16
        s.update(codes=torch.zeros(rows, stride, dtype=torch.uint8, device="cuda"),
                 scales=torch.zeros(rows, blocks, dtype=torch.uint8, device="cuda"))
        if op == "act8":
            s.update(x=x, out=torch.empty_like(x))
        else:
            codes, exponent = _encode(x)
            s["codes"][:, :cols] = codes.view(torch.uint8)
            s["scales"] = (exponent + 127).to(torch.uint8)
            s["weight"] = 1 + 0.2 * torch.randn(cols, device="cuda", generator=g)
            if case["grad"]:
                s["dy"] = torch.randn(rows, cols, device="cuda", generator=g).mul_(1e-2).to(dt)
                s["dres"] = torch.randn(rows, cols, device="cuda", generator=g).mul_(1e-2).to(dt) if case["residual"] else None
                s.update(dx=torch.empty_like(x), dw=torch.empty(cols, device="cuda"))
                # scratch for the weight gradient: what the package says it needs is at most this
                s["workspace"] = torch.empty(16 << 20, dtype=torch.uint8, device="cuda")
            else:
                s.update(y=torch.empty_like(x), rstd=torch.empty(rows, device="cuda"))
    return s


# ---------------------------------------------------------------------------------------------------------
# the package's calls
# ---------------------------------------------------------------------------------------------------------

_package = None


def _pkg():
    global _package
    if _package is None:
        name = "rlcu_b200"
        if name not in sys.modules:
            at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rl.cu_b200")
            spec = importlib.util.spec_from_file_location(name, os.path.join(at, "__init__.py"), submodule_search_locations=[at])
            sys.modules[name] = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(sys.modules[name])
        _package = sys.modules[name]
    return _package


def _at(t):
    return None if t is None else t.data_ptr()


def _policy_answer(s, *more):
    return {"stat": s["stat"].view(torch.float32)[:4], "counts": s["stat"][4:6], **dict(more)}


def _run_own(s):
    p, case, stream = _pkg(), s["case"], torch.cuda.current_stream().cuda_stream
    op = case["op"]
    if op in ("logprob", "policy"):
        block = (_at(s["logits"]), {"f16": p.F16, "bf16": p.BF16, "f32": p.F32}[case["dtype"]], case["rows"], case["vocab"], _at(s["targets"]))
    if op == "logprob":
        p.token_logprob(*block, _at(s["logp"]), lse=_at(s["lse"]), inv_temperature=1.0 / s["temperature"], stream=stream)
        if not case["grad"]:
            return {"logp": s["logp"], "lse": s["lse"]}
        p.token_logprob_grad(*block, _at(s["lse"]), _at(s["coef"]), _at(s["grad"]), inv_temperature=1.0 / s["temperature"],
                             scaler=_at(s["scaler"]), stream=stream)
        return {"logp": s["logp"], "lse": s["lse"], "grad": s["grad"]}
    if op in ("policy", "policy_logp"):
        hp = p.policy_hparams(CLIP_LOW, CLIP_HIGH, DUAL_CLIP, case["kl"])
    if op == "policy":
        p.policy_loss(*block, _at(s["advantage"]), _at(s["weight"]), hp, _at(s["logp"]), _at(s["grad"]), _at(s["stat"]), old_logp=_at(s["old"]),
                      ref_logp=_at(s["ref"]), inv_temperature=1.0 / s["temperature"], scaler=_at(s["scaler"]), stream=stream)
        return _policy_answer(s, ("logp", s["logp"]), ("grad", s["grad"]))
    if op == "policy_logp":
        p.policy_loss_logp(_at(s["logp"]), case["rows"], _at(s["advantage"]), _at(s["weight"]), hp, _at(s["stat"]), coef=_at(s["coef"]),
                           old_logp=_at(s["old"]), ref_logp=_at(s["ref"]), stream=stream)
        return _policy_answer(s, ("coef", s["coef"]))
    if op == "preference":
        kind = {"sigmoid": p.PREF_SIGMOID, "hinge": p.PREF_HINGE, "ipo": p.PREF_IPO}[case["kind"]]
        hp = p.preference_hparams(BETA, label_smoothing=SMOOTH if case["kind"] == "sigmoid" else 0.0, kind=kind, length_mean=case["mean"])
        p.preference_loss(_at(s["logp"]), s["tokens"], _at(s["offsets"]), case["pairs"], hp, _at(s["stat"]), coef=_at(s["coef"]),
                          rewards=_at(s["rewards"]), ref_logp=_at(s["ref"]), mask=_at(s["mask"]), stream=stream)
        return {"stat": s["stat"].view(torch.float32)[:2], "counts": s["stat"][2:4], "coef": s["coef"], "rewards": s["rewards"]}
    rows, cols, stride = case["rows"], case["cols"], s["codes"].shape[1]
    dt = {"f16": p.F16, "bf16": p.BF16, "f32": p.F32}[case["dtype"]]
    held = (_at(s["codes"]), _at(s["scales"]), rows, cols)
    if op == "act8":
        p.act8_store(_at(s["x"]), dt, rows, cols, _at(s["codes"]), _at(s["scales"]), code_stride=stride, stream=stream)
        p.act8_load(*held, _at(s["out"]), dt, code_stride=stride, stream=stream)
        return {"out": s["out"], "scales": s["scales"]}
    if not case["grad"]:
        p.act8_rmsnorm(*held, _at(s["weight"]), p.F32, EPS, _at(s["y"]), dt, rstd=_at(s["rstd"]), code_stride=stride, stream=stream)
        return {"y": s["y"], "rstd": s["rstd"]}
    p.act8_rmsnorm_grad(*held, _at(s["weight"]), p.F32, EPS, _at(s["dy"]), dt, _at(s["dx"]), _at(s["dw"]), _at(s["workspace"]), s["workspace"].numel(),
                        dresidual=_at(s["dres"]), code_stride=stride, stream=stream)
    return {"dx": s["dx"], "dw": s["dw"]}


# ---------------------------------------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------------------------------------

def _logprob(z, y, taking):
    """(logp, lse) of FP32 logits; rows that take no part get zeros."""
    top = z.max(1, keepdim=True).values
    log_sum = (z - top).exp().sum(1, keepdim=True).log()
    at = z.gather(1, y.clamp(0, z.shape[1] - 1)[:, None])
    zero = torch.zeros((), device=z.device)
    return torch.where(taking, (at - top - log_sum)[:, 0], zero), torch.where(taking, (top + log_sum)[:, 0], zero)


def _logits_grad(z, y, taking, logp, coef):
    """coef * (one-hot - softmax) with the softmax taken relative to the target's own probability."""
    at = z.gather(1, y.clamp(0, z.shape[1] - 1)[:, None])
    grad = -((z - at + logp[:, None]).exp())
    grad.scatter_add_(1, y.clamp(0, z.shape[1] - 1)[:, None], torch.ones_like(at))
    return torch.where((taking & (coef != 0))[:, None], grad * coef[:, None], torch.zeros((), device=z.device))


def _policy(s, case, logp, taking):
    """(stat, counts, coef) of the clipped policy loss on log-probabilities."""
    zero = torch.zeros((), device=logp.device)
    a, w = s["advantage"], s["weight"]
    ratio = (logp - s["old"]).exp() if s["old"] is not None else torch.ones_like(logp)
    clipped = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * a
    cut = clipped < ratio * a
    gain = torch.where(cut, clipped, ratio * a)
    slope = torch.where(cut, zero, ratio * a)
    floor = DUAL_CLIP * a
    dual = (a < 0) & (floor > gain)
    gain, slope, cut = torch.where(dual, floor, gain), torch.where(dual, zero, slope), cut | dual
    kl, kl_slope = torch.zeros_like(logp), torch.zeros_like(logp)
    if case["kl"]:
        d = s["ref"] - logp
        kl, kl_slope = d.expm1() - d, -d.expm1()
    coef = torch.where(taking, w * (case["kl"] * kl_slope - slope), zero)
    policy, kl = (torch.where(taking, w * v, zero).double().sum() for v in (-gain, kl))
    stat = torch.stack([policy + case["kl"] * kl, policy, kl, torch.where(taking, w, zero).double().sum()]).float()
    return stat, torch.stack([taking.sum(), (taking & cut).sum()]).int(), coef


def _preference(s, case):
    pairs, offsets = case["pairs"], s["offsets"].long()
    place = torch.arange(s["tokens"], device="cuda")
    of = torch.searchsorted(offsets[1:], place, right=True)
    counts = of < 2 * pairs
    if s["mask"] is not None:
        counts = counts & (s["mask"] != 0)
    of = of.clamp(max=2 * pairs - 1)
    value = s["logp"] - s["ref"] if s["ref"] is not None else s["logp"]
    total = torch.zeros(2 * pairs, dtype=torch.float64, device="cuda").index_add_(0, of, torch.where(counts, value, 0.0).double())
    share = torch.ones(2 * pairs, dtype=torch.float64, device="cuda")
    if case["mean"]:
        share = 1 / torch.zeros_like(total).index_add_(0, of, counts.double()).clamp(min=1)
    total = total * share
    h = BETA * (total[0::2] - total[1::2])
    e = SMOOTH
    if case["kind"] == "sigmoid":
        loss = (1 - e) * torch.log1p(torch.exp(-h.abs())) + (1 - e) * (-h).clamp(min=0) + e * torch.log1p(torch.exp(-h.abs())) + e * h.clamp(min=0)
        slope = BETA * (e / (1 + torch.exp(-h)) - (1 - e) / (1 + torch.exp(h)))
    elif case["kind"] == "hinge":
        loss, slope = (1 - h).clamp(min=0), torch.where(h < 1, -BETA, 0.0).double()
    else:
        d = h / BETA - 1 / (2 * BETA)
        loss, slope = d * d, 2 * d
    per = torch.stack([slope, -slope], 1).reshape(-1) * share / pairs
    coef = torch.where(counts, per.float()[of], 0.0)
    stat = torch.stack([loss.mean(), h.mean()]).float()
    right = torch.stack([torch.tensor(pairs, device="cuda"), (total[0::2] > total[1::2]).sum()]).int()
    return {"stat": stat, "counts": right, "coef": coef, "rewards": (BETA * total).float()}


def _blocks(x):
    """[rows, cols] as [rows, blocks, BLOCK], filled up with zeros."""
    return torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK)).reshape(x.shape[0], -1, BLOCK)


def _encode(x):
    """(e4m3 codes, exponents of two) of each block of 128 columns."""
    b = _blocks(x.float())
    part, power = torch.frexp(b.abs().amax(2))
    exponent = torch.where(part > 0.875, power - 8, power - 9).clamp(-127, 120)      # 448 = 0.875 * 2^9
    exponent = torch.where(part == 0, torch.full_like(exponent, -127), exponent)
    codes = torch.ldexp(b, -exponent[:, :, None]).to(torch.float8_e4m3fn)
    return codes.reshape(x.shape[0], -1)[:, :x.shape[1]], exponent


def _decode(codes, exponent):
    b = _blocks(codes.float())
    return torch.ldexp(b, exponent[:, :, None]).reshape(codes.shape[0], -1)[:, :codes.shape[1]]


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op in ("logprob", "policy"):
        z, y = s["logits"].float() / s["temperature"], s["targets"].long()
        taking = (y >= 0) & (y < case["vocab"])
        scale = s["scaler"][0] / s["temperature"]
    if op == "logprob":
        logp, lse = _logprob(z, y, taking)
        if not case["grad"]:
            return {"logp": logp, "lse": lse}
        return {"logp": logp, "lse": lse, "grad": _logits_grad(z, y, taking, logp, s["coef"] * scale).to(s["logits"].dtype)}
    if op == "policy":
        taking = taking & (s["weight"] != 0)
        logp, _ = _logprob(z, y, taking)
        stat, counts, coef = _policy(s, case, logp, taking)
        return {"stat": stat, "counts": counts, "logp": logp, "grad": _logits_grad(z, y, taking, logp, coef * scale).to(s["logits"].dtype)}
    if op == "policy_logp":
        stat, counts, coef = _policy(s, case, s["logp"], s["weight"] != 0)
        return {"stat": stat, "counts": counts, "coef": coef}
    if op == "preference":
        return _preference(s, case)
    if op == "act8":
        codes, exponent = _encode(s["x"])
        return {"out": _decode(codes, exponent).to(s["x"].dtype), "scales": (exponent + 127).to(torch.uint8)}
    x = _decode(s["codes"][:, :case["cols"]].view(torch.float8_e4m3fn), s["scales"].int() - 127)
    rstd = (x.square().mean(1, keepdim=True) + EPS).rsqrt()
    if not case["grad"]:
        return {"y": (x * rstd * s["weight"]).to(s["y"].dtype), "rstd": rstd[:, 0]}
    dy = s["dy"].float()
    wdy = dy * s["weight"]
    dx = rstd * (wdy - x * (rstd.square() * (wdy * x).mean(1, keepdim=True)))
    if s["dres"] is not None:
        dx = dx + s["dres"].float()
    return {"dx": dx.to(s["dx"].dtype), "dw": (dy * x * rstd).sum(0)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------

def _exact_policy(s, case, logp, taking):
    """Token by token on the host: (stat, counts, coef)."""
    host = lambda t: None if t is None else t.double().cpu().tolist()  # noqa: E731
    logp, old, ref, a, w, taking = host(logp), host(s["old"]), host(s["ref"]), host(s["advantage"]), host(s["weight"]), taking.cpu().tolist()
    coef, policy, kl, weight, tokens, cuts = [0.0] * len(logp), [], [], [], 0, 0
    for t, takes in enumerate(taking):
        if not takes:
            continue
        r = math.exp(logp[t] - old[t]) if old else 1.0
        free, held = r * a[t], min(max(r, 1 - CLIP_LOW), 1 + CLIP_HIGH) * a[t]
        best, slope = (free, free) if free <= held else (held, 0.0)
        if a[t] < 0 and best < DUAL_CLIP * a[t]:
            best, slope = DUAL_CLIP * a[t], 0.0
        cuts += slope == 0.0 and free != 0.0
        tokens += 1
        k = slope_k = 0.0
        if case["kl"]:
            u = math.exp(ref[t] - logp[t])
            k, slope_k = u - (ref[t] - logp[t]) - 1, 1 - u
        policy.append(-w[t] * best)
        kl.append(w[t] * k)
        weight.append(w[t])
        coef[t] = w[t] * (case["kl"] * slope_k - slope)
    p, k = math.fsum(policy), math.fsum(kl)
    stat = torch.tensor([p + case["kl"] * k, p, k, math.fsum(weight)], dtype=torch.float64, device="cuda")
    return stat, torch.tensor([tokens, cuts], dtype=torch.int32, device="cuda"), torch.tensor(coef, dtype=torch.float64, device="cuda")


def _exact_logits(s, case):
    z, y, dt = s["logits"], s["targets"].long(), torch.float64
    rows, vocab = z.shape
    taking = (y >= 0) & (y < vocab)
    if case["op"] == "policy":
        taking = taking & (s["weight"] != 0)
    logp, lse = torch.zeros(rows, dtype=dt, device="cuda"), torch.zeros(rows, dtype=dt, device="cuda")
    parts = [range(i, min(i + 128, rows)) for i in range(0, rows, 128)]
    for p in parts:
        at = slice(p.start, p.stop)
        full = torch.logsumexp(z[at].double() / s["temperature"], 1)
        own_z = z[at].double().gather(1, y[at].clamp(0, vocab - 1)[:, None])[:, 0] / s["temperature"]
        lse[at] = full * taking[at]
        logp[at] = (own_z - full) * taking[at]
    answer = {"logp": logp}
    if case["op"] == "policy":
        answer["stat"], answer["counts"], coef = _exact_policy(s, case, logp, taking)
    else:
        answer["lse"] = lse
        if not case["grad"]:
            return answer
        coef = s["coef"].double()
    coef = coef * s["scaler"][0].double() / s["temperature"] * taking
    grad = torch.zeros(rows, vocab, dtype=dt, device="cuda")
    for p in parts:
        at = slice(p.start, p.stop)
        hot = torch.zeros(len(p), vocab, dtype=dt, device="cuda").scatter_(1, y[at].clamp(0, vocab - 1)[:, None], 1.0)
        grad[at] = coef[at, None] * (hot - torch.softmax(z[at].double() / s["temperature"], 1))
    answer["grad"] = grad
    return answer


def _exact_preference(s, case):
    host = lambda t: None if t is None else t.double().cpu().tolist()  # noqa: E731
    logp, ref, mask, offsets = host(s["logp"]), host(s["ref"]), host(s["mask"]), s["offsets"].cpu().tolist()
    pairs = case["pairs"]
    coef, sums, lengths, losses, hs, right = [0.0] * len(logp), [], [], [], [], 0
    places = [[t for t in range(offsets[q], offsets[q + 1]) if mask is None or mask[t]] for q in range(2 * pairs)]
    for at in places:
        n = max(1, len(at)) if case["mean"] else 1
        lengths.append(n)
        sums.append(math.fsum(logp[t] - (ref[t] if ref else 0.0) for t in at) / n)
    for i in range(pairs):
        c, r = sums[2 * i], sums[2 * i + 1]
        h = BETA * (c - r)
        if case["kind"] == "sigmoid":
            up, down = 1 / (1 + math.exp(-h)), 1 / (1 + math.exp(h))
            loss, slope = -(1 - SMOOTH) * math.log(up) - SMOOTH * math.log(down), BETA * (SMOOTH * up - (1 - SMOOTH) * down)
        elif case["kind"] == "hinge":
            loss, slope = max(0.0, 1 - h), -BETA if h < 1 else 0.0
        else:
            loss, slope = (c - r - 1 / (2 * BETA)) ** 2, 2 * (c - r - 1 / (2 * BETA))
        losses.append(loss)
        hs.append(h)
        right += c > r
        for q, sign in ((2 * i, 1), (2 * i + 1, -1)):
            for t in places[q]:
                coef[t] = sign * slope / lengths[q] / pairs
    tensor = lambda v, dt=torch.float64: torch.tensor(v, dtype=dt, device="cuda")  # noqa: E731
    return {"stat": tensor([math.fsum(losses) / pairs, math.fsum(hs) / pairs]), "counts": tensor([pairs, right], torch.int32),
            "coef": tensor(coef), "rewards": tensor([BETA * v for v in sums])}


def _exact_values(x):
    """(values, exponents + 127) an 8-bit checkpoint of x stands for: rounding spelled out on the grid of e4m3."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -cols % BLOCK)).reshape(rows, -1, BLOCK)
    top = x.abs().amax(2, keepdim=True)
    e = torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** -127)))
    e = torch.where(top > 448 * torch.exp2(e), e + 1, e)                   # log2 may be off by its last bit
    e = torch.where(top <= 448 * torch.exp2(e - 1), e - 1, e).clamp(-127, 120)
    q = x / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    values = torch.round(q / step) * step * torch.exp2(e)
    return values.reshape(rows, -1)[:, :cols], (e[:, :, 0] + 127).to(torch.uint8)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op in ("logprob", "policy"):
        return _exact_logits(s, case)
    if op == "policy_logp":
        stat, counts, coef = _exact_policy(s, case, s["logp"], s["weight"] != 0)
        return {"stat": stat, "counts": counts, "coef": coef}
    if op == "preference":
        return _exact_preference(s, case)
    if op == "act8":
        out, scales = _exact_values(s["x"])
        return {"out": out, "scales": scales}
    cols = case["cols"]
    byte = s["codes"][:, :cols].long()
    field, part = (byte >> 3) & 15, (byte & 7).double()
    x = torch.where(field == 0, part * 2.0 ** -9, (8 + part) * torch.exp2(field.double() - 10)) * (1 - 2 * (byte >> 7)).double()
    x = x * torch.exp2(s["scales"].double() - 127).repeat_interleave(BLOCK, 1)[:, :cols]
    rstd = 1 / torch.sqrt((x * x).sum(1, keepdim=True) / cols + EPS)
    w = s["weight"].double()
    if not case["grad"]:
        return {"y": x * rstd * w, "rstd": rstd[:, 0]}
    dy = s["dy"].double()
    xhat = x * rstd
    dx = rstd * (w * dy - xhat * ((w * dy * xhat).sum(1, keepdim=True) / cols))
    if s["dres"] is not None:
        dx = dx + s["dres"].double()
    return {"dx": dx, "dw": (dy * xhat).sum(0)}
