"""The training-step operators in 64 bits (torch on the CPU), written from their definitions, and the buffers the
GPU tests put their data in: rows with a stride, at an odd offset, with guard elements around and between them."""
from __future__ import annotations

import math

import torch

F64 = torch.float64
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def kind(pkg, name):
    return {"f16": pkg.F16, "bf16": pkg.BF16, "f32": pkg.F32}[name]


def half_ulp(dtype):
    """Largest relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def rounding(values, dtype):
    """Largest absolute error of rounding `values` to `dtype` once: half a step, or half the smallest subnormal."""
    return values.abs() * half_ulp(dtype) + torch.finfo(dtype).smallest_normal * half_ulp(dtype)


class Rows:
    """A rows x cols device matrix with `pad` guard elements behind each row, starting `offset` elements into its
    allocation.  The guards hold a bit pattern that must survive every call."""

    def __init__(self, values, pad=0, offset=0):
        rows, cols = values.shape
        self.rows, self.cols, self.stride, self.offset = rows, cols, cols + pad, offset
        size = values.element_size()
        self.word = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[size]
        self.raw = torch.full((offset + rows * self.stride + 16,), 0x5A, dtype=self.word, device="cuda")
        self.all = self.raw.view(values.dtype)
        self.t = self.all[offset:offset + rows * self.stride].view(rows, self.stride)[:, :cols]
        self.t.copy_(values)

    @property
    def ptr(self):
        return self.raw.data_ptr() + self.offset * self.raw.element_size()

    def get(self):
        return self.t.cpu()

    def guards_intact(self):
        raw = self.raw.cpu()
        body = raw[self.offset:self.offset + self.rows * self.stride].view(self.rows, self.stride)
        return bool((raw[:self.offset] == 0x5A).all() and (raw[self.offset + self.rows * self.stride:] == 0x5A).all()
                    and (body[:, self.cols:] == 0x5A).all())


# ---- logits -------------------------------------------------------------------

NO_LOGIT = -1e30      # a row without a larger logit is a row of nothing but masks


def logprob(z, targets, inv_temperature=1.0, taking=None):
    """(logp, lse, softmax, taking) of logits z in 64 bits."""
    z = z.to(F64) * inv_temperature
    rows, vocab = z.shape
    y = targets.long()
    takes = (y >= 0) & (y < vocab)
    if taking is not None:
        takes = takes & taking
    masked = (z < NO_LOGIT * inv_temperature) & ~torch.isnan(z)
    z = torch.where(masked, torch.full_like(z, -math.inf), z)
    lse = torch.logsumexp(z, 1)
    lse = torch.where((z == math.inf).any(1), torch.full_like(lse, math.nan), lse)       # inf - inf
    empty = masked.all(1)
    lse = torch.where(empty, torch.full_like(lse, -math.inf), lse)
    at = z.gather(1, y.clamp(0, vocab - 1)[:, None])[:, 0]
    logp = torch.where(empty, torch.full_like(lse, -math.inf), at - lse)
    p = torch.where(empty[:, None], torch.zeros_like(z), torch.exp(z - lse[:, None]))
    zero = torch.zeros((), dtype=F64)
    return torch.where(takes, logp, zero), torch.where(takes, lse, zero), p, takes


def logits_grad(p, targets, takes, coef, factor=1.0):
    hot = torch.zeros_like(p)
    inside = (targets >= 0) & (targets < p.shape[1])
    rows = torch.nonzero(inside)[:, 0]
    hot[rows, targets.long()[rows]] = 1.0
    return torch.where((takes & (coef != 0))[:, None], coef.to(F64)[:, None] * factor * (hot - p), torch.zeros((), dtype=F64))


def logprob_error(z, targets, inv_temperature):
    """Bound on the error of a log-probability computed in FP32, per row.

    c = inv_temperature * log2 e carries two roundings (2^-23 relative), which acts like that relative change of the
    temperature: 2^-23 times the spread of the scaled logits.  Each term 2^x is off by the rounding of x (2^-24 |x| ln 2,
    x at most the spread) and by the exponential (2^-22); a sum of n positive terms taken by 128 or more threads adds
    (n / 128 + 24) roundings of 2^-24 each at most; the logarithm and the last products add a few more of the result."""
    z = z.to(F64) * inv_temperature
    fine = torch.isfinite(z) & (z > NO_LOGIT * inv_temperature)
    lo = torch.where(fine, z, torch.full_like(z, math.inf)).amin(1)
    hi = torch.where(fine, z, torch.full_like(z, -math.inf)).amax(1)
    spread = torch.where(fine.any(1), hi - lo, torch.zeros_like(hi))
    n = z.shape[1]
    return spread * 2.0 ** -22 + 2.0 ** -21 + (n / 128 + 24) * 2.0 ** -24


# ---- policy loss ----------------------------------------------------------------

def policy(logp, old, ref, advantage, weight, takes, clip_low, clip_high, dual_clip, kl_coef, kl_kind):
    """(l, k, coef, cut) per token in 64 bits, token by token."""
    n = logp.numel()
    out = torch.zeros(4, n, dtype=F64)
    value = lambda t, i: float(t[i].double())  # noqa: E731
    for i in range(n):
        if not bool(takes[i]):
            continue
        lp, a, w = value(logp, i), value(advantage, i), value(weight, i)
        r = math.exp(lp - value(old, i)) if old is not None else 1.0
        free = r * a
        held = min(max(r, 1.0 - clip_low), 1.0 + clip_high) * a
        best, slope, cut = (free, free, 0.0) if not held < free else (held, 0.0, 1.0)
        if dual_clip and a < 0 and best < dual_clip * a:
            best, slope, cut = dual_clip * a, 0.0, 1.0
        k = dk = 0.0
        if kl_coef:
            d = lp - value(ref, i)
            k, dk = {1: (d, 1.0), 2: (d * d / 2, d), 3: (math.exp(-d) + d - 1, 1 - math.exp(-d))}[kl_kind]
        out[:, i] = torch.tensor([-best, k, w * (kl_coef * dk - slope), cut], dtype=F64)
    return out


def policy_error(logp_error, old, ref, logp, advantage, weight, takes, kl_coef):
    """Bound on the error of coef per token: a log-probability off by e makes the ratio and exp(-d) off by e of
    themselves, their own arguments and functions add 2^-21 of the argument's size and of the result."""
    logp = logp.to(F64)
    r = torch.exp(logp - old.to(F64)) if old is not None else torch.ones_like(logp)
    size = logp.abs() + (old.to(F64).abs() if old is not None else 0)
    e = r * advantage.to(F64).abs() * (logp_error + 2.0 ** -22 * (size + 8))
    if kl_coef:
        d = logp - ref.to(F64)
        e = e + abs(kl_coef) * (1 + torch.exp(-d) + d.abs()) * (logp_error + 2.0 ** -22 * (logp.abs() + ref.to(F64).abs() + 8))
    return torch.where(takes, weight.to(F64).abs() * e, torch.zeros((), dtype=F64))


# ---- preference loss --------------------------------------------------------------

def preference(logp, ref, mask, offsets, pairs, beta, margin=0.0, smoothing=0.0, kind=0, mean=False, pair_weight=None):
    """(loss, margin, correct, coef, rewards) in 64 bits."""
    tokens = logp.numel()
    value = logp.to(F64) - (ref.to(F64) if ref is not None else 0)
    coef, sums, places = torch.zeros(tokens, dtype=F64), [], []
    for q in range(2 * pairs):
        at = [t for t in range(int(offsets[q]), int(offsets[q + 1])) if mask is None or int(mask[t])]
        places.append(at)
        sums.append(math.fsum(float(value[t]) for t in at) / (max(1, len(at)) if mean else 1))
    loss = total_margin = 0.0
    correct = 0
    for i in range(pairs):
        c, r = sums[2 * i], sums[2 * i + 1]
        h = beta * (c - r) - margin
        w = float(pair_weight[i]) if pair_weight is not None else 1.0 / pairs
        if kind == 0:
            up, down = 1 / (1 + math.exp(-h)), 1 / (1 + math.exp(h))
            one, slope = -(1 - smoothing) * math.log(up) - smoothing * math.log(down), smoothing * up - (1 - smoothing) * down
        elif kind == 1:
            one, slope = max(0.0, 1 - h), -1.0 if h < 1 else 0.0
        else:
            one = (h / beta - 0.5 / beta) ** 2
            slope = 2 * (h / beta - 0.5 / beta) / beta
        loss += w * one
        total_margin += w * h
        correct += c > r
        for q, sign in ((2 * i, 1), (2 * i + 1, -1)):
            for t in places[q]:
                coef[t] = sign * beta * slope * w / (max(1, len(places[q])) if mean else 1)
    return loss, total_margin, correct, coef, torch.tensor([beta * s for s in sums], dtype=F64)


# ---- 8-bit checkpoints --------------------------------------------------------------

def act8_encode(x):
    """(codes as float8_e4m3fn, scale bytes) of x [rows, cols]; inf and NaN become NaN."""
    rows, cols = x.shape
    b = torch.nn.functional.pad(x.to(F64), (0, -cols % 128)).reshape(rows, -1, 128)
    fine = torch.isfinite(b)
    top = torch.where(fine, b, torch.zeros_like(b)).abs().amax(2)
    byte = torch.zeros(top.shape, dtype=torch.int64)
    for s in range(0, 255):      # the smallest exponent that holds the block
        byte = torch.where(top > 448.0 * 2.0 ** (s - 127), torch.full_like(byte, s + 1), byte)
    q = b * torch.exp2(127.0 - byte.to(F64))[:, :, None]
    # e4m3: 4 bits from the leading one on, down to the grid of its smallest normal number, 2^-6
    grid = torch.where(fine, q, torch.zeros_like(q)).abs().clamp(min=2.0 ** -6)
    step = torch.exp2((torch.frexp(grid).exponent - 4).to(F64))
    q = torch.where(fine, torch.round(q / step) * step, torch.full_like(q, math.nan))
    codes = q.to(torch.float32).to(torch.float8_e4m3fn)
    assert bool(((codes.to(F64) == q) | ~fine).all())
    return codes.reshape(rows, -1)[:, :cols].contiguous(), byte.to(torch.uint8)


def act8_decode(codes, scales):
    """The values codes (float8_e4m3fn) and scale bytes stand for, in 64 bits."""
    rows, cols = codes.shape
    s = torch.exp2(scales.to(F64) - 127).repeat_interleave(128, 1)[:, :cols]
    return codes.to(torch.float32).to(F64) * s


def rmsnorm(x, w, eps):
    rstd = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + eps)
    return x * rstd * w.to(F64), rstd[:, 0]


def rmsnorm_grad(x, w, eps, dy, dres=None):
    rstd = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + eps)
    g = dy.to(F64) * w.to(F64)
    dx = rstd * (g - x * rstd ** 2 * (g * x).mean(1, keepdim=True))
    if dres is not None:
        dx = dx + dres.to(F64)
    return dx, (dy.to(F64) * x * rstd).sum(0)
