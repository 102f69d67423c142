"""The operators as a training step uses them together: a layer's input kept as an 8-bit checkpoint, the norm recomputed
from it, the loss on the logits with the loss scale on its gradient, the weight gradients in the pools, then the gradient
statistics and the AdamW step of this library.  Matrix products are torch's.  The same step in 64 bits, by autograd, is the
reference."""
import pytest
import torch

import operator_oracle as Q
from helpers import read_stat

pytestmark = pytest.mark.gpu

TOKENS, WIDTH, VOCAB, EPS = 96, 256, 1000, 1e-6


@pytest.fixture(autouse=True)
def device():
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    torch.cuda.set_device(0)


class Step:
    """norm weight (FP32), head (FP16 with an FP32 master) and their optimizer state."""

    def __init__(self, pkg, seed=0, scale=1024.0):
        g = torch.Generator().manual_seed(seed)
        self.pkg = pkg
        self.x = torch.randn(TOKENS, WIDTH, generator=g).half()
        self.y = torch.randint(0, VOCAB, (TOKENS,), generator=g, dtype=torch.int32)
        self.y[::7] = -100
        self.norm0 = 1 + 0.1 * torch.randn(WIDTH, generator=g)
        self.head0 = (torch.randn(VOCAB, WIDTH, generator=g) * 0.05).half()
        self.norm, self.head = self.norm0.cuda(), self.head0.cuda()
        self.master = self.head.float()
        self.norm_grad, self.head_grad = torch.zeros(WIDTH, device="cuda"), torch.zeros(VOCAB, WIDTH, dtype=torch.float32, device="cuda")
        state = lambda t: (torch.zeros(t.numel(), device="cuda"), torch.zeros(t.numel(), device="cuda"))  # noqa: E731
        self.m1, self.v1 = state(self.norm)
        self.m2, self.v2 = state(self.head)
        self.list = pkg.TensorList([
            pkg.TensorDesc(self.norm.data_ptr(), self.norm_grad.data_ptr(), self.m1.data_ptr(), self.v1.data_ptr(), None, WIDTH, 0.0, pkg.F32, 0, 0),
            pkg.TensorDesc(self.head.data_ptr(), self.head_grad.data_ptr(), self.m2.data_ptr(), self.v2.data_ptr(), self.master.data_ptr(),
                           VOCAB * WIDTH, 0.01, pkg.F16, 0, pkg.GRAD_F32)])
        host = pkg.ScalerState(scale, 0, 0, 0, 1000, 0.9, 0.999, 0.0)
        self.scaler = torch.frombuffer(bytearray(bytes(host)), dtype=torch.uint8).cuda()
        self.stat, self.record = torch.zeros(16, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
        # checkpoint of the layer's input
        self.codes = torch.empty(TOKENS, WIDTH, dtype=torch.uint8, device="cuda")
        self.scales = torch.empty(TOKENS, pkg.act8_blocks(WIDTH), dtype=torch.uint8, device="cuda")
        self.workspace = torch.empty(pkg.act8_rmsnorm_grad_workspace(TOKENS, WIDTH), dtype=torch.uint8, device="cuda")
        xb = self.x.cuda()
        pkg.act8_store(xb.data_ptr(), pkg.F16, TOKENS, WIDTH, self.codes.data_ptr(), self.scales.data_ptr())
        torch.cuda.synchronize()

    def backward(self, loss):
        """One micro-batch: logits, loss and gradients, accumulated into the pools."""
        pkg, t = self.pkg, torch
        h = t.empty(TOKENS, WIDTH, dtype=t.float16, device="cuda")
        held = (self.codes.data_ptr(), self.scales.data_ptr(), TOKENS, WIDTH, self.norm.data_ptr(), pkg.F32, EPS)
        pkg.act8_rmsnorm(*held, h.data_ptr(), pkg.F16)
        logits = (h.float() @ self.head.float().t()).half()
        self.logits = logits.clone()
        loss(self, logits)                                # leaves the gradient in the logits' place
        self.dlogits = logits.clone()
        dh = (logits.float() @ self.head.float()).half()
        self.head_grad += logits.float().t() @ h.float()
        dx = t.empty_like(h)
        pkg.act8_rmsnorm_grad(*held, dh.data_ptr(), pkg.F16, dx.data_ptr(), self.norm_grad.data_ptr(), self.workspace.data_ptr(), self.workspace.numel(),
                              flags=pkg.ACT8_ACCUMULATE)
        return dx

    def update(self, max_norm=0.0):
        pkg = self.pkg
        self.list.gradstat(self.stat.data_ptr(), 1.0, max_norm, self.scaler.data_ptr())
        self.list.step(pkg.hparams(1e-3, 0.9, 0.999, 1e-8, 1), self.stat.data_ptr(), pkg.STEP_DEVICE_BIAS_CORRECTION)
        torch.cuda.synchronize()
        return read_stat(pkg, self.stat)

    def reference(self, loss):
        """Gradients of the two weights in 64 bits, from the checkpoint's values, the loss of (logits -> scalar)."""
        x = Q.act8_decode(*Q.act8_encode(self.x))
        norm, head = self.norm0.double().requires_grad_(), self.head0.double().requires_grad_()
        y, _ = Q.rmsnorm(x, norm, EPS)
        loss(y @ head.t()).backward()
        return norm.grad, head.grad


def sft(step, logits):
    """-mean log p through the log-probabilities and their gradient."""
    pkg = step.pkg
    yb, n = step.y.cuda(), int((step.y >= 0).sum())
    logp, lse, coef = torch.empty(TOKENS, device="cuda"), torch.empty(TOKENS, device="cuda"), torch.full((TOKENS,), -1.0 / n, device="cuda")
    block = (logits.data_ptr(), pkg.F16, TOKENS, VOCAB, yb.data_ptr())
    pkg.token_logprob(*block, logp.data_ptr(), lse.data_ptr())
    pkg.token_logprob_grad(*block, lse.data_ptr(), coef.data_ptr(), logits.data_ptr(), scaler=step.scaler.data_ptr())
    step.loss = -float(logp.sum()) / n


def on_policy(step, logits):
    """The policy loss on the policy's own samples: advantage 1 everywhere has the gradient of the SFT loss."""
    pkg = step.pkg
    yb, n = step.y.cuda(), int((step.y >= 0).sum())
    logp, a, w = torch.empty(TOKENS, device="cuda"), torch.ones(TOKENS, device="cuda"), torch.full((TOKENS,), 1.0 / n, device="cuda")
    pkg.policy_loss(logits.data_ptr(), pkg.F16, TOKENS, VOCAB, yb.data_ptr(), a.data_ptr(), w.data_ptr(), pkg.policy_hparams(), logp.data_ptr(),
                    logits.data_ptr(), step.record.data_ptr(), scaler=step.scaler.data_ptr())


def preference(step, logits):
    """Three pairs of sequences of 16 tokens."""
    pkg = step.pkg
    yb, mask = step.y.cuda(), (step.y >= 0).to(torch.uint8).cuda()
    offsets = torch.arange(0, TOKENS + 1, 16, dtype=torch.int32).cuda()
    logp, lse, coef = (torch.empty(TOKENS, device="cuda") for _ in range(3))
    block = (logits.data_ptr(), pkg.F16, TOKENS, VOCAB, yb.data_ptr())
    pkg.token_logprob(*block, logp.data_ptr(), lse.data_ptr())
    pkg.preference_loss(logp.data_ptr(), TOKENS, offsets.data_ptr(), 3, pkg.preference_hparams(0.1), step.record.data_ptr(), coef.data_ptr(), mask=mask.data_ptr())
    pkg.token_logprob_grad(*block, lse.data_ptr(), coef.data_ptr(), logits.data_ptr(), scaler=step.scaler.data_ptr())


def reference_nll(step):
    rows = torch.nonzero(step.y >= 0)[:, 0]
    return lambda z: -z.log_softmax(1)[rows, step.y[rows].long()].mean()


def reference_preference(step):
    def loss(z):
        keep = (step.y >= 0).double()
        logp = z.log_softmax(1).gather(1, step.y.clamp(min=0).long()[:, None])[:, 0] * keep
        s = logp.view(3, 2, 16).sum(2)
        return -torch.nn.functional.logsigmoid(0.1 * (s[:, 0] - s[:, 1])).mean()
    return loss


@pytest.mark.parametrize("loss,reference", [(sft, reference_nll), (on_policy, reference_nll), (preference, reference_preference)])
def test_a_step(pkg, loss, reference):
    """Each of h, the logits, their gradient and dh is rounded to FP16 (2^-11 each): the gradients of the weights, sums over
    tokens of products of two of them, are off by at most 4 * 2^-11 of the sum of the sizes of their terms, here bounded by
    the 2-norm over all entries with a factor of 4 for the logits' rounding passing through the exponential (|logit| < 8)."""
    step = Step(pkg)
    step.backward(loss)
    want_norm, want_head = step.reference(reference(step))
    scale = 1024.0
    for got, want in ((step.norm_grad, want_norm), (step.head_grad, want_head)):
        off = (got.cpu().double() / scale - want).norm() / want.norm()
        assert off <= 16 * 2.0 ** -11, float(off)
    grads = [step.norm_grad.double() / scale, step.head_grad.double() / scale]
    norm = float(torch.cat([g.flatten() for g in grads]).norm())
    stat = step.update()
    assert stat.found_inf == 0 and abs(stat.norm - norm) <= 1e-5 * norm
    # the first step of AdamW moves every weight by lr * sign(g) (and the decay)
    moved = step.norm.cpu().double() - step.norm0.double()
    sure = want_norm.abs() > want_norm.abs().mean() * 0.1
    assert (moved[sure] + 1e-3 * want_norm[sure].sign()).abs().max() < 1e-5
    if loss is sft:
        assert abs(step.loss - float(reference(step)(step.logits.double().cpu()))) < 1e-5


def test_micro_batches_accumulate(pkg):
    """Two micro-batches into the pools are twice one."""
    one, two = Step(pkg), Step(pkg)
    one.backward(sft)
    two.backward(sft)
    two.backward(sft)
    assert torch.equal(two.head_grad, 2 * one.head_grad) and torch.equal(two.norm_grad, 2 * one.norm_grad)


def test_an_overflowing_loss_scale_skips_the_step(pkg):
    """A loss scale that pushes the logits' FP16 gradient to infinity is found by the statistics: nothing moves, it halves."""
    step = Step(pkg, scale=2.0 ** 60)
    step.backward(sft)
    assert not bool(torch.isfinite(step.dlogits).all())
    before = step.head.clone(), step.norm.clone()
    stat = step.update()
    assert stat.found_inf == 1 and torch.equal(step.head, before[0]) and torch.equal(step.norm, before[1])
    assert pkg.ScalerState.from_buffer_copy(step.scaler.cpu().numpy().tobytes()).scale == 2.0 ** 59


def test_a_masked_out_batch_leaves_zero_gradients(pkg):
    step = Step(pkg)
    step.y[:] = -1
    step.backward(on_policy_of_nothing)
    assert float(step.head_grad.abs().sum()) == 0.0 and float(step.norm_grad.abs().sum()) == 0.0
    assert step.update().norm == 0.0


def on_policy_of_nothing(step, logits):
    pkg = step.pkg
    yb, a, w, logp = step.y.cuda(), torch.ones(TOKENS, device="cuda"), torch.ones(TOKENS, device="cuda"), torch.empty(TOKENS, device="cuda")
    pkg.policy_loss(logits.data_ptr(), pkg.F16, TOKENS, VOCAB, yb.data_ptr(), a.data_ptr(), w.data_ptr(), pkg.policy_hparams(), logp.data_ptr(),
                    logits.data_ptr(), step.record.data_ptr(), scaler=step.scaler.data_ptr())
