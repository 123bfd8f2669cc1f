"""Token log-probabilities, policy loss and preference loss on the CPU path: against torch's own
functions in 64 bits, against differences, and what they refuse."""
import math

import pytest
import torch
import torch.nn.functional as F

from gpubridge_b200.ops.logprob import policy_loss, preference_loss, token_logprobs

F64 = torch.float64


def _batch(shape=(4, 6), vocab=11, ld=13, seed=0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(*shape, ld, generator=g, dtype=F64) * 2).requires_grad_(True)
    targets = torch.randint(vocab, shape, generator=g)
    targets[..., 0] = -100
    return logits, targets, g


def test_logprobs_equal_log_softmax():
    logits, targets, _ = _batch()
    got = token_logprobs(logits, targets, 11, temperature=0.7)
    want = F.log_softmax(logits[..., :11] / 0.7, -1).gather(-1, targets.clamp(min=0)[..., None])[..., 0]
    assert torch.allclose(got[:, 1:], want[:, 1:], atol=1e-12)
    assert (got[:, 0] == 0).all()
    grad, = torch.autograd.grad(got.sum(), logits)
    assert (grad[:, 0] == 0).all() and (grad[..., 11:] == 0).all()


def test_policy_loss_formula_and_differences():
    logits, targets, g = _batch()
    old = token_logprobs(logits, targets, 11).detach() + 0.3 * torch.randn(4, 6, generator=g, dtype=F64)
    ref = old + 0.2
    advantages = torch.randn(4, 1, generator=g, dtype=F64)
    weights = torch.rand(4, 6, generator=g, dtype=F64)
    weights[2, 3] = 0
    out = policy_loss(logits, targets, old, advantages, ref_logprobs=ref, weights=weights, kl_coef=0.1,
                      clip=(0.1, 0.3), vocab=11)
    total = count = kl = 0.0
    for b in range(4):
        for t in range(1, 6):
            w, a = float(weights[b, t]), float(advantages[b, 0])
            lp = float(F.log_softmax(logits[b, t, :11].detach(), -1)[targets[b, t]])
            ratio, gap = math.exp(lp - float(old[b, t])), float(ref[b, t]) - lp
            k = math.exp(gap) - 1 - gap
            total += w * (-min(ratio * a, min(max(ratio, 0.9), 1.3) * a) + 0.1 * k)
            kl += w * k
            count += w
    assert abs(float(out.loss.detach()) - total / count) < 1e-12 and abs(float(out.kl) - kl / count) < 1e-12
    assert 0 <= float(out.clipped) <= 1
    f = lambda x: policy_loss(x, targets, old, advantages, ref_logprobs=ref, weights=weights, kl_coef=0.1,  # noqa: E731
                              clip=(0.1, 0.3), vocab=11).loss
    assert torch.autograd.gradcheck(f, (logits,))
    halved = policy_loss(logits, targets, old, advantages, weights=weights, vocab=11,
                         denominator=2 * weights[targets >= 0].sum())
    plain = policy_loss(logits, targets, old, advantages, weights=weights, vocab=11)
    assert torch.allclose(halved.loss * 2, plain.loss)


@pytest.mark.parametrize("average", [False, True])
def test_preference_loss_formula_and_differences(average):
    logits, targets, g = _batch()
    ref = torch.randn(4, generator=g, dtype=F64) * 3 - 12
    out = preference_loss(logits, targets, ref, beta=0.3, label_smoothing=0.1, average=average, vocab=11)
    logprobs = token_logprobs(logits, targets, 11).detach()
    sums = logprobs.sum(1) / (5 if average else 1)
    margin = 0.3 * ((sums - ref)[:2] - (sums - ref)[2:])
    want = (-0.9 * F.logsigmoid(margin) - 0.1 * F.logsigmoid(-margin)).mean()
    assert torch.allclose(out.loss, want, atol=1e-12)
    assert torch.allclose(out.rewards.double(), 0.3 * (sums - ref), atol=1e-5)
    f = lambda x: preference_loss(x, targets, ref, beta=0.3, label_smoothing=0.1, average=average, vocab=11).loss  # noqa: E731
    assert torch.autograd.gradcheck(f, (logits,))
    # the same sequences packed one behind the other, with a row before and two behind
    packed = torch.cat([logits[:1, 0], logits.reshape(24, 13), logits[0, :2]]).detach()
    marks = torch.tensor([1, 7, 13, 19, 25])
    flat = torch.cat([targets[:1, 1], targets.reshape(-1), targets[0, 1:3]])
    again = preference_loss(packed, flat, ref, offsets=marks, beta=0.3, label_smoothing=0.1, average=average, vocab=11)
    assert torch.allclose(again.loss, out.loss, atol=1e-12)


def test_what_does_not_count_takes_no_part():
    logits, targets, _ = _batch()
    zeros = torch.zeros(4, 6, dtype=F64)
    ones = torch.ones(4, 6, dtype=F64)
    clean = policy_loss(logits, targets, zeros, ones, ref_logprobs=zeros, kl_coef=0.1, vocab=11)
    dirty = logits.detach().clone()
    dirty[:, 0] = math.nan
    dirty.requires_grad_(True)
    old = zeros.clone()
    old[:, 0] = math.nan
    got = policy_loss(dirty, targets, old, ones, ref_logprobs=old, kl_coef=0.1, vocab=11)
    assert torch.equal(got.loss, clean.loss)
    grad, = torch.autograd.grad(got.loss, dirty)
    assert torch.isfinite(grad).all() and (grad[:, 0] == 0).all()
    nothing = policy_loss(logits, torch.full((4, 6), -100), zeros, ones)
    assert float(nothing.loss) == 0.0
    assert (torch.autograd.grad(nothing.loss, logits)[0] == 0).all()


def test_refusals():
    logits, targets, _ = _batch()
    z = torch.zeros(4, 6)
    with pytest.raises(ValueError, match="targets have shape"):
        token_logprobs(logits, targets[:, 1:])
    with pytest.raises(ValueError, match="int64"):
        token_logprobs(logits, targets.float())
    with pytest.raises(ValueError, match="vocab must"):
        token_logprobs(logits, targets, 14)
    for t in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="temperature"):
            token_logprobs(logits, targets, temperature=t)
    with pytest.raises(ValueError, match="broadcast"):
        policy_loss(logits, targets, z, torch.zeros(4))
    with pytest.raises(ValueError, match="no gradient"):
        policy_loss(logits, targets, z.clone().requires_grad_(True), z)
    with pytest.raises(ValueError, match="kl_coef needs"):
        policy_loss(logits, targets, z, z, kl_coef=0.1)
    with pytest.raises(ValueError, match="clip"):
        policy_loss(logits, targets, z, z, clip=(1.5, 0.2))
    with pytest.raises(ValueError, match="denominator"):
        policy_loss(logits, targets, z, z, denominator=torch.zeros(2))
    with pytest.raises(TypeError, match="tensor"):
        policy_loss(logits, targets, z, 1.0)
    ref = torch.zeros(4)
    with pytest.raises(ValueError, match="pairs"):
        preference_loss(logits[:3], targets[:3], ref[:3])
    with pytest.raises(ValueError, match="ref_logprobs"):
        preference_loss(logits, targets, ref.half())
    with pytest.raises(ValueError, match="label_smoothing"):
        preference_loss(logits, targets, ref, label_smoothing=1.5)
    with pytest.raises(ValueError, match="without offsets"):
        preference_loss(logits.reshape(24, 13), targets.reshape(-1), ref)
    flat = (logits.reshape(24, 13), targets.reshape(-1), ref)
    for bad in ([0, 6, 12, 18, 25], [0, 12, 6, 18, 24], [-1, 6, 12, 18, 24]):
        with pytest.raises(ValueError, match="offsets must"):
            preference_loss(*flat, offsets=torch.tensor(bad))
    with pytest.raises(ValueError, match="offsets is"):
        preference_loss(*flat, offsets=torch.tensor([0, 12, 24]))
