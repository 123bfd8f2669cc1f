"""Token log-probabilities, policy and preference loss on the GPU against 64 bits.

Tolerances, with H = 2^-24.  A row's sum has its maximum as a term, so it is at least 1; an
exponential is taken of k (x - m) with |x - m| <= 20 here: two roundings of the argument (40 H of
20 log2 e in the exponent, 60 H in all) and 2 ulp of the unit, and a thread adds up to 300 terms
and 512 of them are joined: the sum is good to 500 H at worst, and so is a softmax value to 600 H
of itself.  A log-probability adds half steps of the numbers up to 32 it is made of: 32 H each,
three of them.  Stored gradients add half a step of their type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
H = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
LOGPROB_TOL = 600 * H


def _logits(shape, dtype, seed=0, std=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype), g


def _targets(shape, vocab, g, ignore=0.25):
    t = torch.randint(vocab, shape, device=DEV, generator=g)
    return torch.where(torch.rand(shape, device=DEV, generator=g) < ignore, torch.full_like(t, -100), t)


def _wide(logits, targets, vocab, temperature=1.0):
    """(log-probabilities, softmax, counted) in 64 bits."""
    x = logits.detach()[..., :vocab].double() / temperature
    logp = torch.log_softmax(x, -1)
    counted = (targets >= 0) & (targets < vocab)
    picked = logp.gather(-1, torch.where(counted, targets, 0)[..., None])[..., 0]
    return torch.where(counted, picked, 0.0), logp.exp(), counted


def _check_grad(got, coef, p, targets, counted, vocab, temperature=1.0, coef_error=0.0):
    """`coef`: gradient of each log-probability, `coef_error` what it may be off by."""
    coef, p = torch.where(counted, coef, 0.0)[..., None], torch.where(counted[..., None], p, 0.0)
    want = -coef * p
    want.scatter_add_(-1, torch.where(counted, targets, 0)[..., None], coef)
    want = want / temperature
    half = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype is F16 else 1e-37
    size = (coef.abs() * p).scatter_add(-1, torch.where(counted, targets, 0)[..., None], coef.abs()) / temperature
    off = coef_error[..., None] if isinstance(coef_error, torch.Tensor) else coef_error
    # the hit adds its own coefficient's error on top of the softmax value's
    limit = half * want.abs() * 1.001 + 600 * H * size + off * (p + 1.0) / temperature + tiny
    wrong = (got[..., :vocab].double() - want).abs() / limit
    assert float(wrong.max()) <= 1, float(wrong.max())
    assert (got[..., vocab:] == 0).all()
    assert (got[~counted] == 0).all()


SHAPES = [((5, 7), 1000, 1000), ((3, 11), 257, 257), ((33,), 50257, 50304), ((2, 2, 3), 33, 40), ((4,), 1, 1),
          ((6,), 2, 9), ((3,), 128256, 128256), ((9,), 4097, 4097), ((700,), 64, 64)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape,vocab,ld", SHAPES)
@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_logprobs_and_their_gradient(dtype, shape, vocab, ld, temperature):
    from gpubridge_b200.ops.logprob import token_logprobs
    logits, g = _logits((*shape, ld), dtype, seed=vocab)
    targets = _targets(shape, vocab, g)
    logits.requires_grad_(True)
    before = logits.detach().clone()
    got = token_logprobs(logits, targets, vocab, temperature=temperature)
    want, p, counted = _wide(logits, targets, vocab, temperature)
    assert got.dtype == F32 and ((got - want).abs() <= LOGPROB_TOL).all()
    assert (got[~counted] == 0).all()
    d = torch.randn(shape, device=DEV, generator=g)
    grad, = torch.autograd.grad(got, logits, d)
    _check_grad(grad, d.double(), p, targets, counted, vocab, temperature)
    assert torch.equal(logits.detach(), before)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_every_start_of_a_row(dtype):
    """Views that begin at every distance from a 16-byte boundary, and strided ones."""
    from gpubridge_b200.ops.logprob import token_logprobs
    base, g = _logits((20_000,), dtype, seed=3)
    for start in range(9):
        for width in (1, 7, 8, 9, 101):
            logits = base[start:start + 5 * width].view(5, width).detach().requires_grad_(True)
            targets = _targets((5,), width, g, ignore=0.1)
            got = token_logprobs(logits, targets)
            want, p, counted = _wide(logits, targets, width)
            assert ((got - want).abs() <= LOGPROB_TOL).all()
            grad, = torch.autograd.grad(got.sum(), logits)
            _check_grad(grad, torch.ones_like(want), p, targets, counted, width)
    whole, g = _logits((3, 9, 104), dtype, seed=4)
    for view in (whole[:, :-1], whole[:, 1:, :96], whole.transpose(0, 1), whole[:, ::2], whole[1], whole[:, 4], whole[..., 3:70]):
        logits = view.detach().requires_grad_(True)
        targets = _targets(view.shape[:-1], 60, g)
        got = token_logprobs(logits, targets, 60)
        want, p, counted = _wide(logits, targets, 60)
        assert ((got - want).abs() <= LOGPROB_TOL).all()
        grad, = torch.autograd.grad(got.sum(), logits)
        _check_grad(grad, torch.ones_like(want), p, targets, counted, 60)


def test_masked_columns_infinities_and_nan():
    """-inf or the type's lowest value in masked columns; what a row that does not count holds; a
    NaN or an infinity where it does count; a row with nothing left."""
    from gpubridge_b200.ops.logprob import token_logprobs
    for dtype in (F32, BF16):
        logits, g = _logits((8, 1003), dtype, seed=5)
        logits[0, 5:900] = -math.inf
        logits[1, ::2] = torch.finfo(dtype).min
        logits[1, 3::2] = -math.inf
        logits[2] = math.nan
        logits[3, 17] = math.nan
        logits[4, 17] = math.inf
        logits[5] = -math.inf
        logits[6] = torch.finfo(dtype).min
        targets = torch.tensor([3, 1, -100, 9, 9, 9, 9, 10], device=DEV)
        leaf = logits.clone().requires_grad_(True)
        got = token_logprobs(leaf, targets)
        want, p, counted = _wide(logits, targets, 1003)
        fine = [0, 1, 2, 6, 7]
        assert ((got - want).abs()[fine] <= LOGPROB_TOL).all(), (got, want)
        assert got[[3, 4, 5]].isnan().all() and want[[3, 4, 5]].isnan().all()
        grad, = torch.autograd.grad(got[fine].sum(), leaf)
        _check_grad(grad[fine], torch.ones(5, device=DEV, dtype=torch.float64), p[fine], targets[fine],
                    counted[fine], 1003)
        assert (grad[[3, 4, 5]] == 0).all()


@pytest.mark.parametrize("level", [-1e9, 1e7, -3e8, -744261120.0, 1e10, -1e20, 1e30])
def test_rows_far_from_zero(level):
    """All columns at a mask's value or beyond, some around 2^30 / log2(e).  From 1e8 on neighbours are
    so far apart that only ties share a row's weight; below 2^30 an exponent is then off by the roundings
    of numbers of up to 96 (2^-18 twice, 2^-19) and of 2^30 times log2(e)'s 2^-48: 1.4e-5, less than
    600 H.  At 1e7, in steps of 2.4, what a probability of 2^-87 misses is 87 * 2^-24 of itself."""
    from gpubridge_b200.ops.logprob import token_logprobs
    logits, g = _logits((6, 3001), F32, seed=15)
    step = abs(level) * 2.0 ** -22
    logits = (level + torch.round(logits.double() * 2) * step).float()
    logits[1, ::2] = 0.5 * level                            # half the columns elsewhere
    logits[2, 5:] = -math.inf
    targets = torch.randint(3001, (6,), device=DEV, generator=g)
    targets[2] = 3
    leaf = logits.requires_grad_(True)
    got = token_logprobs(leaf, targets)
    want, p, counted = _wide(logits, targets, 3001)
    assert ((got - want).abs() <= LOGPROB_TOL + 64 * H * want.abs()).all(), (got, want)
    grad, = torch.autograd.grad(got.sum(), leaf)
    off = (grad.double() + p - torch.nn.functional.one_hot(targets, 3001)).abs()
    assert (off <= 600 * H * p + 4 * H + 1e-37).all()


def test_large_logits_and_a_dominant_target():
    from gpubridge_b200.ops.logprob import token_logprobs
    logits, g = _logits((6, 5000), F32, seed=6, std=5.0)
    logits += 3000.0
    targets = torch.randint(5000, (6,), device=DEV, generator=g)
    logits[torch.arange(3), targets[:3]] += 200.0
    got = token_logprobs(logits, targets)
    want, _, _ = _wide(logits, targets, 5000)
    assert ((got - want).abs() <= LOGPROB_TOL + 64 * H * want.abs()).all()
    # the sum is the target's own term: 2^r with |r| < 1, put right by 2^-r.  Each of the two powers is
    # off by 2 ulp, their product and the rescalings by half a step each: 16 H at most, and the sum is
    # not let below 1, so no log-probability is above 0
    assert (got[:3] <= 0).all() and (got[:3] >= -16 * H).all()


def _policy(dtype=BF16, shape=(6, 40), vocab=1001, ld=1008, seed=0, weights=False, ref=True):
    logits, g = _logits((*shape, ld), dtype, seed=seed)
    targets = _targets(shape, vocab, g)
    lp, _, _ = _wide(logits, targets, vocab)
    drift = torch.randn(shape, device=DEV, generator=g) * 0.2
    edge = ((drift.exp() - 1.3).abs() < 1e-3) | ((drift.exp() - 0.9).abs() < 1e-3)
    old = (lp.float() - torch.where(edge, 0.0, drift))
    adv = torch.randn(shape, device=DEV, generator=g)
    adv[0] = 0.0
    return {"logits": logits.requires_grad_(True), "targets": targets, "old": old, "adv": adv,
            "ref": lp.float() + torch.randn(shape, device=DEV, generator=g) * 0.2 if ref else None,
            "weights": torch.rand(shape, device=DEV, generator=g).masked_fill_(
                torch.rand(shape, device=DEV, generator=g) < 0.2, 0.0) if weights else None, "vocab": vocab}


def _policy_wide(c, kl_coef, low, high, denominator=None):
    lp, p, counted = _wide(c["logits"], c["targets"], c["vocab"])
    if c["weights"] is not None:
        counted = counted & (c["weights"] != 0)
    w = counted.double() if c["weights"] is None else torch.where(counted, c["weights"].double(), 0.0)
    w = w / (w.sum() if denominator is None else denominator)
    leaf = torch.where(counted, lp, 0.0).requires_grad_(True)
    ratio = (leaf - torch.where(counted, c["old"].double(), 0.0)).exp()
    a = c["adv"].double()
    each = -torch.minimum(ratio * a, ratio.clamp(1 - low, 1 + high) * a)
    kl = torch.zeros_like(each)
    if c["ref"] is not None:
        gap = torch.where(counted, c["ref"].double(), 0.0) - leaf
        kl = gap.expm1() - gap
    outside = ((a > 0) & (ratio > 1 + high)) | ((a < 0) & (ratio < 1 - low))
    loss = (w * (each + kl_coef * kl)).sum()
    coef, = torch.autograd.grad(loss, leaf)
    # what a log-probability's error does to each coefficient and term: all are exponentials of it
    slope = w * ((ratio * a).abs() + abs(kl_coef) * (kl + 1.5))
    return loss.detach(), (w * kl).sum().detach(), (w * outside).sum(), coef, p, counted, slope.detach(), leaf.detach()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("unit_grad", [False, True])
@pytest.mark.parametrize("weights,ref", [(False, True), (True, False), (True, True)])
def test_policy_loss(dtype, unit_grad, weights, ref):
    from gpubridge_b200.ops.logprob import policy_loss
    c = _policy(dtype, weights=weights, ref=ref)
    kl_coef = 0.1 if ref else 0.0
    out = policy_loss(c["logits"], c["targets"], c["old"], c["adv"], ref_logprobs=c["ref"], weights=c["weights"],
                      clip=(0.1, 0.3), kl_coef=kl_coef, vocab=c["vocab"], unit_grad=unit_grad)
    loss, kl, clipped, coef, p, counted, slope, lp = _policy_wide(c, kl_coef, 0.1, 0.3)
    off = LOGPROB_TOL * slope.sum() + 8 * H
    assert ((out.logprobs - lp).abs() <= LOGPROB_TOL).all()
    assert abs(float(out.loss.detach()) - float(loss)) <= float(off)
    assert abs(float(out.kl) - float(kl)) <= LOGPROB_TOL * 2
    assert abs(float(out.clipped) - float(clipped)) <= 4 * H
    if unit_grad:
        grad, = torch.autograd.grad(out.loss, c["logits"], retain_graph=True)
        _check_grad(grad, coef, p, c["targets"], counted, c["vocab"], coef_error=LOGPROB_TOL * slope)
        with pytest.raises(RuntimeError, match="once"):
            out.loss.backward()
    else:
        grad, = torch.autograd.grad(out.loss * 3.0, c["logits"])
        _check_grad(grad, 3 * coef, p, c["targets"], counted, c["vocab"], coef_error=3 * LOGPROB_TOL * slope)


def test_policy_loss_denominator_and_broadcast_advantages():
    from gpubridge_b200.ops.logprob import policy_loss
    c = _policy(F32)
    c["adv"] = torch.randn(6, 1, device=DEV).expand(6, 40)
    d = torch.tensor(1234.5, device=DEV)
    out = policy_loss(c["logits"], c["targets"], c["old"], c["adv"][:, :1], denominator=d, vocab=c["vocab"],
                      clip=(0.1, 0.3), unit_grad=True)
    c["ref"] = None
    loss, _, _, coef, p, counted, slope, _ = _policy_wide(c, 0.0, 0.1, 0.3, denominator=1234.5)
    assert abs(float(out.loss) - float(loss)) <= float(LOGPROB_TOL * slope.sum() + 8 * H)
    out.loss.backward()
    _check_grad(c["logits"].grad, coef, p, c["targets"], counted, c["vocab"], coef_error=LOGPROB_TOL * slope)
    out.loss.detach().mul_(2.0)


def test_policy_loss_without_a_counting_token():
    from gpubridge_b200.ops.logprob import policy_loss
    for unit_grad in (False, True):
        for kind in ("ignored", "weightless", "empty"):
            logits = torch.full((0 if kind == "empty" else 3, 4, 100), math.nan, device=DEV).requires_grad_(True)
            shape = logits.shape[:2]
            z = torch.full(shape, math.nan, device=DEV)
            targets = torch.full(shape, -100 if kind == "ignored" else 5, device=DEV)
            weights = torch.zeros(shape, device=DEV) if kind == "weightless" else None
            out = policy_loss(logits, targets, z, z, ref_logprobs=z, weights=weights, kl_coef=0.1, unit_grad=unit_grad)
            assert float(out.loss) == 0.0 and float(out.kl) == 0.0 and float(out.clipped) == 0.0
            out.loss.backward()
            assert (logits.grad == 0).all()


def test_policy_loss_keeps_a_nan():
    """exp overflows against an old log-probability far below: 0 times inf is a NaN, in loss and gradient."""
    from gpubridge_b200.ops.logprob import policy_loss
    logits = torch.randn(2, 50, device=DEV).requires_grad_(True)
    targets = torch.tensor([3, 4], device=DEV)
    old = torch.tensor([-200.0, -3.0], device=DEV)
    for unit_grad in (False, True):
        out = policy_loss(logits, targets, old, torch.tensor([0.0, 1.0], device=DEV), unit_grad=unit_grad)
        assert out.loss.isnan()
        grad, = torch.autograd.grad(out.loss, logits)
        assert grad[0].isnan().all() and torch.isfinite(grad[1]).all()


def _preference_wide(lp, counted, bounds, ref, beta, smoothing, average):
    leaf = lp.clone().requires_grad_(True)
    sums = torch.stack([leaf.reshape(-1)[a:b].sum() / (max(1, int(counted.reshape(-1)[a:b].sum())) if average else 1)
                        for a, b in bounds])
    rewards = beta * (sums - ref.double())
    n = len(bounds) // 2
    m = rewards[:n] - rewards[n:]
    ls = torch.nn.functional.logsigmoid
    loss = (-(1 - smoothing) * ls(m) - smoothing * ls(-m)).mean()
    coef, = torch.autograd.grad(loss, leaf)
    return loss.detach(), rewards.detach(), sums.detach(), coef


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_preference_loss(dtype, packed, average, smoothing):
    from gpubridge_b200.ops.logprob import preference_loss
    vocab, ld = 513, 520
    if packed:      # a row before the first, five behind the last, an empty sequence, one of a single token
        marks = [1, 30, 30, 31, 95, 200, 264]
        shape = (269,)
    else:
        shape, marks = (6, 40), [40 * i for i in range(7)]
    logits, g = _logits((*shape, ld), dtype, seed=8)
    targets = _targets(shape, vocab, g)
    logits.requires_grad_(True)
    lp, p, counted = _wide(logits, targets, vocab)
    bounds = list(zip(marks, marks[1:]))
    scale = 1.0 if average else 20.0
    ref = (torch.stack([lp.reshape(-1)[a:b].sum() / (max(1, int(counted.reshape(-1)[a:b].sum())) if average else 1)
                        for a, b in bounds]) + torch.randn(6, device=DEV, generator=g) * scale).to(F32)
    offsets = torch.tensor(marks, device=DEV) if packed else None
    out = preference_loss(logits, targets, ref, offsets=offsets, beta=0.1, label_smoothing=smoothing,
                          average=average, vocab=vocab)
    loss, rewards, sums, coef = _preference_wide(lp, counted, bounds, ref, 0.1, smoothing, average)
    longest = 1 if average else max(b - a for a, b in bounds)
    off = longest * LOGPROB_TOL                       # of a sum
    assert ((out.logprobs - sums).abs() <= off + H * sums.abs()).all()
    assert ((out.rewards - rewards).abs() <= 0.1 * off + H * rewards.abs()).all()
    assert abs(float(out.loss) - float(loss)) <= 0.2 * off + 2 * H * float(loss)
    grad, = torch.autograd.grad(out.loss * 2.0, logits, retain_graph=True)
    # sigmoid has slope at most 1/4 in the margin
    error = 2 * 0.1 / 3 * 0.25 * 0.2 * off
    _check_grad(grad, 2 * coef, p, targets, counted, vocab, coef_error=torch.where(coef != 0, error, 0.0))
    again, = torch.autograd.grad(out.loss, logits)     # the logits are still there
    assert torch.allclose(again.float() * 2, grad.float(), rtol=2 * torch.finfo(dtype).eps, atol=1e-6)


def test_preference_loss_many_and_far_margins():
    from gpubridge_b200.ops.logprob import preference_loss
    logits, g = _logits((2600, 3, 48), F32, seed=9)
    targets = _targets((2600, 3), 48, g, ignore=0.0)
    lp, p, counted = _wide(logits, targets, 48)
    ref = (torch.randn(2600, device=DEV, generator=g) * 3000).double()      # margins of some hundreds
    out = preference_loss(logits, targets, ref)
    loss, rewards, sums, _ = _preference_wide(lp, counted, [(3 * i, 3 * i + 3) for i in range(2600)], ref, 0.1, 0.0, False)
    assert abs(float(out.loss) - float(loss)) <= 3 * LOGPROB_TOL + 2 * H * float(loss)
    assert torch.isfinite(out.loss)


def test_offsets_on_the_gpu_are_held_inside_the_rows():
    from gpubridge_b200.ops.logprob import preference_loss
    logits, g = _logits((50, 64), BF16, seed=10)
    targets = _targets((50,), 64, g)
    logits.requires_grad_(True)
    out = preference_loss(logits, targets, torch.zeros(2, device=DEV),
                          offsets=torch.tensor([-7, 20, 2 ** 40], device=DEV))
    want = preference_loss(logits, targets, torch.zeros(2, device=DEV), offsets=torch.tensor([0, 20, 50]))
    assert torch.equal(out.loss, want.loss)
    out.loss.backward()
    assert torch.isfinite(logits.grad).all()


def test_same_bits_two_streams_and_a_replayed_graph():
    from gpubridge_b200.ops.logprob import policy_loss, preference_loss
    a, b = _policy(seed=11), _policy(seed=12, vocab=999)

    def step(c):
        out = policy_loss(c["logits"], c["targets"], c["old"], c["adv"], ref_logprobs=c["ref"], kl_coef=0.1,
                          vocab=c["vocab"], unit_grad=True)
        pref = preference_loss(c["logits"], c["targets"], torch.zeros(6, device=DEV), vocab=c["vocab"])
        return (out.loss.detach(), out.logprobs, pref.loss.detach(),
                *torch.autograd.grad(out.loss, c["logits"]), *torch.autograd.grad(pref.loss, c["logits"]))

    want = [[t.clone() for t in step(c)] for c in (a, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        with torch.cuda.stream(side):
            other = step(b)
        mine = step(a)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(mine, want[0]))
    assert all(torch.equal(x, y) for x, y in zip(other, want[1]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(a)
    for seed in (13, 14):
        fresh = _policy(seed=seed)
        with torch.no_grad():
            for name in ("logits", "targets", "old", "adv", "ref"):
                a[name].copy_(fresh[name])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, step(fresh)))


def test_offsets_past_32_bits():
    """A row that begins more than 2^31 values into the logits."""
    from gpubridge_b200.ops.logprob import token_logprobs
    rows, vocab = 17_000, 131_072
    logits = torch.zeros(rows, vocab, dtype=BF16, device=DEV)
    targets = torch.full((rows,), -100, device=DEV)
    for r in (0, 16_383, 16_384, 16_999):
        logits[r] = torch.randn(vocab, device=DEV).to(BF16)
        targets[r] = r
    leaf = logits.requires_grad_(True)
    got = token_logprobs(leaf, targets)
    grad, = torch.autograd.grad(got.sum(), leaf)
    for r in (0, 16_383, 16_384, 16_999):
        want, p, counted = _wide(logits[r:r + 1], targets[r:r + 1], vocab)
        assert abs(float(got[r]) - float(want)) <= LOGPROB_TOL
        _check_grad(grad[r:r + 1], torch.ones_like(want), p, targets[r:r + 1], counted, vocab)
    assert (grad[1] == 0).all() and (grad[16_998] == 0).all()


def test_refusals_on_the_gpu():
    from gpubridge_b200.ops.logprob import policy_loss, token_logprobs
    logits = torch.randn(4, 10, device=DEV)
    targets = torch.zeros(4, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError, match="float32, bfloat16"):
        token_logprobs(logits.double(), targets)
    with pytest.raises(ValueError, match="targets are on cpu"):
        token_logprobs(logits, targets.cpu())
    with pytest.raises(ValueError, match="advantages is on cpu"):
        policy_loss(logits, targets, torch.zeros(4, device=DEV), torch.zeros(4))
