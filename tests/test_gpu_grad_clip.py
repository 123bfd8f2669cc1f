"""Gradient norm, clipping and the clipped AdamW step on the GPU, against 64 bits.

Tolerances: the norm's squares and sums are in 64 bits, so what is left is its one rounding to
fp32 and the host's own last bits: two half steps.  A clipped gradient is rounded once in its
type, and its factor once in fp32 from a norm of 64 bits."""
import math

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F32_HALF = torch.finfo(torch.float32).eps / 2


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _wide_norm(tensors, norm_type=2.0):
    flat = torch.cat([t.detach().double().reshape(-1) for t in tensors])
    return float(flat.norm() if norm_type == 2.0 else flat.abs().max())


def _tensors(dtype, sizes, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(n, device=DEV, generator=g) * scale).to(dtype) for n in sizes]


SIZES = [1, 7, 0, 8, 9, 31, 32, 33, 255, 32767, 32768, 32769, 100_003, 262_144]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_norm_of_many_sizes(dtype, norm_type):
    from gpubridge_b200.ops.grad_clip import grad_norm
    tensors = _tensors(dtype, SIZES)
    want = _wide_norm(tensors, norm_type)
    assert abs(float(grad_norm(tensors, norm_type)) - want) <= 2 * F32_HALF * want
    # every start that a view can have inside a vector
    base = _tensors(dtype, [70_000], seed=1)[0]
    for start in range(17):
        for length in (0, 1, 15, 16, 17, 40_001):
            part = base[start:start + length]
            want = _wide_norm([part], norm_type) if length else 0.0
            assert abs(float(grad_norm(part, norm_type)) - want) <= 2 * F32_HALF * want, (start, length)


def test_norm_of_more_tensors_than_a_launch_carries_and_of_mixed_types():
    from gpubridge_b200.ops.grad_clip import grad_norm
    tensors = _tensors(torch.float32, [1 + i % 37 for i in range(2500)])
    tensors += _tensors(torch.bfloat16, [40, 3], seed=2) + _tensors(torch.float16, [77], seed=3)
    want = _wide_norm(tensors)
    assert abs(float(grad_norm(tensors)) - want) <= 2 * F32_HALF * want
    assert float(grad_norm([])) == 0.0
    assert float(grad_norm([torch.empty(0, device=DEV)])) == 0.0


@pytest.mark.parametrize("scale", [1e30, 1e-30])
def test_norm_neither_overflows_nor_vanishes(scale):
    from gpubridge_b200.ops.grad_clip import grad_norm
    tensors = _tensors(torch.float32, [5000, 17], scale=scale)
    want = _wide_norm(tensors)
    assert abs(float(grad_norm(tensors)) - want) <= 2 * F32_HALF * want


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_non_finite_values_reach_the_norm(value, norm_type):
    from gpubridge_b200.ops.grad_clip import clip_grad_norm_, grad_norm
    for at in (0, 33, 99_999):
        t = _tensors(torch.float32, [100_000])[0]
        t[at] = value
        got = float(grad_norm(t, norm_type))
        assert math.isnan(got) if math.isnan(value) else got == math.inf
    p = nn.Parameter(torch.zeros(100_000, device=DEV))
    p.grad = t
    before = t.clone()
    with pytest.raises(RuntimeError, match="not clipped"):
        clip_grad_norm_([p], 1.0, norm_type, error_if_nonfinite=True)
    assert torch.equal(p.grad.nan_to_num(), before.nan_to_num())


def _with_grads(tensors):
    out = []
    for t in tensors:
        p = nn.Parameter(torch.zeros(t.shape, dtype=t.dtype, device=DEV))
        p.grad = t
        out.append(p)
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_clip_in_place(dtype, norm_type):
    from gpubridge_b200.ops.grad_clip import clip_grad_norm_
    tensors = _tensors(dtype, SIZES, seed=4)
    base = _tensors(dtype, [9000], seed=5)[0]
    tensors += [base[3:3 + 4001], _tensors(dtype, [600], seed=6)[0].view(20, 30).t()]
    guard = base[4004:].clone()
    gaps = _tensors(dtype, [640], seed=7)[0].view(20, 32)
    tensors.append(gaps[:, 3:20])                       # values with gaps between them
    outside = torch.cat([gaps[:, :3], gaps[:, 20:]], 1).clone()
    before = [t.double().clone() for t in tensors]
    want = _wide_norm(tensors, norm_type)
    max_norm = want / 3
    got = clip_grad_norm_(_with_grads(tensors), max_norm, norm_type)
    assert abs(float(got) - want) <= 2 * F32_HALF * want
    coef = max_norm / (want + 1e-6)
    for t, b in zip(tensors, before):
        # fp16 has steps of 2^-24 near zero: half of one there
        tiny = 2.0 ** -25 if dtype is torch.float16 else 0.0
        assert ((t.double() - b * coef).abs()
                <= (b * coef).abs() * (_half_step(dtype) + 4 * F32_HALF) + tiny).all()
    assert torch.equal(base[4004:], guard)
    assert torch.equal(torch.cat([gaps[:, :3], gaps[:, 20:]], 1), outside)


def test_within_the_limit_nothing_changes():
    from gpubridge_b200.ops.grad_clip import clip_grad_norm_
    tensors = _tensors(torch.bfloat16, SIZES, seed=8)
    before = [t.clone() for t in tensors]
    clip_grad_norm_(_with_grads(tensors), 1e9)
    assert all(torch.equal(a, b) for a, b in zip(tensors, before))


def test_norm_found_elsewhere():
    from gpubridge_b200.ops.grad_clip import clip_grads_with_norm_
    t = _tensors(torch.float32, [4097])[0]
    before = t.clone()
    clip_grads_with_norm_(_with_grads([t]), 1.0, torch.tensor(8.0, device=DEV))
    assert torch.allclose(t, before * (1.0 / (8.0 + 1e-6)), rtol=4 * F32_HALF, atol=0)
    with pytest.raises(ValueError, match="total_norm is on"):
        clip_grads_with_norm_(_with_grads([t]), 1.0, torch.tensor(8.0))


def test_refusals():
    from gpubridge_b200.ops.grad_clip import clip_grad_norm_, grad_norm
    t = _tensors(torch.float32, [64])[0]
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        grad_norm([t.double()])
    with pytest.raises(ValueError, match="one device"):
        grad_norm([t, t.cpu()])
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm_(_with_grads([t[:40], t[20:]]), 1.0)
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm_(_with_grads([t, t]), 1.0)
    square = _tensors(torch.float32, [64])[0].view(8, 8)
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm_(_with_grads([square[:, 2:], square[:, 2:]]), 1.0)


def test_two_streams_and_a_replayed_graph():
    from gpubridge_b200.ops.grad_clip import clip_grad_norm_, grad_norm
    a, b = _tensors(torch.float32, [500_000, 300_001], seed=9)
    wants = [_wide_norm([a]), _wide_norm([b])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            nb = grad_norm(b)
        na = grad_norm(a)
    torch.cuda.synchronize()
    for got, want in zip((na, nb), wants):
        assert abs(float(got) - want) <= 2 * F32_HALF * want
    params = _with_grads([a, b])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(params, 2.0)
    for seed in (11, 12):
        fresh = _tensors(torch.float32, [500_000, 300_001], seed=seed)
        for t, f in zip((a, b), fresh):
            t.copy_(f)
        want = _wide_norm(fresh)
        graph.replay()
        torch.cuda.synchronize()
        assert abs(float(norm) - want) <= 2 * F32_HALF * want
        assert torch.allclose(a, fresh[0] * (2.0 / (want + 1e-6)), rtol=5 * F32_HALF, atol=0)


@pytest.mark.parametrize("n", [1, 3, 8, 1003, 262_147])
@pytest.mark.parametrize("clip", [0.2, 1e6])
def test_clipped_adamw_against_64_bits(n, clip):
    """Three steps; every step starts from the kernel's own fp32 state, so one step's error is
    measured.  m and v are two products and a sum (three half steps of the larger terms); p adds
    an update of at most a few lr, whose own error is some ten half steps."""
    from gpubridge_b200.ops.optim import FlatAdamW
    g = torch.Generator(device=DEV).manual_seed(n)
    p = torch.randn(n, device=DEV, generator=g)
    grad = torch.zeros(n, device=DEV)
    lr, (b1, b2), eps, wd = 1e-2, (0.9, 0.999), 1e-8, 0.1
    opt = FlatAdamW(p, grad, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd)
    for step in range(1, 4):
        fresh = torch.randn(n, device=DEV, generator=g) * 3
        grad.copy_(fresh)
        p0, m0, v0 = opt.p.double(), opt.m.double(), opt.v.double()
        scale = 0.5
        norm = float((fresh.double() * scale).norm())
        max_norm = clip * norm
        opt.step(grad_scale=scale, zero_grad=step != 2, max_norm=max_norm)
        assert abs(float(opt.grad_norm) - norm) <= 2 * F32_HALF * norm
        ge = fresh.double() * scale * min(1.0, max_norm / (norm + 1e-6))
        m = b1 * m0 + (1 - b1) * ge
        v = b2 * v0 + (1 - b2) * ge * ge
        update = lr / (1 - b1 ** step) * m / ((v / (1 - b2 ** step)).sqrt() + eps)
        want = p0 * (1 - lr * wd) - update
        # the factors b, 1 - b, the clip and the products: each half a step of its term
        assert ((opt.m - m).abs() <= 8 * F32_HALF * (b1 * m0.abs() + (1 - b1) * ge.abs())).all()
        assert ((opt.v - v).abs() <= 12 * F32_HALF * v).all()
        dm = 8 * F32_HALF * (b1 * m0.abs() + (1 - b1) * ge.abs())
        du = lr / (1 - b1 ** step) * dm / ((v / (1 - b2 ** step)).sqrt() + eps) + 14 * F32_HALF * update.abs()
        assert ((opt.p - want).abs() <= 4 * F32_HALF * p0.abs() + du).all()
        assert bool((grad == 0).all()) == (step != 2)
    assert float(opt.state[2]) == 3.0


@pytest.mark.parametrize("graph", [False, True])
def test_trainer_with_clipping_equals_the_stock_loop(graph):
    import copy
    from gpubridge_b200.models import gpt2
    from gpubridge_b200.parallel.trainer import DataParallelTrainer
    torch.manual_seed(0)
    model = gpt2.build("gpt2-tiny").to(DEV)
    stock = copy.deepcopy(model)
    trainer = DataParallelTrainer(model, lambda m, x, y: m.loss(x, y), lr=1e-3, autocast=None,
                                  graph=graph, graph_warmup=2, max_grad_norm=0.1)
    optimizer = torch.optim.AdamW(stock.parameters(), lr=1e-3)
    x, y = (t.to(DEV) for t in gpt2.synthetic_tokens(model.config, 4, 32)[0])
    for _ in range(6):
        trainer.step(x, y)
        optimizer.zero_grad()
        torch.nn.functional.cross_entropy(stock(x).reshape(-1, model.config.vocab), y.reshape(-1)).backward()
        want = torch.nn.utils.clip_grad_norm_(stock.parameters(), 0.1)
        optimizer.step()
        assert float(want) > 0.1
        assert abs(float(trainer.grad_norm) - float(want)) <= 1e-3 * float(want)
    a = torch.cat([p.detach().reshape(-1) for p in model.parameters()])
    b = torch.cat([p.detach().reshape(-1) for p in stock.parameters()])
    assert float((a - b).norm() / b.norm()) < 2e-3        # the bound of the unclipped comparison
