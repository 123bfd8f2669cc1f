"""Gradient norm and clipping on the CPU path, what the entry points refuse, the trainer's and the
sharded model's clipping against torch.nn.utils on one process holding the whole model."""
import copy
import math

import pytest
import torch
import torch.nn as nn

from _harness import LAYOUTS, run_ranks
from gpubridge_b200.ops.grad_clip import clip_grad_norm_, clip_grads_with_norm_, grad_norm
from gpubridge_b200.ops.optim import FlatAdamW
from gpubridge_b200.parallel.trainer import DataParallelTrainer

HALF_STEP = torch.finfo(torch.float32).eps / 2


def _parameters(seed=0, shapes=((5, 7), (), (0, 3), (11,))):
    g = torch.Generator().manual_seed(seed)
    out = []
    for shape in shapes:
        p = nn.Parameter(torch.zeros(shape))
        p.grad = torch.randn(shape, generator=g)
        out.append(p)
    return out


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("max_norm", [0.5, 1e6, 0.0])
def test_clips_as_torch_does(norm_type, max_norm):
    ours, theirs = _parameters(), _parameters()
    got = clip_grad_norm_(ours, max_norm, norm_type)
    # torch refuses the largest magnitude of an empty gradient: its side goes without that one
    want = torch.nn.utils.clip_grad_norm_([p for p in theirs if p.numel()], max_norm, norm_type)
    # torch's norm is a sum of 47 squares in fp32; each of its additions is off by half a step
    assert abs(float(got) - float(want)) <= 50 * HALF_STEP * float(want)
    for a, b in zip(ours, theirs):
        assert torch.allclose(a.grad, b.grad, rtol=60 * HALF_STEP, atol=0)


def test_empty_lists_and_missing_gradients():
    assert float(grad_norm([])) == 0.0
    assert float(clip_grad_norm_([nn.Parameter(torch.zeros(3))], 1.0)) == 0.0
    assert grad_norm(torch.tensor([3.0, 4.0])).shape == ()


def test_refusals():
    p = _parameters()
    with pytest.raises(ValueError, match="norm_type"):
        grad_norm([p[0].grad], 1.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip_grad_norm_(p, -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip_grad_norm_(p, math.nan)
    with pytest.raises(TypeError, match="tensors"):
        grad_norm([1.0])
    with pytest.raises(ValueError, match="sparse"):
        grad_norm([torch.eye(3).to_sparse()])
    with pytest.raises(ValueError, match="floating|float32"):
        grad_norm([torch.ones(3, dtype=torch.int32)])
    with pytest.raises(ValueError, match="total_norm"):
        clip_grads_with_norm_(p, 1.0, torch.tensor(1.0, dtype=torch.float64))
    shared = torch.randn(8)
    a, b = nn.Parameter(torch.zeros(6)), nn.Parameter(torch.zeros(6))
    a.grad, b.grad = shared[:6], shared[2:]
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm_([a, b], 1.0)
    q = _parameters()
    q[0].grad[0, 0] = math.inf
    before = q[3].grad.clone()
    with pytest.raises(RuntimeError, match="not clipped"):
        clip_grad_norm_(q, 1.0, error_if_nonfinite=True)
    assert torch.equal(q[3].grad, before)


def test_flat_adamw_clips_on_the_way():
    torch.manual_seed(0)
    n = 1003
    p, g = torch.randn(n), torch.zeros(n)
    stock = nn.Parameter(p.clone())
    theirs = torch.optim.AdamW([stock], lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1)
    ours = FlatAdamW(p, g, lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1)
    for step in range(4):
        grad = torch.randn(n) * (1 + step)
        g.copy_(grad * 2)
        stock.grad = grad.clone()
        want = torch.nn.utils.clip_grad_norm_([stock], 3.0)
        theirs.step()
        ours.step(grad_scale=0.5, max_norm=3.0)
        assert torch.allclose(ours.grad_norm, want, rtol=1e-5)
        assert torch.allclose(p, stock.detach(), rtol=1e-5, atol=1e-6)
        assert (g == 0).all()
    with pytest.raises(ValueError, match="max_norm"):
        ours.step(max_norm=-1.0)


def test_trainer_clips_and_reports_the_norm():
    torch.manual_seed(3)
    model = nn.Sequential(nn.Linear(24, 40), nn.GELU(), nn.Linear(40, 8))
    stock = copy.deepcopy(model)
    loss_fn = lambda m, x, y: nn.functional.mse_loss(m(x), y)  # noqa: E731
    trainer = DataParallelTrainer(model, loss_fn, autocast=None, lr=1e-2, max_grad_norm=0.05)
    optimizer = torch.optim.AdamW(stock.parameters(), lr=1e-2)
    g = torch.Generator().manual_seed(0)
    for _ in range(3):
        x, y = torch.randn(16, 24, generator=g), torch.randn(16, 8, generator=g)
        trainer.step(x, y)
        optimizer.zero_grad()
        loss_fn(stock, x, y).backward()
        want = torch.nn.utils.clip_grad_norm_(stock.parameters(), 0.05)
        optimizer.step()
        assert torch.allclose(trainer.grad_norm, want, rtol=1e-4)
    for a, b in zip(model.parameters(), stock.parameters()):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)
    with pytest.raises(ValueError, match="optimizer_in_backward"):
        DataParallelTrainer(stock, loss_fn, autocast=None, max_grad_norm=1.0, optimizer_in_backward=True)
    with pytest.raises(ValueError, match="max_grad_norm"):
        DataParallelTrainer(stock, loss_fn, autocast=None, max_grad_norm=-1.0)


def _sharded(rank, topology):
    from gpubridge_b200.parallel.sharded_model import ReplicatedSync, shard_linears
    world = topology.world_size
    torch.manual_seed(5)
    whole = nn.Sequential(nn.Linear(12, 16, bias=False), nn.GELU(), nn.Linear(16, 8, bias=False),
                          nn.LayerNorm(8))
    model = copy.deepcopy(whole)
    shard_linears(model, topology)
    sync = ReplicatedSync(model, topology)
    xs = [torch.randn(6, 12, generator=torch.Generator().manual_seed(r)) for r in range(world)]
    (model(xs[rank]) ** 3).sum().backward()
    sync.average_gradients()
    norm = sync.clip_gradients(0.25)
    (sum((whole(x) ** 3).sum() for x in xs) / world).backward()
    want = torch.nn.utils.clip_grad_norm_(whole.parameters(), 0.25)
    assert torch.allclose(norm, want, rtol=1e-4), (norm, want)
    assert float(norm) > 0.25
    rows = 16 // world
    assert torch.allclose(model[0].weight.grad, whole[0].weight.grad[rank * rows:(rank + 1) * rows],
                          rtol=1e-3, atol=1e-6)
    assert torch.allclose(model[3].weight.grad, whole[3].weight.grad, rtol=1e-3, atol=1e-6)
    return float(norm)


def test_sharded_model_clips_by_the_norm_over_all_ranks(tmp_path):
    norms = run_ranks(LAYOUTS["2+2"], _sharded, tmp_path)
    assert len(set(norms)) == 1
