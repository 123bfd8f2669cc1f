"""The models' joined blocks and fine-tuning losses on the CPU: against the separate operations, and
a few training steps with every operator together."""
import copy

import pytest
import torch
import torch.nn.functional as F

from gpubridge_b200.models import gpt2, llama
from gpubridge_b200.models.llama import apply_rope, rope_tables
from gpubridge_b200.parallel.trainer import DataParallelTrainer


def _tokens(vocab, batch=4, seq=12, prompt=4, seed=0):
    g = torch.Generator().manual_seed(seed)
    tokens = torch.randint(vocab, (batch, seq + 1), generator=g)
    targets = tokens[:, 1:].clone()
    targets[:, :prompt] = -100
    return tokens[:, :-1].contiguous(), targets


def _sandwich_by_hand(model, idx):
    c = model.config
    cos, sin = rope_tables(c.width // c.heads, idx.shape[1], c.rope_base, idx.device)
    x = model.embed(idx)
    rms = lambda x, w: F.rms_norm(x, (c.width,), w, c.eps)  # noqa: E731
    for b in model.blocks:
        h = rms(x, b.attn_norm.weight)
        q, k, v = (lin(h).view(*idx.shape, -1, b.head_dim).transpose(1, 2) for lin in (b.wq, b.wk, b.wv))
        y = F.scaled_dot_product_attention(apply_rope(q, cos, sin), apply_rope(k, cos, sin), v, is_causal=True,
                                           enable_gqa=True)
        y = b.wo(y.transpose(1, 2).reshape(*idx.shape, -1))
        x = x + c.residual_scale * b.attn_gate * rms(y, b.attn_post)
        h = rms(x, b.ffn_norm.weight)
        y = b.down(F.silu(b.gate(h)) * b.up(h))
        x = x + c.residual_scale * b.ffn_gate * rms(y, b.ffn_post)
    return model.head(rms(x, model.norm.weight))


def test_sandwich_blocks_equal_the_separate_operations():
    model = llama.build("llama-tiny-sandwich")
    with torch.no_grad():
        for p in model.parameters():
            if p.dim() == 1:
                p.add_(0.2 * torch.randn(p.shape, generator=torch.Generator().manual_seed(p.numel())))
    idx, _ = _tokens(256)
    # the same fp32 sums in another order, through two blocks
    assert torch.allclose(model(idx), _sandwich_by_hand(model, idx), rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("module,name", [(gpt2, "gpt2-tiny"), (llama, "llama-tiny")])
def test_plain_models_join_fused_only_when_asked(monkeypatch, module, name):
    torch.manual_seed(0)
    model = module.build(name)
    idx, _ = _tokens(model.config.vocab)
    plain = model(idx)
    monkeypatch.setenv("GPUBRIDGE_FUSED_JOIN", "1")
    calls = []
    real = module.residual_norm
    monkeypatch.setattr(module, "residual_norm", lambda *a, **k: calls.append(1) or real(*a, **k))
    fused = model(idx)
    assert calls
    assert torch.allclose(plain, fused, rtol=1e-4, atol=1e-5)
    monkeypatch.delenv("GPUBRIDGE_FUSED_JOIN")
    calls.clear()
    assert torch.equal(model(idx), plain) and not calls


@pytest.mark.parametrize("module,name", [(gpt2, "gpt2-tiny"), (llama, "llama-tiny-sandwich")])
def test_losses_of_the_models(module, name):
    torch.manual_seed(1)
    model = module.build(name)
    vocab = model.config.vocab
    idx, targets = _tokens(vocab)
    logp = F.log_softmax(model(idx).float(), -1)
    counted = targets >= 0
    want = torch.where(counted, logp.gather(-1, targets.clamp(min=0)[..., None])[..., 0], torch.zeros(()))
    got = model.logprobs(idx, targets)
    assert torch.allclose(got, want, atol=1e-5)
    old, advantages = got.detach() - 0.1, torch.randn(4, 1)
    out = model.policy_loss(idx, targets, old, advantages, got.detach(), kl_coef=0.1)
    ratio = torch.exp(want - old)
    each = -torch.minimum(ratio * advantages, ratio.clamp(0.8, 1.2) * advantages)
    assert torch.allclose(out.loss, each[counted].mean(), atol=1e-5)
    ref = want.sum(1).detach() + torch.randn(4)
    out = model.preference_loss(idx, targets, ref, beta=0.5)
    margin = 0.5 * ((want.sum(1) - ref)[:2] - (want.sum(1) - ref)[2:])
    assert torch.allclose(out.loss, -F.logsigmoid(margin).mean(), atol=1e-5)


def test_a_policy_step_with_everything_equals_the_stock_operations():
    torch.manual_seed(2)
    model = llama.build("llama-tiny-sandwich")
    stock = copy.deepcopy(model)
    trainer = DataParallelTrainer(model, lambda m, *b: m.policy_loss(*b, kl_coef=0.05).loss, autocast=None, lr=1e-3,
                                  max_grad_norm=0.05)
    optimizer = torch.optim.AdamW(stock.parameters(), lr=1e-3)
    idx, targets = _tokens(256, seed=3)
    counted = targets >= 0
    with torch.no_grad():
        old = model.logprobs(idx, targets) + 0.1 * torch.randn(idx.shape)
    advantages = torch.randn(4, 1).expand(idx.shape).contiguous()
    for _ in range(3):
        loss = trainer.step(idx, targets, old, advantages, old)
        optimizer.zero_grad()
        lp = F.log_softmax(_sandwich_by_hand(stock, idx), -1).gather(-1, targets.clamp(min=0)[..., None])[..., 0]
        ratio, gap = torch.exp(lp - old), old - lp
        each = -torch.minimum(ratio * advantages, ratio.clamp(0.8, 1.2) * advantages) + 0.05 * (gap.exp() - 1 - gap)
        want = each[counted].mean()
        want.backward()
        norm = torch.nn.utils.clip_grad_norm_(stock.parameters(), 0.05)
        optimizer.step()
        assert torch.allclose(loss, want, rtol=1e-3, atol=1e-5)
        assert torch.allclose(trainer.grad_norm, norm, rtol=1e-3)
        assert float(norm) > 0.05
    a = torch.cat([p.detach().reshape(-1) for p in model.parameters()])
    b = torch.cat([p.detach().reshape(-1) for p in stock.parameters()])
    assert float((a - b).norm() / b.norm()) < 2e-3
