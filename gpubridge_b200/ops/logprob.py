"""Log-probabilities of tokens and the fine-tuning losses made of them (``csrc/gb_logprob.cu``):

    logprobs = token_logprobs(logits, targets)                    # one read of the logits
    out = policy_loss(logits, targets, old, advantages, ref_logprobs=ref, kl_coef=0.02)
    out = preference_loss(logits, targets, ref_sums, beta=0.1)    # first half chosen, second rejected
    out.loss.backward()

Next to ``ops/xent.py``: the same padded vocabularies (``vocab`` of the last dimension's columns
count), targets outside ``[0, vocab)`` (-100) mark tokens that do not count, and the gradient of
the logits is written by one kernel in their type.  Unlike there the logits are left as they are:
the gradient is a tensor of its own.  ``models/gpt2.py`` and ``models/llama.py`` offer each as a
method (``logprobs``, ``policy_loss``, ``preference_loss``) that a trainer's ``loss_fn`` may call.

Log-probabilities, losses and coefficients are in float32, sums over tokens in 64 bits and in a
fixed order.  On the CPU the same formulas run as plain torch operations.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

from gpubridge_b200.ops import _build_ops

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


class PolicyLoss(NamedTuple):
    loss: torch.Tensor          # 0-dim, differentiable
    logprobs: torch.Tensor      # of every token, 0 where it does not count
    kl: torch.Tensor            # 0-dim: weighted mean of exp(gap) - 1 - gap, gap = ref - logprob
    clipped: torch.Tensor       # 0-dim: weighted share of tokens whose ratio is past its clip


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor          # 0-dim, differentiable
    rewards: torch.Tensor       # [sequences]: beta * (logprob - reference)
    logprobs: torch.Tensor      # [sequences]: sum (or mean) over a sequence's tokens


# -- checks and the plain form ---------------------------------------------------------------------

def _check(logits, targets, vocab, temperature) -> tuple[torch.Tensor, int]:
    if logits.dim() < 1 or logits.shape[-1] == 0:
        raise ValueError(f"logits are [..., vocabulary], got shape {tuple(logits.shape)}")
    if targets.shape != logits.shape[:-1]:
        raise ValueError(f"targets have shape {tuple(targets.shape)}, logits {tuple(logits.shape)}")
    if targets.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"targets are int64 or int32, got {targets.dtype}")
    if targets.device != logits.device:
        raise ValueError(f"targets are on {targets.device}, logits on {logits.device}")
    vocab = logits.shape[-1] if vocab is None else int(vocab)
    if not 0 < vocab <= logits.shape[-1]:
        raise ValueError(f"vocab must be in [1, {logits.shape[-1]}], got {vocab}")
    if not (math.isfinite(temperature) and temperature > 0):
        raise ValueError(f"temperature must be positive, got {temperature}")
    if logits.is_cuda and logits.dtype not in _FLOATS or not logits.is_floating_point():
        raise ValueError(f"logits are float32, bfloat16 or float16 on the GPU, got {logits.dtype}")
    if logits.is_cuda and (logits.layout is not torch.strided or hasattr(logits, "to_local")):
        raise ValueError("logits are an ordinary strided tensor: not sparse and no DTensor")
    return targets.to(torch.int64).contiguous(), vocab


def _per_token(name, t, targets, like):
    """A constant of each token: float32 in the targets' shape."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} is a tensor, got {type(t).__name__}")
    if t.device != targets.device:
        raise ValueError(f"{name} is on {t.device}, targets on {targets.device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} takes no gradient: detach it")
    if t.shape != targets.shape:
        try:
            t = t.expand(targets.shape)
        except RuntimeError:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, which does not broadcast to the targets' "
                             f"{tuple(targets.shape)}") from None
    wide = torch.float64 if like.dtype == torch.float64 else torch.float32
    return t.to(wide).contiguous()


def _plain_logprobs(logits, targets, vocab, temperature, weights=None):
    wide = torch.float64 if logits.dtype == torch.float64 else torch.float32
    counted = (targets >= 0) & (targets < vocab)
    if weights is not None:
        counted = counted & (weights != 0)
    x = torch.where(counted[..., None], logits[..., :vocab].to(wide), torch.zeros((), dtype=wide)) / temperature
    at = torch.where(counted, targets, torch.zeros_like(targets))[..., None]
    picked = x.gather(-1, at)[..., 0] - torch.logsumexp(x, -1)
    return torch.where(counted, picked, torch.zeros_like(picked)), counted


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, vocab: int | None = None, *,
                   temperature: float = 1.0) -> torch.Tensor:
    """``log softmax(logits[..., :vocab] / temperature)`` at ``targets``: float32 in the targets'
    shape, 0 where a target lies outside ``[0, vocab)``.  Differentiable in the logits."""
    targets, vocab = _check(logits, targets, vocab, temperature)
    if logits.is_cuda:
        return _build_ops.load().token_logprobs(logits, targets, vocab, temperature)
    return _plain_logprobs(logits, targets, vocab, temperature)[0]


def policy_loss(logits: torch.Tensor, targets: torch.Tensor, old_logprobs: torch.Tensor,
                advantages: torch.Tensor, *, ref_logprobs: torch.Tensor | None = None,
                weights: torch.Tensor | None = None, denominator: torch.Tensor | None = None,
                clip: tuple[float, float] = (0.2, 0.2), kl_coef: float = 0.0, temperature: float = 1.0,
                vocab: int | None = None, unit_grad: bool = False) -> PolicyLoss:
    """The clipped policy loss over the tokens that count:

        sum over tokens of w (-min(ratio A, clip(ratio, 1 - clip[0], 1 + clip[1]) A) + kl_coef KL) / D

    Args:
        old_logprobs, advantages, ref_logprobs, weights: constants that broadcast to the targets
            (an advantage for each sequence as ``[batch, 1]``).  ``ratio = exp(logprob - old)``,
            ``KL = exp(gap) - 1 - gap`` with ``gap = ref - logprob`` (0 without a reference).
        weights: of each token, 1 where absent; a token of weight 0 does not count and its logits
            are not looked at.
        denominator: ``D``, a tensor of one value; by default the sum of the counting tokens'
            weights.  Where it is 0, loss and gradient are 0.
        unit_grad: promises one backward pass that starts at this loss (``loss.backward()``): the
            gradient is then written in the forward launch, while a row is still in the cache.
    """
    targets, vocab = _check(logits, targets, vocab, temperature)
    low, high = (float(c) for c in clip)
    if not (0 <= low <= 1 and 0 <= high < math.inf):
        raise ValueError(f"clip is (how far below 1, how far above 1), the first at most 1; got {clip}")
    if not math.isfinite(kl_coef):
        raise ValueError(f"kl_coef must be finite, got {kl_coef}")
    if kl_coef and ref_logprobs is None:
        raise ValueError("kl_coef needs ref_logprobs")
    old, advantages, ref, weights = (
        _per_token(name, t, targets, logits) for name, t in (
            ("old_logprobs", old_logprobs), ("advantages", advantages), ("ref_logprobs", ref_logprobs),
            ("weights", weights)))
    if old is None or advantages is None:
        raise TypeError("old_logprobs and advantages are tensors")
    if denominator is not None:
        if not isinstance(denominator, torch.Tensor) or denominator.numel() != 1 or denominator.device != logits.device:
            raise ValueError("denominator is a tensor of one value on the logits' device")
        denominator = denominator.detach().to(torch.float32).reshape(())
    if logits.is_cuda:
        return PolicyLoss(*_build_ops.load().policy_loss(logits, targets, vocab, old, advantages, ref, weights,
                                                         denominator, low, high, kl_coef, temperature, unit_grad))
    logprobs, counted = _plain_logprobs(logits, targets, vocab, temperature, weights)
    w = counted.to(logprobs.dtype) if weights is None else torch.where(counted, weights, torch.zeros_like(weights))
    total = w.double().sum() if denominator is None else denominator.double()
    w = w * torch.where(total == 0, torch.zeros_like(total), 1.0 / total).to(w.dtype)
    # what does not count takes no part, whatever it holds
    old, advantages = (torch.where(counted, t, torch.zeros_like(t)) for t in (old, advantages))
    ratio = torch.exp(logprobs - old)
    each = -torch.minimum(ratio * advantages, ratio.clamp(1 - low, 1 + high) * advantages)
    kl = torch.zeros_like(each)
    if ref is not None:
        gap = torch.where(counted, ref, torch.zeros_like(ref)) - logprobs
        kl = torch.expm1(gap) - gap
    outside = ((advantages > 0) & (ratio > 1 + high)) | ((advantages < 0) & (ratio < 1 - low))
    return PolicyLoss((w * (each + kl_coef * kl)).sum(), logprobs.detach(), (w * kl).sum().detach(),
                      (w * outside).sum().detach())


def preference_loss(logits: torch.Tensor, targets: torch.Tensor, ref_logprobs: torch.Tensor, *,
                    offsets: torch.Tensor | None = None, beta: float = 0.1, label_smoothing: float = 0.0,
                    average: bool = False, vocab: int | None = None) -> PreferenceLoss:
    """The preference loss over pairs of sequences, the first half of them chosen over the second:

        mean over pairs of -(1 - e) log sigmoid(m) - e log sigmoid(-m),   m = reward chosen - rejected

    with ``reward = beta (S - ref)`` and ``S`` the sum (``average``: the mean) of the log-probabilities
    of a sequence's counting tokens.

    Args:
        logits, targets: ``[sequences, length, ...]``, or with ``offsets`` packed rows ``[tokens, ...]``.
        ref_logprobs: ``[sequences]``, float32 or float64: ``S`` under the reference model.
        offsets: ``[sequences + 1]`` int64, the first row of each sequence and the end of the last;
            rows outside take no part.  On the CPU it is checked; on the GPU it is taken as it is,
            with every value held inside the rows.
    """
    targets, vocab = _check(logits, targets, vocab, 1.0)
    beta, smoothing = float(beta), float(label_smoothing)
    if not math.isfinite(beta):
        raise ValueError(f"beta must be finite, got {beta}")
    if not 0.0 <= smoothing <= 1.0:
        raise ValueError(f"label_smoothing is in [0, 1], got {smoothing}")
    if ref_logprobs.dim() != 1 or ref_logprobs.dtype not in (torch.float32, torch.float64):
        raise ValueError("ref_logprobs is [sequences] in float32 or float64")
    if ref_logprobs.device != logits.device:
        raise ValueError(f"ref_logprobs is on {ref_logprobs.device}, logits on {logits.device}")
    if ref_logprobs.requires_grad and torch.is_grad_enabled():
        raise ValueError("ref_logprobs takes no gradient: detach it")
    sequences = ref_logprobs.numel()
    if sequences < 2 or sequences % 2:
        raise ValueError(f"sequences come in pairs, got {sequences}")
    if offsets is None:
        if targets.dim() != 2 or targets.shape[0] != sequences:
            raise ValueError(f"targets are [{sequences}, length] without offsets, got {list(targets.shape)}")
    else:
        if targets.dim() != 1:
            raise ValueError("packed targets have one dimension")
        if offsets.shape != (sequences + 1,) or offsets.dtype != torch.int64:
            raise ValueError(f"offsets is [{sequences + 1}] int64, got {list(offsets.shape)} {offsets.dtype}")
        if offsets.device.type == "cpu":
            marks = offsets.tolist()
            if marks[0] < 0 or marks[-1] > targets.numel() or any(a > b for a, b in zip(marks, marks[1:])):
                raise ValueError(f"offsets must not fall and stay within the {targets.numel()} rows")
        offsets = offsets.to(logits.device).contiguous()
    ref_logprobs = ref_logprobs.contiguous()
    if logits.is_cuda:
        return PreferenceLoss(*_build_ops.load().preference_loss(logits, targets, vocab, ref_logprobs, offsets, beta,
                                                                 smoothing, average))
    logprobs, counted = _plain_logprobs(logits, targets, vocab, 1.0)
    if offsets is None:
        sums, tokens = logprobs.double().sum(1), counted.sum(1)
    else:
        pairs = list(zip(marks, marks[1:]))
        sums = torch.stack([logprobs[a:b].double().sum() for a, b in pairs])
        tokens = torch.stack([counted[a:b].sum() for a, b in pairs])
    if average:
        sums = sums / tokens.clamp(min=1)
    rewards = beta * (sums - ref_logprobs.double())
    margin = rewards[:sequences // 2] - rewards[sequences // 2:]
    log_sigmoid = torch.nn.functional.logsigmoid
    loss = (-(1 - smoothing) * log_sigmoid(margin) - smoothing * log_sigmoid(-margin)).mean()
    return PreferenceLoss(loss.to(logprobs.dtype), rewards.detach().float(), sums.detach().float())
