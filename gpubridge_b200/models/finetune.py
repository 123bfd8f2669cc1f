"""What a language model of this package is fine-tuned with: log-probabilities of tokens, the clipped
policy loss and the preference loss, each from token ids to the loss (``ops/logprob.py`` holds the
formulas).  ``models/gpt2.py`` and ``models/llama.py`` take these methods over; a trainer calls them
from its ``loss_fn``:

    trainer = DataParallelTrainer(model, lambda m, *batch: m.policy_loss(*batch).loss, max_grad_norm=1.0)
"""
from __future__ import annotations

import os

import torch

from gpubridge_b200.ops.logprob import PolicyLoss, PreferenceLoss, policy_loss, preference_loss, token_logprobs


def fused_join() -> bool:
    """Whether models whose configuration does not ask for it join their blocks with the fused
    kernel as well (``GPUBRIDGE_FUSED_JOIN=1``; off by default)."""
    return os.environ.get("GPUBRIDGE_FUSED_JOIN", "0") == "1"


class FineTuned:
    """Mixed into a module with ``config.vocab``, ``unit_grad`` and ``logits(idx)`` ->
    ``[batch, time, columns]`` of which the first ``config.vocab`` columns count.  Targets outside
    the vocabulary (-100) mark prompt and padding."""

    def logprobs(self, idx: torch.Tensor, targets: torch.Tensor, temperature: float = 1.0) -> torch.Tensor:
        """Log-probability of each target, ``[batch, time]`` float32 (under ``torch.no_grad()`` for the
        sampling policy's and the reference model's)."""
        return token_logprobs(self.logits(idx), targets, self.config.vocab, temperature=temperature)

    def policy_loss(self, idx: torch.Tensor, targets: torch.Tensor, old_logprobs: torch.Tensor,
                    advantages: torch.Tensor, ref_logprobs: torch.Tensor | None = None, **options) -> PolicyLoss:
        """Clipped policy loss of sampled tokens; ``options`` as in :func:`ops.logprob.policy_loss`."""
        options.setdefault("unit_grad", self.unit_grad)
        return policy_loss(self.logits(idx), targets, old_logprobs, advantages, ref_logprobs=ref_logprobs,
                           vocab=self.config.vocab, **options)

    def preference_loss(self, idx: torch.Tensor, targets: torch.Tensor, ref_logprobs: torch.Tensor,
                        **options) -> PreferenceLoss:
        """Preference loss of a batch whose first half was chosen over its second half, with the
        reference model's log-probability of each sequence; ``options`` as in
        :func:`ops.logprob.preference_loss`."""
        return preference_loss(self.logits(idx), targets, ref_logprobs, vocab=self.config.vocab, **options)
