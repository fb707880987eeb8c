"""Distillation from a teacher's top log-probabilities, differentiable in the student's logits.

The teacher's side is the sampler's: ``top_logprobs`` after a sampling call leaves, for each row,
the most likely ids and their log-probabilities (id -1 for an empty entry, -inf outside the kept
set), on the device and in the layout taken here. For rows of student logits ``x``, temperature
``T`` and ``q = softmax(x / T)``, with ``p_j = exp(logprobs_j)``:

* without ``tail`` the list is renormalised to one: ``loss = sum_j p_j (ln p_j - ln q_j)``;
* with ``tail`` the mass the list leaves over, ``p_t = 1 - sum_j p_j``, is matched with the
  student's mass outside the list: ``... + p_t (ln p_t - ln q_t)``.

The sums run over entries: an id listed twice has the gradient of one entry with its masses' sum, and a
loss that is lower by a constant (the teacher's ``p ln p`` are taken entry by entry).

The log-probabilities are the teacher's at the same temperature. The reference trains nothing; the
losses carry no factor ``T ** 2`` (a weight may).
"""

from __future__ import annotations

from typing import TYPE_CHECKING

import torch
from torch.autograd import forward_ad

if TYPE_CHECKING:
    from vinfer_b200.kernels.sampler.b200 import B200Sampler


class _ListLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, backend, ids, logprobs, weights, temperature, tail):
        loss, saved = backend.distill_loss(
            logits, ids, logprobs, weights, temperature=temperature, tail=tail,
            for_grad=ctx.needs_input_grad[0])
        ctx.save_for_backward(logits, ids, logprobs, weights, saved)
        ctx.backend, ctx.temperature, ctx.tail = backend, temperature, tail
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        logits, ids, logprobs, weights, saved = ctx.saved_tensors
        grad = ctx.backend.distill_grad(
            logits, ids, logprobs, weights, saved, grad_out,
            temperature=ctx.temperature, tail=ctx.tail)
        return grad, None, None, None, None, None, None


def distillation_loss(backend: B200Sampler, logits: torch.Tensor, ids: torch.Tensor,
                      logprobs: torch.Tensor, weights: torch.Tensor | None = None, *,
                      temperature: float = 1.0, tail: bool = False) -> torch.Tensor:
    """Each row's loss, float32 ``[rows]``: ``logits`` ``[rows, vocab]`` (float32 or bfloat16, any
    row stride), ``ids`` int32 and ``logprobs`` float32 ``[rows, k]`` with ``k <= 128``,
    ``weights`` float32 ``[rows]`` (a row of weight 0 is not read and gets loss and gradient 0).
    Gradients flow to ``logits`` alone, once: there is no second derivative. Where the weights of the
    sum are known ahead, ``backend.distill_step`` computes loss and gradient in one call. As with every
    torch operation, a backward pass is captured into a CUDA graph only while no eager graph of the
    same leaves is alive; ``distill_step`` knows no leaves."""
    if not (logits.requires_grad and torch.is_grad_enabled()) and forward_ad._current_level < 0:
        # nothing to record (the autograd function costs a call 6 us): the loss alone
        return backend.distill_loss(logits, ids, logprobs, weights, temperature=temperature,
                                    tail=tail)[0]
    return _ListLoss.apply(logits, backend, ids, logprobs, weights, temperature, tail)
