"""train-gpt's `losses.py` on the CUDA path: the capped-logit cross-entropy and its gradient from
one pass over the logits.

The reference computes `cross_entropy_loss(params, input_ids, target_ids, cfg)` as
`forward(...)` (which ends with `cap * tanh(logits / cap)`, model.py:97), a float32 cast,
`log_softmax`, a gather and a mean (losses.py:8-12).  Here the part after the unembedding
GEMM is `capped_cross_entropy(logits, target_ids, cap)`: it takes the GEMM's raw bf16 output,
so the capped logits and their float32 copy are never written to memory.

`top_logits` and `capped_distillation` have no counterpart in the reference: a teacher's largest logits with their
log-probabilities, and a student's loss against them, on the same capped logits.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import ops


def capped_cross_entropy(logits: torch.Tensor, target_ids: torch.Tensor, cap: float) -> torch.Tensor:
    """Mean over tokens of -log_softmax(cap * tanh(logits / cap))[target] (model.py:97, losses.py:8-12).

    logits: (..., vocab) bf16, the unembedding GEMM's output BEFORE the cap; target_ids: (...)
    integer.  Any vocabulary size (the reference's default 50257 is not a multiple of 8).
    Differentiable with respect to logits.

    With gradients on and logits that require one, the FORWARD writes the gradient too (for an upstream
    gradient of 1; another one is seen in the backward pass and the gradient made again from the logits): one
    read of the logits serves both.  The logits and a tensor of their size stay allocated until the backward pass
    or the result's end, and a loss that is never differentiated pays for the write: 8192 x 50257 359 us with it,
    230 under `torch.no_grad()`.  (A vocabulary or cap that a row in shared memory cannot hold
    takes two passes, which keep one tensor of that size.)"""
    return ops._host().capped_cross_entropy(logits, target_ids, cap)


class TopLogits(NamedTuple):
    """A teacher's answer for every token: the ids of its largest logits (..., k) int32 or int64, their log-probabilities
    (..., k) float32, and the log of the probability that all other ids share (...) float32, or None where the k
    probabilities are to stand for the whole distribution.  An id outside the vocabulary (-1) is no entry."""

    ids: torch.Tensor
    logp: torch.Tensor
    log_rest: Optional[torch.Tensor] = None


def top_logits(logits: torch.Tensor, cap: float, k: int, temperature: float = 1.0) -> TopLogits:
    """The k largest logits of every token in descending order (equal ones by id; -0 is 0, a NaN above all), with
    log_softmax(cap * tanh(logits / cap) / temperature) at them and the log of the sum over the rest, in float32.

    logits: (..., vocab) bf16, uncapped as `capped_cross_entropy` takes them; rows may have a pitch (a slice of a padded
    vocabulary).  1 <= k <= 256, vocab <= 2**20, 2**-10 <= cap <= 64, 0 < temperature <= 1024, cap / temperature <= 64.
    Nothing is differentiated.  A row is read once and, for a first bound, an eighth of it (all of it below 16400 logits; rows of up to
    249, 505 and 1017 logits with at most 64, 48 and 20 kept are read once); the result does not depend on scheduling.  A row with hundreds of
    logits equal to the k-th, or with a NaN, is read some five to twenty times."""
    return TopLogits(*ops._host().top_logits(logits, cap, k, temperature))


def capped_distillation(logits: torch.Tensor, teacher: TopLogits, cap: float, target_ids: Optional[torch.Tensor] = None,
                        temperature: float = 1.0, weight: float = 1.0) -> torch.Tensor:
    """The student's loss against a teacher's top logits, the mean over tokens of

        weight T^2 [ sum_j p_j (log p_j - log q_j) + p_rest (log p_rest - log q_rest) ] + (1 - weight) CE(target)

    with q = softmax(cap * tanh(logits / cap) / T), p_j and p_rest the teacher's probabilities (`top_logits` at the same
    temperature) and q_rest the student's probability of all ids that the teacher does not name; without log_rest the second
    term is left out.  CE is the cross-entropy at temperature 1 of target_ids, needed where weight < 1.  Everything in float32
    (`capped_cross_entropy` rounds the capped logits to bf16 as the reference does).

    logits (..., vocab) bf16 as top_logits takes them; teacher.ids (..., k) with k <= 256; target_ids (...) int32 or int64.
    Ids and targets outside the vocabulary take no part (their logp is not read): a padded token with ids of -1, a target of -1
    and log_rest 0 adds 0 to the sum and has gradient 0, but counts in the mean.  An id named twice is one logit with both
    probabilities.  Differentiable once, in reverse mode, with respect to logits.

    As with `capped_cross_entropy`, with gradients on the FORWARD writes the gradient too, from the same read of the logits
    (from a second one beyond some 100000 logits a row); logits and
    gradient stay allocated until the backward pass or the result's end.  An upstream gradient other than 1 makes the gradient again from
    the inputs, or scales the one at hand where they were overwritten in between; tensors made under `torch.inference_mode()`, which count
    no changes, are copied."""
    return ops._host().capped_distillation(logits, teacher.ids, teacher.logp, teacher.log_rest, cap, target_ids, temperature, weight)
