"""The language-model loss of a fine-tuning step, straight from the hidden states: softmax cross entropy against the
head's rows, without the logits (tokens x vocabulary) ever in memory, and its gradients.

A frozen head (LoRA) takes two products with the head, both in the forward call: the probabilities, in pieces of the
vocabulary, and the hidden states' gradient up to the loss's own upstream gradient; the backward call scales it. A
head that is trained too has its logits computed again in the backward call, since its gradient sums over tokens whose
log-sums have to be known first.
"""

import torch

from . import _lib

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}  # enum meep2b_reduction
# columns of a vocabulary piece (a multiple of 256) and planes of the gradient's sums; 0: as meep2b_linear_ce_plan says
PLAN = (0, 0)


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of the logits hidden @ weight.T against targets, without keeping the logits.

    hidden (..., H) bf16, weight (V, H) bf16 (H a multiple of 8), targets (...) integers, `ignore_index` where a token
    has none: its loss and its gradient are zero, whatever its hidden state holds. Returns float32: the mean over the
    tokens with a target ("mean"; zero where there are none), their sum ("sum"), or every token's loss, shaped as
    targets ("none"). Differentiable in hidden and weight (once). Sums and the softmax's statistics are float32; the
    probabilities are rounded to bf16 where they enter the gradients' products, and each gradient once at its end. A
    target outside the vocabulary makes its token's loss and gradients NaN."""
    if not hidden.is_cuda:
        raise RuntimeError("linear_cross_entropy runs on a CUDA GPU")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction {reduction!r}: 'none', 'mean' or 'sum' expected")
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden states {tuple(hidden.shape)} and head {tuple(weight.shape)}: (..., H) and (V, H) "
                         "expected")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"targets {tuple(targets.shape)}: {tuple(hidden.shape[:-1])} expected")
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError(f"hidden states in {hidden.dtype} and head in {weight.dtype}: the loss computes in bf16")
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"targets in {targets.dtype}: int64 or int32 expected")
    if weight.device != hidden.device or targets.device != hidden.device:
        raise ValueError("hidden states, head and targets are on different devices")
    if weight.shape[0] < 1 or weight.shape[1] < 1 or weight.shape[1] % 8:
        raise ValueError(f"head {tuple(weight.shape)}: at least one row, and a width that is a multiple of 8, expected")
    flat = hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])
    t = targets.reshape(-1).to(torch.int64).contiguous()
    if t.numel() == 0:  # nothing to compute; the graph is kept
        zero = (hidden.sum(dtype=torch.float32) + weight[:0].sum(dtype=torch.float32))
        return zero + hidden.new_zeros(targets.shape, dtype=torch.float32) if reduction == "none" else zero
    loss = _lib.native().linear_cross_entropy(flat, weight, t, ignore_index, _REDUCTIONS[reduction], *PLAN)
    return loss.view(targets.shape) if reduction == "none" else loss
