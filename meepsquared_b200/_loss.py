"""The language-model loss of a fine-tuning step, straight from the hidden states: softmax cross entropy against the
head's rows, without the logits (tokens x vocabulary) ever in memory, and its gradients.

A frozen head (LoRA) takes two products with the head, both in the forward call: the probabilities, in pieces of the
vocabulary, and the hidden states' gradient up to the loss's own upstream gradient; the backward call scales it. A
head that is trained too has its logits computed again in the backward call, since its gradient sums over tokens whose
log-sums have to be known first.
"""

import ctypes

import torch

from . import _lib

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}  # enum meep2b_reduction


def _plan(tokens, hidden_size, vocab):
    rows_pad, piece_cols, planes = ctypes.c_int64(), ctypes.c_int64(), ctypes.c_int32()
    _lib.check(_lib.load().meep2b_linear_ce_plan(tokens, hidden_size, vocab, ctypes.byref(rows_pad),
                                                 ctypes.byref(piece_cols), ctypes.byref(planes)),
               "meep2b_linear_ce_plan")
    return rows_pad.value, piece_cols.value, planes.value


def _rows(t):
    """A 2-D tensor as rows that TMA and 16-byte loads can address: itself, or a copy."""
    if t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _struct(weight, targets, ignore_index, reduction, kept, plan):
    rows_pad, _, planes = plan
    ints, values, compact = kept
    at = ints.data_ptr()
    a = _lib.LinearCE(tokens=targets.numel(), hidden_size=weight.shape[1], weight=weight.data_ptr(),
                      vocab=weight.shape[0], ld_weight=weight.stride(0), targets=targets.data_ptr(),
                      ignore_index=ignore_index, reduction=_REDUCTIONS[reduction], planes=planes, rows_pad=rows_pad,
                      piece_cols=0, row_values=values.data_ptr(), compact=compact.data_ptr())
    # state (8), flags (rows_pad / 256), source, slot and target (rows_pad each) in one tensor
    flags = rows_pad // 256
    a.state, a.flags = at, at + 32
    at += 4 * (8 + flags)
    a.source, a.slot, a.target = at, at + 4 * rows_pad, at + 8 * rows_pad
    return a


def _forward(hidden, weight, targets, ignore_index, reduction, accumulate):
    """The loss, and what the backward pass needs; with `accumulate` the planes of the hidden states' gradient."""
    tokens, size = hidden.shape
    vocab = weight.shape[0]
    dev = hidden.device
    plan = _plan(tokens, size, vocab)
    rows_pad, piece_cols, planes = plan
    ints = torch.empty(8 + rows_pad // 256 + 3 * rows_pad, dtype=torch.int32, device=dev)
    slots = 2 * ((vocab + 255) // 256)
    values = torch.empty(5 * rows_pad, dtype=torch.float32, device=dev)
    scratch = torch.empty((slots + 1) * rows_pad, dtype=torch.float32, device=dev)
    compact = torch.empty((rows_pad, size), dtype=torch.bfloat16, device=dev)
    loss = torch.empty(tokens if reduction == "none" else (), dtype=torch.float32, device=dev)
    a = _struct(weight, targets, ignore_index, reduction, (ints, values, compact), plan)
    a.hidden, a.ld_hidden = hidden.data_ptr(), hidden.stride(0)
    a.part, a.row_loss, a.loss = scratch.data_ptr(), scratch.data_ptr() + 4 * slots * rows_pad, loss.data_ptr()
    acc = None
    if accumulate:
        acc = torch.empty((planes, rows_pad, size), dtype=torch.float32, device=dev)
        piece = torch.empty((rows_pad, piece_cols), dtype=torch.bfloat16, device=dev)
        a.acc, a.piece, a.piece_cols = acc.data_ptr(), piece.data_ptr(), piece_cols
    _lib.check(_lib.load().meep2b_linear_ce_forward(ctypes.byref(a), _lib.stream_of(hidden)),
               "meep2b_linear_ce_forward")
    return loss, (ints, values, compact), acc, plan


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore_index, reduction):
        train_head = ctx.needs_input_grad[1]
        accumulate = ctx.needs_input_grad[0] and not train_head
        h, w = _rows(hidden.detach()), _rows(weight.detach())
        loss, (ints, values, compact), acc, ctx.plan = _forward(h, w, targets, ignore_index, reduction, accumulate)
        if train_head:  # of the hidden states the backward pass reads the copied rows alone
            ctx.save_for_backward(weight, targets, ints, values, compact)
        else:
            ctx.save_for_backward(weight, targets, ints, values, acc)
        ctx.train_head, ctx.reduction, ctx.ignore_index, ctx.tokens = train_head, reduction, ignore_index, h.shape[0]
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        weight, targets, ints, values, last = ctx.saved_tensors
        w = _rows(weight.detach())
        tokens, size = ctx.tokens, w.shape[1]
        rows_pad, piece_cols, planes = ctx.plan
        dev = w.device
        upstream = grad.to(torch.float32).contiguous()
        d_hidden = torch.empty((tokens, size), dtype=torch.bfloat16, device=dev) if ctx.needs_input_grad[0] else None
        d_weight = None
        a = _struct(w, targets, ctx.ignore_index, ctx.reduction, (ints, values, last), ctx.plan)
        a.upstream = upstream.data_ptr()
        if ctx.train_head:
            d_weight = torch.empty((w.shape[0], size), dtype=torch.bfloat16, device=dev)
            piece = torch.empty((rows_pad, piece_cols), dtype=torch.bfloat16, device=dev)
            a.piece, a.piece_cols, a.d_weight = piece.data_ptr(), piece_cols, d_weight.data_ptr()
            if d_hidden is not None:
                acc = torch.empty((planes, rows_pad, size), dtype=torch.float32, device=dev)
                a.acc, a.d_hidden = acc.data_ptr(), d_hidden.data_ptr()
        else:
            a.acc, a.d_hidden = last.data_ptr(), d_hidden.data_ptr()
        _lib.check(_lib.load().meep2b_linear_ce_backward(ctypes.byref(a), _lib.stream_of(w)),
                   "meep2b_linear_ce_backward")
        return d_hidden, d_weight, None, None, None


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
    if tuple(targets.shape) != tuple(hidden.shape[:-1]):
        raise ValueError(f"targets {tuple(targets.shape)}: {tuple(hidden.shape[:-1])} expected")
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError(f"hidden states in {hidden.dtype} and head in {weight.dtype}: the loss computes in bf16")
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"targets in {targets.dtype}: int64 or int32 expected")
    if weight.device != hidden.device or targets.device != hidden.device:
        raise ValueError("hidden states, head and targets are on different devices")
    if weight.shape[0] < 1 or weight.shape[1] < 1 or weight.shape[1] % 8:
        raise ValueError(f"head {tuple(weight.shape)}: at least one row, and a width that is a multiple of 8, expected")
    flat = hidden.reshape(-1, hidden.shape[-1])
    t = targets.reshape(-1).to(torch.int64).contiguous()
    if t.numel() == 0:  # nothing to compute; the graph is kept
        zero = (hidden.sum(dtype=torch.float32) + weight[:0].sum(dtype=torch.float32))
        return zero + hidden.new_zeros(targets.shape, dtype=torch.float32) if reduction == "none" else zero
    if torch.is_grad_enabled() and (flat.requires_grad or weight.requires_grad):
        loss = _LinearCrossEntropy.apply(flat, weight, t, ignore_index, reduction)
    else:
        loss = _forward(_rows(flat.detach()), _rows(weight.detach()), t, ignore_index, reduction, False)[0]
    return loss.view(targets.shape) if reduction == "none" else loss
