"""The language-model loss of a fine-tuning step, straight from the hidden states: softmax cross entropy against the
head's rows, without the logits (tokens x vocabulary) ever in memory, and its gradients.

A frozen head (LoRA) takes two products with the head, both in the forward call: the probabilities, in pieces of the
vocabulary, and the hidden states' gradient up to the loss's own upstream gradient; the backward call scales it. A
head that is trained too has its logits computed again in the backward call, since its gradient sums over tokens whose
log-sums have to be known first.
"""

import ctypes
import functools

import torch

from . import _lib

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}  # enum meep2b_reduction
_pack = _lib.packer(_lib.LinearCE).pack


@functools.lru_cache(maxsize=256)
def _plan(tokens, hidden_size, vocab):
    rows_pad, piece_cols, planes = ctypes.c_int64(), ctypes.c_int64(), ctypes.c_int32()
    _lib.check(_lib.load().meep2b_linear_ce_plan(tokens, hidden_size, vocab, ctypes.byref(rows_pad),
                                                 ctypes.byref(piece_cols), ctypes.byref(planes)),
               "meep2b_linear_ce_plan")
    return rows_pad.value, piece_cols.value, planes.value


def _rows(t):
    """A 2-D tensor as rows that TMA and 16-byte loads can address: itself, or a copy."""
    ld, inner = t.stride()
    if inner == 1 and ld % 8 == 0 and ld >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _call(what, weight, targets, ignore_index, reduction, plan, piece_cols, kept, hidden=0, ld_hidden=0, compact=0,
          acc=0, piece=0, part=0, row_loss=0, loss=0, upstream=0, d_hidden=0, d_weight=0):
    rows_pad, _, planes = plan
    vocab, size = weight.shape
    # what the passes keep of every row: state (8), flags (rows_pad / 256), source, slot, target and the row values
    state = kept.data_ptr()
    source = state + 4 * (8 + rows_pad // 256)
    step = 4 * rows_pad
    args = _pack(hidden, targets.numel(), size, ld_hidden, weight.data_ptr(), vocab, weight.stride(0),
                 targets.data_ptr(), ignore_index, _REDUCTIONS[reduction], planes, rows_pad, piece_cols, state, state + 32,
                 source, source + step, source + 2 * step, source + 3 * step, compact, acc, piece, part, row_loss, loss,
                 upstream, d_hidden, d_weight)
    _lib.check(getattr(_lib.load(), what)(args, _lib.stream_of(weight)), what)


def _bytes(sizes, device):
    """One buffer for all of these sizes, and the address of each (256 bytes apart at least)."""
    at, ends = 0, []
    for n in sizes:
        ends.append(at)
        at += (n + 255) & ~255
    buffer = torch.empty(at, dtype=torch.uint8, device=device)
    base = buffer.data_ptr()
    return buffer, [base + e for e in ends]


def _forward(hidden, weight, targets, ignore_index, reduction, accumulate, keep_rows):
    """The loss, and what the backward pass needs: the rows' values, with `accumulate` the planes of the hidden states'
    gradient, with `keep_rows` the copied rows."""
    tokens, size = hidden.shape
    vocab = weight.shape[0]
    dev = hidden.device
    plan = rows_pad, piece_cols, planes = _plan(tokens, size, vocab)
    kept = torch.empty(8 + rows_pad // 256 + 8 * rows_pad, dtype=torch.int32, device=dev)
    loss = torch.empty(tokens if reduction == "none" else (), dtype=torch.float32, device=dev)
    slots = 2 * ((vocab + 255) // 256)
    rows = torch.empty((rows_pad, size), dtype=torch.bfloat16, device=dev) if keep_rows else None
    acc = torch.empty((planes, rows_pad, size), dtype=torch.float32, device=dev) if accumulate else None
    scratch, (part, row_loss, compact, piece) = _bytes(
        (4 * slots * rows_pad, 4 * rows_pad, 0 if keep_rows else 2 * rows_pad * size,
         2 * rows_pad * piece_cols if accumulate else 0), dev)
    _call("meep2b_linear_ce_forward", weight, targets, ignore_index, reduction, plan, piece_cols if accumulate else 0,
          kept, hidden=hidden.data_ptr(), ld_hidden=hidden.stride(0),
          compact=rows.data_ptr() if keep_rows else compact, acc=acc.data_ptr() if accumulate else 0,
          piece=piece if accumulate else 0, part=part, row_loss=row_loss, loss=loss.data_ptr())
    return loss, kept, rows, acc, plan


def _backward(ctx, grad):
    weight, targets, kept, last = ctx.saved_tensors
    need_hidden, need_weight = ctx.needs_input_grad[:2]
    w = _rows(weight)
    vocab, size = w.shape
    rows_pad, piece_cols, planes = ctx.plan
    upstream = grad.to(torch.float32).contiguous()
    d_hidden = w.new_empty((targets.numel(), size)) if need_hidden else None
    d_weight = None
    where = dict(upstream=upstream.data_ptr(), d_hidden=d_hidden.data_ptr() if need_hidden else 0)
    if need_weight:
        d_weight = w.new_empty((vocab, size))
        scratch, (piece, acc) = _bytes((2 * rows_pad * piece_cols, 4 * planes * rows_pad * size if need_hidden else 0),
                                       w.device)
        where.update(piece=piece, acc=acc if need_hidden else 0, compact=last.data_ptr(), d_weight=d_weight.data_ptr())
    else:
        where.update(acc=last.data_ptr())
    _call("meep2b_linear_ce_backward", w, targets, ctx.ignore_index, ctx.reduction, ctx.plan, piece_cols, kept, **where)
    return d_hidden, d_weight, None, None, None


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore_index, reduction):
        train_head = ctx.needs_input_grad[1]
        accumulate = ctx.needs_input_grad[0] and not train_head
        loss, kept, rows, acc, ctx.plan = _forward(_rows(hidden), _rows(weight), targets, ignore_index, reduction,
                                                   accumulate, train_head)
        # of the hidden states the backward pass reads the copied rows, and those with a trained head alone
        ctx.save_for_backward(weight, targets, kept, rows if train_head else acc)
        ctx.reduction, ctx.ignore_index = reduction, ignore_index
        return loss

    @staticmethod
    def backward(ctx, grad):
        return _lib.once(_backward)(ctx, grad)


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
    if torch.is_grad_enabled() and (flat.requires_grad or weight.requires_grad):
        loss = _LinearCrossEntropy.apply(flat, weight, t, ignore_index, reduction)
    else:
        loss = _forward(_rows(flat.detach()), _rows(weight.detach()), t, ignore_index, reduction, False, False)[0]
    return loss.view(targets.shape) if reduction == "none" else loss
