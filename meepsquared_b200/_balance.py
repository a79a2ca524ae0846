"""The load-balancing loss of the routers (Transformers' ``load_balancing_loss_func``) and the tokens each expert got,
over one layer or all of them in one call, with the gradient of the router logits."""

import array

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_pack = _lib.packer(_lib.Balance).pack
MAX_LAYERS, MAX_EXPERTS, MAX_TOKENS = 128, 1024, 1 << 27


def _table(pointers):
    """A host array of device pointers; it has to outlive the call that its address goes to."""
    return array.array("Q", pointers)


def _rows(logits):
    """The layers' logits as contiguous tensors, and the table of their pointers."""
    rows = [x if x.is_contiguous() else x.contiguous() for x in logits]
    return rows, _table([x.data_ptr() for x in rows])


def _call(what, first, table, top_k, mask, coef, index=0, counts=0, loss=0, workspace=0, upstream=0, grads=0):
    tokens, experts = first.shape
    args = _pack(table.buffer_info()[0], len(table), experts, tokens, top_k, _DTYPES[first.dtype],
                 0 if mask is None else mask.data_ptr(), index, counts, loss, coef, workspace, upstream, grads)
    _lib.check(getattr(_lib.load(), what)(args, _lib.stream_of(first)), what)


def _forward(logits, top_k, mask, index):
    rows, table = _rows(logits)
    first = rows[0]
    dev = first.device
    experts = first.shape[1]
    counts = torch.empty((len(rows), experts) if len(rows) > 1 else (experts,), dtype=torch.int64, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    # the kernel's sums (64-bit), then the coefficients that the backward pass reads
    work = torch.empty(2 * (experts + 3) + experts, dtype=torch.float32, device=dev)
    at = work.data_ptr()
    ids = None if index is None else _table([i.data_ptr() for i in index])
    _call("meep2b_balance_loss", first, table, top_k, mask, at + 8 * (experts + 3),
          0 if ids is None else ids.buffer_info()[0], counts.data_ptr(), loss.data_ptr(), at)
    return loss, counts, work


def _backward(ctx, grad, _):
    work, mask, *logits = ctx.saved_tensors
    rows, table = _rows(logits)
    first = rows[0]
    layers = len(rows)
    upstream = grad if grad.dtype == torch.float32 else grad.to(torch.float32)
    if layers == 1:
        grads = (torch.empty_like(first),)
        base = grads[0].data_ptr()
    else:  # one allocation for all layers: the gradients are its slices
        every = torch.empty((layers, *first.shape), dtype=first.dtype, device=first.device)
        grads, base = every.unbind(0), every.data_ptr()
    step = first.numel() * first.element_size()
    outs = _table(range(base, base + layers * step, step) if step else [base] * layers)
    _call("meep2b_balance_loss_backward", first, table, ctx.top_k, mask, work.data_ptr() + 8 * (first.shape[1] + 3),
          upstream=upstream.data_ptr(), grads=outs.buffer_info()[0])
    need = ctx.needs_input_grad
    return (None, None, None, *(grads if all(need[3:]) else [g if n else None for g, n in zip(grads, need[3:])]))


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, top_k, mask, index, *logits):
        loss, counts, work = _forward(logits, top_k, mask, index)
        ctx.save_for_backward(work, mask, *logits)
        ctx.top_k = top_k
        ctx.mark_non_differentiable(counts)
        return loss, counts

    @staticmethod
    def backward(ctx, grad, _):
        return _lib.once(_backward)(ctx, grad, _)


def balance_loss(router_logits, top_k: int, mask=None, top_k_index=None):
    """The routers' load-balancing loss and the tokens of each expert: (loss, counts).

    router_logits: (T, E) float32 or bf16, or a list or tuple of them, one per layer (up to 128 layers, 1024 experts and
    2^27 tokens in all). Over the N unmasked tokens of all layers, with f_e the share of the tokens that chose expert e (each token chooses
    top_k) and m_e the mean of its softmax probability, loss = E * sum_e f_e m_e: float32, differentiable in the logits
    (once; the choice carries no gradient). The choice is the top_k largest logits, the lower expert first where they are
    equal, or top_k_index ((T, top_k) integers per layer; ids outside the experts count for none). mask (T): tokens
    where it is zero (padding) are left out, whatever their logits hold, and get a zero gradient; with no token left the
    loss is zero. counts: int64, (E,) for one tensor and (layers, E) for a list of more than one."""
    logits = [router_logits] if isinstance(router_logits, torch.Tensor) else list(router_logits)
    if not logits:
        raise ValueError("no router logits")
    first = logits[0]
    if not first.is_cuda:
        raise RuntimeError("balance_loss runs on a CUDA GPU")
    shape, dtype, dev = first.shape, first.dtype, first.device
    if len(shape) != 2 or any(x.shape != shape or x.dtype != dtype or x.device != dev for x in logits[1:]):
        raise ValueError("router logits: (tokens, experts) of one shape, type and device expected for every layer")
    if dtype not in _DTYPES:
        raise TypeError(f"router logits in {dtype}: float32 or bf16 expected")
    tokens, experts = shape
    if not 1 <= experts <= MAX_EXPERTS or len(logits) > MAX_LAYERS or tokens * len(logits) > MAX_TOKENS:
        raise ValueError(f"{len(logits)} layers of {tokens} tokens and {experts} experts: at most {MAX_LAYERS} layers, "
                         f"{MAX_TOKENS} tokens in all of them and {MAX_EXPERTS} experts")
    if not 1 <= top_k <= experts:
        raise ValueError(f"top_k {top_k} of {experts} experts")
    if mask is not None:
        if mask.shape != (tokens,) or mask.device != dev:
            raise ValueError(f"mask {tuple(mask.shape)}: ({tokens},) on the logits' device expected")
        mask = (mask if mask.dtype == torch.bool else mask != 0).contiguous()
    index = None
    if top_k_index is not None:
        index = [top_k_index] if isinstance(top_k_index, torch.Tensor) else list(top_k_index)
        if len(index) != len(logits) or any(i.shape != (tokens, top_k) or i.device != dev for i in index):
            raise ValueError(f"top_k_index: ({tokens}, {top_k}) per layer on the logits' device expected")
        if any(i.is_floating_point() for i in index):
            raise TypeError("top_k_index: integers expected")
        index = [i.to(torch.int64).contiguous() for i in index]
    if torch.is_grad_enabled() and any(x.requires_grad for x in logits):
        return _BalanceLoss.apply(top_k, mask, index, *logits)
    return _forward(logits, top_k, mask, index)[:2]
