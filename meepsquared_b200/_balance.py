"""The load-balancing loss of the routers (Transformers' ``load_balancing_loss_func``) and the tokens each expert got,
over one layer or all of them in one call, with the gradient of the router logits."""

import ctypes

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
MAX_LAYERS, MAX_EXPERTS = 128, 1024


def _pointers(tensors):
    return (ctypes.c_void_p * len(tensors))(*[t.data_ptr() for t in tensors])


def _struct(logits, top_k, mask, coef):
    tokens, experts = logits[0].shape
    table = _pointers(logits)
    a = _lib.Balance(logits=ctypes.addressof(table), layers=len(logits), experts=experts, tokens=tokens, top_k=top_k,
                     dtype=_DTYPES[logits[0].dtype], mask=None if mask is None else mask.data_ptr(),
                     coef=coef.data_ptr())
    return a, table  # the table has to outlive the call


def _forward(logits, top_k, mask, index):
    lib = _lib.load()
    dev = logits[0].device
    experts = logits[0].shape[1]
    counts = torch.empty((len(logits), experts), dtype=torch.int64, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    coef = torch.empty(experts, dtype=torch.float32, device=dev)
    work = torch.empty(lib.meep2b_balance_workspace_bytes(experts), dtype=torch.uint8, device=dev)
    a, table = _struct(logits, top_k, mask, coef)
    ids = None if index is None else _pointers(index)
    if ids is not None:
        a.index = ctypes.addressof(ids)
    a.counts, a.loss, a.workspace = counts.data_ptr(), loss.data_ptr(), work.data_ptr()
    _lib.check(lib.meep2b_balance_loss(ctypes.byref(a), _lib.stream_of(logits[0])), "meep2b_balance_loss")
    return loss, counts, coef


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, top_k, mask, index, *logits):
        rows = [x.detach().contiguous() for x in logits]
        loss, counts, coef = _forward(rows, top_k, mask, index)
        ctx.save_for_backward(coef, mask, *logits)
        ctx.top_k = top_k
        ctx.mark_non_differentiable(counts)
        return loss, counts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        coef, mask, *logits = ctx.saved_tensors
        rows = [x.detach().contiguous() for x in logits]
        upstream = grad.to(torch.float32).contiguous()
        # one allocation for all layers: the gradients are its slices
        grads = list(torch.empty((len(rows), *rows[0].shape), dtype=rows[0].dtype, device=rows[0].device).unbind(0))
        a, table = _struct(rows, ctx.top_k, mask, coef)
        outs = _pointers(grads)
        a.grads, a.upstream = ctypes.addressof(outs), upstream.data_ptr()
        _lib.check(_lib.load().meep2b_balance_loss_backward(ctypes.byref(a), _lib.stream_of(rows[0])),
                   "meep2b_balance_loss_backward")
        return (None, None, None, *[g if need else None for g, need in zip(grads, ctx.needs_input_grad[3:])])


def balance_loss(router_logits, top_k: int, mask=None, top_k_index=None):
    """The routers' load-balancing loss and the tokens of each expert: (loss, counts).

    router_logits: (T, E) float32 or bf16, or a list or tuple of them, one per layer (up to 128 layers, 1024 experts).
    Over the N unmasked tokens of all layers, with f_e the share of the tokens that chose expert e (each token chooses
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
    if first.dim() != 2 or any(x.shape != first.shape or x.dtype != first.dtype or x.device != first.device
                               for x in logits):
        raise ValueError("router logits: (tokens, experts) of one shape, type and device expected for every layer")
    if first.dtype not in _DTYPES:
        raise TypeError(f"router logits in {first.dtype}: float32 or bf16 expected")
    tokens, experts = first.shape
    if not 1 <= experts <= MAX_EXPERTS or len(logits) > MAX_LAYERS:
        raise ValueError(f"{len(logits)} layers of {experts} experts: at most {MAX_LAYERS} and {MAX_EXPERTS}")
    if not 1 <= top_k <= experts:
        raise ValueError(f"top_k {top_k} of {experts} experts")
    if mask is not None:
        if tuple(mask.shape) != (tokens,) or mask.device != first.device:
            raise ValueError(f"mask {tuple(mask.shape)}: ({tokens},) on the logits' device expected")
        mask = (mask if mask.dtype == torch.bool else mask != 0).contiguous()
    index = None
    if top_k_index is not None:
        index = [top_k_index] if isinstance(top_k_index, torch.Tensor) else list(top_k_index)
        if len(index) != len(logits) or any(tuple(i.shape) != (tokens, top_k) or i.device != first.device
                                            for i in index):
            raise ValueError(f"top_k_index: ({tokens}, {top_k}) per layer on the logits' device expected")
        if any(i.is_floating_point() for i in index):
            raise TypeError("top_k_index: integers expected")
        index = [i.to(torch.int64).contiguous() for i in index]
    if torch.is_grad_enabled() and any(x.requires_grad for x in logits):
        loss, counts = _BalanceLoss.apply(top_k, mask, index, *logits)
    else:
        loss, counts, _ = _forward([x.detach().contiguous() for x in logits], top_k, mask, index)
    return loss, counts[0] if len(logits) == 1 else counts
