"""The load-balancing loss of the routers (Transformers' ``load_balancing_loss_func``) and the tokens each expert got,
over one layer or all of them in one call, with the gradient of the router logits."""

import torch

from . import _lib

_DTYPES = (torch.float32, torch.bfloat16)
MAX_LAYERS, MAX_EXPERTS, MAX_TOKENS = 128, 1024, 1 << 27


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
    index = []
    if top_k_index is not None:
        index = [top_k_index] if isinstance(top_k_index, torch.Tensor) else list(top_k_index)
        if len(index) != len(logits) or any(i.shape != (tokens, top_k) or i.device != dev for i in index):
            raise ValueError(f"top_k_index: ({tokens}, {top_k}) per layer on the logits' device expected")
        if any(i.is_floating_point() for i in index):
            raise TypeError("top_k_index: integers expected")
        index = [i.to(torch.int64).contiguous() for i in index]
    return _lib.native().balance_loss(logits, top_k, mask, index)
