"""LoRA on every routed-expert stack of a Transformers mixture-of-experts model, computed by this package's routed
layer: the model-level step of the reference's ``meepsquared._moe.apply`` (meepsquared/_moe.py:208-227), which
patches each PEFT-wrapped experts module so that its forward runs the routed layer with the adapters' factors.

The reference finds the experts modules PEFT wrapped (``target_parameters`` on ``gate_up_proj`` / ``down_proj``)
and reads each wrapper's lora_A / lora_B as PEFT lays them out (``_delta_factors``, :148-163). Here the factors
are held by the experts module itself, in PEFT's layout and with PEFT's initialisation (lora_A kaiming-uniform,
lora_B zero), so that a model without PEFT installed gets the same trainable parameters:

* ``install(model, rank, alpha)`` adds ``lora_<stack>_lhs`` (experts, out, rank) and ``lora_<stack>_rhs``
  (experts, rank, in) to every experts module (Transformers' ``gate_up_proj (E, 2I, H)`` / ``down_proj (E, H, I)``
  layout, or the transposed one) and makes its forward ``_moe.routed_forward`` with them;
* ``install_attention(model)`` makes the attention modules that norm their query and key heads (q_norm, k_norm) do so
  with the rotation in one pass (``qk_norm_rope``);
* ``training_loss(model, input_ids, labels)`` is a fine-tuning step's loss without the logits (``linear_cross_entropy``
  on the last hidden states and the head), with the routers' balance loss and the tokens of every expert
  (``balance_loss``);
* ``lora_parameters(model)`` lists the factors, in the order a data-parallel gradient bucket wants them (each layer's
  down-projection factors before its gate/up ones, ``ddp.LoraGradBucket`` segments).

Experts modules of Transformers versions that predate the ``has_gate`` / ``has_bias`` / ``is_transposed``
attributes (which ``_moe.routed_forward`` reads, as the reference's ``_routed_forward`` does) get them from the
module's stacks: a ``gate_up_proj`` means gated, no ``*_bias`` means unbiased, and a stack stored (experts, 2I,
hidden) is not transposed.
"""

import inspect
import math
import types

import torch

from . import _moe
from ._balance import balance_loss
from ._heads import qk_norm_rope
from ._loss import linear_cross_entropy

# What makes a module an experts module. The reference asks for ("num_experts", "has_gate", "has_bias",
# "is_transposed") (_moe.py:31), the attributes of Transformers >= 5.17; an experts module of an older Transformers
# has the stacks and the expert count, and _complete() derives the rest.
EXPERTS_ATTRIBUTES = ("num_experts", "down_proj")
STACKS = ("gate_up_proj", "up_proj", "down_proj")  # the reference's STACKS (_moe.py:34)


def experts_modules(model):
    """(name, module) of every Transformers experts module of the model."""
    for name, module in model.named_modules():
        if all(hasattr(module, a) for a in EXPERTS_ATTRIBUTES) and isinstance(getattr(module, "down_proj"),
                                                                               torch.nn.Parameter):
            yield name, module


def _complete(experts):
    """The attributes _moe.routed_forward reads, derived from the stacks where an older module lacks them."""
    if not hasattr(experts, "has_gate"):
        experts.has_gate = hasattr(experts, "gate_up_proj")
    if not hasattr(experts, "has_bias"):
        experts.has_bias = any(hasattr(experts, f"{s}_bias") for s in STACKS)
    if not hasattr(experts, "is_transposed"):
        # (E, out, in) stacks: the first projection's input (hidden) is the down projection's output
        first = experts.gate_up_proj if experts.has_gate else experts.up_proj
        experts.is_transposed = first.shape[2] != experts.down_proj.shape[1]


def _stack_dims(experts, name):
    """(in, out) of the projection a stack computes."""
    w = getattr(experts, name)
    return (w.shape[1], w.shape[2]) if experts.is_transposed else (w.shape[2], w.shape[1])


def _forward(self, hidden_states, top_k_index, top_k_weights, *args, **kwargs):
    """The experts' forward with the adapters (the reference's _moe._forward, :128-145): the routed layer."""
    if args or kwargs:
        raise NotImplementedError("the routed experts take (hidden_states, top_k_index, top_k_weights)")
    factors = {name: (getattr(self, f"lora_{name}_lhs"), getattr(self, f"lora_{name}_rhs"), self.lora_scaling)
               for name in self.lora_stacks}
    return _moe.routed_forward(self, hidden_states, top_k_index, top_k_weights, factors)


def install(model, rank: int = 16, alpha: float = 16, dtype=torch.bfloat16, generator=None) -> int:
    """LoRA of the given rank on every expert stack of the model, computed by the routed layer; returns how many
    experts modules were patched. The stacks are frozen; the factors are trainable parameters of the experts
    module (PEFT's names lora_A / lora_B map to rhs / lhs), initialised as PEFT does (lhs zero, rhs kaiming-uniform
    with a = sqrt(5), that is U(-1/sqrt(in), 1/sqrt(in)))."""
    patched = 0
    for name, experts in experts_modules(model):
        _complete(experts)
        stacks = [s for s in ("gate_up_proj", "up_proj", "down_proj") if isinstance(getattr(experts, s, None),
                                                                                    torch.nn.Parameter)]
        for s in stacks:
            getattr(experts, s).requires_grad_(False)
            fan_in, out = _stack_dims(experts, s)
            e = experts.num_experts
            device = getattr(experts, s).device
            bound = 1.0 / math.sqrt(fan_in)
            rhs = (torch.rand((e, rank, fan_in), generator=generator) * 2 - 1) * bound  # on the CPU, then moved
            lhs = torch.zeros((e, out, rank))
            experts.register_parameter(f"lora_{s}_lhs", torch.nn.Parameter(lhs.to(device, dtype)))
            experts.register_parameter(f"lora_{s}_rhs", torch.nn.Parameter(rhs.to(device, dtype)))
        experts.lora_stacks = tuple(stacks)
        experts.lora_scaling = alpha / rank
        experts.forward = types.MethodType(_forward, experts)
        patched += 1
    return patched


def lora_parameters(model):
    """The factors install() added, each layer's down-projection factors before its gate/up ones."""
    params = []
    for _, experts in experts_modules(model):
        for s in ("down_proj", "gate_up_proj", "up_proj"):
            if s in getattr(experts, "lora_stacks", ()):
                params += [getattr(experts, f"lora_{s}_lhs"), getattr(experts, f"lora_{s}_rhs")]
    return params


def attention_modules(model):
    """(name, module) of every attention module that norms its query and key heads."""
    parts = ("q_proj", "k_proj", "v_proj", "o_proj", "q_norm", "k_norm", "head_dim")
    for name, module in model.named_modules():
        if all(hasattr(module, p) for p in parts):
            yield name, module


def _attention_implementation(module):
    """The attention that the module is configured for, or an error where it is one whose masks say something else.

    torch's attention and the plain one get every boundary as a (batch, 1, queries, keys) mask, and causal attention alone
    as none; the others take packed sequences without a mask, from the positions or from cu_seq_lens."""
    name = getattr(getattr(module, "config", None), "_attn_implementation", None)
    if name not in (None, "sdpa", "eager"):
        raise NotImplementedError(f"attention implementation {name!r}: load the model with attn_implementation='sdpa'")
    return name


def _attention_forward(self, hidden_states, position_embeddings, attention_mask=None, past_key_values=None, **kwargs):
    """The attention's forward with norms and rotation in one pass between the projections and torch's attention."""
    return _attention(self, qk_norm_rope, hidden_states, position_embeddings, attention_mask, past_key_values, **kwargs)


def _attention(self, norm_rotate, hidden_states, position_embeddings, attention_mask, past_key_values=None, **kwargs):
    implementation = _attention_implementation(self)  # (it may have been changed since install_attention)
    if attention_mask is None and any(kwargs.get(n) is not None for n in ("cu_seq_lens_q", "cu_seq_lens_k")):
        raise NotImplementedError("packed sequences (cu_seq_lens) need an attention mask that separates them")
    if kwargs.get("is_causal") is False:
        raise NotImplementedError("attention that is not causal (is_causal)")
    if implementation == "eager" and (kwargs.get("output_attentions") or getattr(self.config, "output_attentions", False)):
        raise NotImplementedError("attention weights (output_attentions) are not computed")
    batch, length = hidden_states.shape[:2]
    heads = (batch, length, -1, self.head_dim)
    q, k, v = (f(hidden_states).view(heads) for f in (self.q_proj, self.k_proj, self.v_proj))
    cos, sin = position_embeddings  # (1 or batch, length, rotated): both halves alike
    half = cos.shape[-1] // 2
    positions = None
    if cos.shape[0] > 1:
        positions = torch.arange(batch * length, device=q.device).view(batch, length)
    cos, sin = (x.reshape(-1, 2 * half)[:, :half] for x in (cos, sin))
    q, k = norm_rotate(q, k, self.q_norm.weight, self.k_norm.weight, cos, sin, positions=positions,
                        eps=self.q_norm.variance_epsilon)
    q, k, v = q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)
    if past_key_values is not None:
        k, v = past_key_values.update(k, v, self.layer_idx)
    if attention_mask is None and 1 < length < k.shape[2]:
        raise NotImplementedError("several new tokens behind cached ones need an attention mask")
    if attention_mask is not None and attention_mask.dim() != 4:
        raise NotImplementedError("an attention mask of (batch, 1, queries, keys) is expected: load the model with "
                                  "attn_implementation='sdpa'")
    out = torch.nn.functional.scaled_dot_product_attention(
        q, k, v, attn_mask=attention_mask, dropout_p=self.attention_dropout if self.training else 0.0,
        is_causal=attention_mask is None and length > 1, scale=self.scaling, enable_gqa=True)
    return self.o_proj(out.transpose(1, 2).reshape(batch, length, -1)), None


def _check_attention(name, module):
    """Refuses an attention module that _attention_forward does not compute: by what it says of itself, then by its own
    forward on a few random tokens."""
    _attention_implementation(module)
    if getattr(module, "sliding_window", None) is not None:
        raise NotImplementedError(f"{name}: attention within a sliding window")
    if not getattr(module, "is_causal", True):
        raise NotImplementedError(f"{name}: attention that is not causal")
    if not isinstance(getattr(module, "scaling", None), (int, float)) or not hasattr(module, "attention_dropout"):
        raise NotImplementedError(f"{name}: the scale or the dropout of its attention is not known")
    parts = ("q_proj", "k_proj", "v_proj", "o_proj", "q_norm", "k_norm")
    other = [n for n, _ in module.named_parameters() if n.split(".")[0] not in parts]
    if other:
        raise NotImplementedError(f"{name}: attention with parameters of its own ({other[0]})")
    for norm in (module.q_norm, module.k_norm):
        if not hasattr(norm, "variance_epsilon") or tuple(getattr(norm, "weight", torch.empty(0)).shape) != (module.head_dim,):
            raise NotImplementedError(f"{name}: norms over each head, with a weight of ({module.head_dim},), are expected")
    if module.q_norm.variance_epsilon != module.k_norm.variance_epsilon:
        raise NotImplementedError(f"{name}: norms of different epsilon")
    if module.head_dim % 16 or module.head_dim > 256:
        raise NotImplementedError(f"{name}: heads of {module.head_dim}: a multiple of 16 up to 256 is expected")
    if getattr(module.forward, "__func__", None) is not _attention_forward:  # not patched before
        _compare_attention(name, module)


def _plain_norm_rotate(q, k, q_weight, k_weight, cos, sin, positions=None, eps=1e-6):
    """qk_norm_rope in elementary operations (positions None), on any device."""
    n = cos.shape[1]
    cos, sin = (x.float()[:, None] for x in (cos, sin))

    def heads(x, w):
        y = x.float()
        y = y * (y.square().mean(-1, keepdim=True) + eps).rsqrt() * w.float()
        a, b = y[..., :n], y[..., n:2 * n]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 2 * n:]], -1).to(x.dtype)

    return heads(q, q_weight), heads(k, k_weight)


@torch.no_grad()
def _compare_attention(name, module, tokens=7):
    """Raises unless the module's own forward does what _attention_forward would, on random tokens, angles and norm weights
    (with its own, order and form of the norms may not show): within 5%, where bf16 rounds to 1% and a gate, a missing
    rotation or another order of norm and rotation change the output altogether."""
    weight = module.q_norm.weight
    if any(p.is_meta for p in module.parameters()):
        raise NotImplementedError(f"{name}: its weights are not loaded")
    gen = torch.Generator().manual_seed(0)
    kind = module.q_proj.weight.dtype  # what a quantised projection stores is not what it takes
    like = dict(device=weight.device, dtype=kind if kind in (torch.float32, torch.bfloat16, torch.float16) else weight.dtype)
    width = getattr(module.q_proj, "in_features", module.q_proj.weight.shape[-1])
    x = torch.randn((1, tokens, width), generator=gen).to(**like)
    angle = (6.28 * torch.rand((1, tokens, module.head_dim // 2), generator=gen)).repeat(1, 1, 2)
    angles = angle.cos().to(**like), angle.sin().to(**like)
    mask = torch.full((1, 1, tokens, tokens), torch.finfo(x.dtype).min).triu(1).to(**like)
    norms = {f"{n}.weight": (0.5 + torch.rand(weight.shape, generator=gen)).to(**like) for n in ("q_norm", "k_norm")}
    modes = [(m, m.training) for m in module.modules()]
    module.eval()
    try:
        call = dict(hidden_states=x, position_embeddings=angles, attention_mask=mask)
        want = torch.func.functional_call(module, norms, kwargs=call)
        before, module.forward = module.__dict__.get("forward"), types.MethodType(
            lambda self, **kwargs: _attention(self, _plain_norm_rotate, **kwargs), module)
        try:
            got = torch.func.functional_call(module, norms, kwargs=call)
        finally:
            del module.forward
            if before is not None:
                module.forward = before
    except (TypeError, ValueError, RuntimeError, AttributeError, IndexError, KeyError) as exc:
        raise NotImplementedError(f"{name}: its forward does not run as a Qwen3 attention's ({exc})") from exc
    finally:
        for m, mode in modes:
            m.training = mode
    want, got = (y[0].float() if isinstance(y, tuple) else y.float() for y in (want, got))
    if got.shape != want.shape or not bool((got - want).norm() <= 0.05 * want.norm()):
        raise NotImplementedError(f"{name}: its forward is not a Qwen3 attention's")


def install_attention(model) -> int:
    """qk_norm_rope in every attention module with normed heads (Transformers' Qwen3 layout: rotary pairs (i, i + n),
    torch's scaled_dot_product_attention behind it); returns how many were patched. Raises NotImplementedError, with none
    patched, if there is one that cannot be."""
    found = list(attention_modules(model))
    for name, module in found:  # all of them before the first is changed
        _check_attention(name, module)
    for _, module in found:
        module.forward = types.MethodType(_attention_forward, module)
    return len(found)


def _routers(model):
    """The routers beside the experts modules, in the layers' order: a `gate` whose weight alone gives the logits."""
    routers = [getattr(model.get_submodule(name.rpartition(".")[0]), "gate", None) for name, _ in experts_modules(model)]
    for r in routers:
        if r is None or [n for n, _ in r.named_parameters()] != ["weight"]:
            raise NotImplementedError("the balance loss: routers with one weight, as `gate` beside the experts, are expected")
    if not routers:
        raise NotImplementedError("the balance loss of a model without experts modules")
    return routers


def _last_hidden(model, head, input_ids, attention_mask):
    """The hidden states whose product with the head's weight is the model's logits.

    The model runs its own forward, with the logits of the last position alone (all of them where it knows no
    logits_to_keep), and is watched: what it gives the head has
    to be its decoder's last hidden states, and what it returns the head's output itself, or that divided by its
    configuration's logits_scaling (Granite) or times its logit_scale (Cohere). The hidden states then take the scale, in
    their own type: one rounding of theirs where the model's own path rounds every scaled logit. A model that does anything
    else to its logits (a cap, an offset) is refused."""
    decoder = model.get_decoder() if hasattr(model, "get_decoder") else model.model
    states, products = [], []
    hooks = [decoder.register_forward_hook(lambda m, args, out: states.append(out.last_hidden_state)),
             head.register_forward_hook(lambda m, args, out: products.append(
                 (args[0], out, out.clone() if out.is_inference() else out._version)), prepend=True)]
    takes = inspect.signature(model.forward).parameters.values()
    one = {"logits_to_keep": 1} if any(p.name == "logits_to_keep" or p.kind is p.VAR_KEYWORD for p in takes) else {}
    try:
        out = model(input_ids=input_ids, attention_mask=attention_mask, use_cache=False, return_dict=True, **one)
    finally:
        for h in hooks:
            h.remove()
    if len(states) != 1 or len(products) != 1:
        raise NotImplementedError("a model that runs its decoder or its head more than once")
    hidden, (given, product, mark) = states[0], products[0]
    if (given.untyped_storage().data_ptr() != hidden.untyped_storage().data_ptr() or given.dtype != hidden.dtype
            or given.shape[-1] != hidden.shape[-1]):
        raise NotImplementedError("a model that changes its last hidden states before the head")
    logits = out.logits
    if (torch.equal(product, mark) if torch.is_tensor(mark) else product._version == mark):  # not changed in place
        if logits.dtype == product.dtype and logits.data_ptr() == product.data_ptr():
            return hidden
        product = product.to(logits.dtype)
        config = model.config.get_text_config() if hasattr(model.config, "get_text_config") else model.config
        divisor, factor = getattr(config, "logits_scaling", None), getattr(config, "logit_scale", None)
        if divisor is not None and torch.equal(logits, product / divisor):
            return hidden / divisor
        if factor is not None and torch.equal(logits, product * factor):
            return hidden * factor
        if logits.dtype != hidden.dtype and torch.equal(logits, product):  # widened, as older Transformers do
            return hidden
    raise NotImplementedError("a model that changes its logits after the head (a cap, for instance)")


def training_loss(model, input_ids, labels, attention_mask=None, balance: float = 0.0, ignore_index: int = -100):
    """A fine-tuning step's loss of a Transformers causal language model, and the tokens of every expert: (loss, counts).

    The mean cross entropy of predicting labels (B, T) from the hidden states before each (labels are shifted here, as
    Transformers does; `ignore_index` where there is none), from the head's weight without the logits but the last
    position's, which show what the model does to them: a scale is applied, anything else refused. Plus `balance`
    times the routers' balance loss over the tokens that attention_mask (B, T) keeps, on the routers' own choices.
    counts: (layers, experts) int64, or None without balance (nothing is collected then)."""
    model = getattr(model, "_orig_mod", model)  # of a compiled model: its modules are watched
    head = model.get_output_embeddings()
    if getattr(head, "bias", None) is not None:
        raise NotImplementedError("a head with a bias")
    if type(head).forward is not torch.nn.Linear.forward:
        raise NotImplementedError(f"a head that is a {type(head).__name__}: a linear layer is expected")
    seen, hooks = [], []

    def collect(router, args, out):
        # the router gives its probabilities, the weights and the choice; its logits are one small product more
        if (not isinstance(out, tuple) or len(out) != 3 or not all(torch.is_tensor(x) and x.dim() == 2 for x in out)
                or out[0].shape[1] != router.weight.shape[0] or out[2].dtype not in (torch.int64, torch.int32)):
            raise NotImplementedError(f"the balance loss of a {type(router).__name__}: what it gives is not known")
        x = args[0]
        seen.append((torch.nn.functional.linear(x.reshape(-1, x.shape[-1]), router.weight), out[2]))

    if balance:
        if getattr(model, "is_gradient_checkpointing", False):
            raise NotImplementedError("the balance loss with gradient checkpointing: its routers run twice")
        hooks = [r.register_forward_hook(collect) for r in _routers(model)]
    try:
        hidden = _last_hidden(model, head, input_ids, attention_mask)
    finally:
        for h in hooks:
            h.remove()
    targets = torch.nn.functional.pad(labels[:, 1:], (0, 1), value=ignore_index)
    loss = linear_cross_entropy(hidden, head.weight, targets, ignore_index=ignore_index)
    if not balance:
        return loss, None
    if len(seen) != len(hooks):
        raise NotImplementedError("the balance loss of routers that are not called as modules, once each")
    logits, index = zip(*seen)
    mask = None if attention_mask is None else attention_mask.reshape(-1)
    extra, counts = balance_loss(logits, index[0].shape[1], mask=mask, top_k_index=index)
    return loss + balance * extra, counts.view(len(logits), -1)
