"""The fine-tuning step's operators without a GPU: the buffers the vocabulary loss plans, and the refusal to run on the
CPU."""

import ctypes

import pytest
import torch

import meepsquared_b200 as mb
from meepsquared_b200 import _lib, build


def plan(tokens, hidden, vocab):
    rows, cols, planes = ctypes.c_int64(), ctypes.c_int64(), ctypes.c_int32()
    _lib.check(_lib.load().meep2b_linear_ce_plan(tokens, hidden, vocab, ctypes.byref(rows), ctypes.byref(cols),
                                                 ctypes.byref(planes)), "meep2b_linear_ce_plan")
    return rows.value, cols.value, planes.value


@pytest.mark.parametrize("tokens", [1, 255, 256, 257, 4096, 16384, 1 << 20])
@pytest.mark.parametrize("vocab", [1, 256, 257, 32003, 131072, 262144])
@pytest.mark.parametrize("hidden", [8, 2048, 8192])
def test_the_plan_of_the_vocabulary_loss(tokens, vocab, hidden):
    rows, cols, planes = plan(tokens, hidden, vocab)
    assert rows % 256 == 0 and tokens <= rows < tokens + 256
    assert cols % 256 == 0 and 256 <= cols < vocab + 256
    assert cols == 256 or rows * cols * 2 <= 1 << 30
    assert 1 <= planes <= 16 and (planes == 1 or planes * rows * hidden * 4 <= 1 << 29)
    pieces = -(-vocab // cols)
    assert pieces * cols - vocab < pieces * 256 + 256  # the pieces are about equal


def test_sizes_beyond_the_entry_point_are_refused():
    with pytest.raises(ValueError):
        plan(1 << 25, 64, 1000)
    with pytest.raises(ValueError):
        plan(16, 0, 1000)


def test_the_autograd_nodes_build_and_load():
    build.build()
    module = _lib.native()
    assert all(callable(getattr(module, f)) for f in ("linear_cross_entropy", "balance_loss", "qk_norm_rope"))


def test_no_cpu_fallback():
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        mb.linear_cross_entropy(x, x, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA"):
        mb.balance_loss(x, 2)
    q = torch.zeros((1, 4, 2, 64))
    with pytest.raises(RuntimeError, match="CUDA"):
        mb.qk_norm_rope(q, q, torch.ones(64), torch.ones(64), torch.ones(4, 32), torch.ones(4, 32))


def test_attention_modules_are_found_and_patched():
    from test_model import tiny_qwen3_moe

    model = tiny_qwen3_moe()
    found = [a for _, a in mb.model.attention_modules(model)]
    assert len(found) == 2
    before = [a.forward for a in found]
    assert mb.model.install_attention(model) == 2
    assert all(a.forward != b for a, b in zip(found, before))
    assert len(mb.model._routers(model)) == 2 and all(hasattr(r, "weight") for r in mb.model._routers(model))
    found[0].sliding_window = 128
    with pytest.raises(NotImplementedError, match="sliding window"):
        mb.model.install_attention(model)


def test_bad_arguments_are_refused_before_anything_runs():
    lib = _lib.load()
    ce = _lib.LinearCE(tokens=4, hidden_size=64, ld_hidden=64, vocab=10, ld_weight=64, rows_pad=256, hidden=4096, weight=4096)
    assert lib.meep2b_linear_ce_forward(None, None) == _lib.ERR_SHAPE
    assert lib.meep2b_linear_ce_forward(ctypes.byref(ce), None) == _lib.ERR_SHAPE  # no loss
    assert lib.meep2b_linear_ce_backward(ctypes.byref(ce), None) == _lib.ERR_SHAPE  # no upstream gradient
    for field, value, status in (("hidden_size", 60, _lib.ERR_ALIGN), ("ld_weight", 56, _lib.ERR_ALIGN),
                                 ("weight", 4098, _lib.ERR_ALIGN), ("rows_pad", 128, _lib.ERR_SHAPE),
                                 ("vocab", 0, _lib.ERR_SHAPE), ("reduction", 3, _lib.ERR_UNSUPPORTED)):
        bad = _lib.LinearCE.from_buffer_copy(ce)
        setattr(bad, field, value)
        assert lib.meep2b_linear_ce_forward(ctypes.byref(bad), None) == status, field
    balance = _lib.Balance(logits=4096, layers=1, experts=8, tokens=4, top_k=2, dtype=_lib.BF16)
    assert lib.meep2b_balance_loss(None, None) == _lib.ERR_SHAPE
    for field, value, status in (("layers", 129, _lib.ERR_SHAPE), ("experts", 1025, _lib.ERR_SHAPE),
                                 ("top_k", 9, _lib.ERR_SHAPE), ("dtype", 7, _lib.ERR_DTYPE)):
        bad = _lib.Balance.from_buffer_copy(balance)
        setattr(bad, field, value)
        assert lib.meep2b_balance_loss(ctypes.byref(bad), None) == status, field
    heads = _lib.HeadNorm(batch=1, length=4, q_heads=2, kv_heads=1, dim=64, half=32, angles=4, dtype=_lib.BF16)
    assert lib.meep2b_head_norm_rotate(None, None) == _lib.ERR_SHAPE
    for field, value, status in (("dim", 72, _lib.ERR_SHAPE), ("half", 36, _lib.ERR_SHAPE), ("half", 40, _lib.ERR_SHAPE),
                                 ("angles", 3, _lib.ERR_SHAPE), ("dtype", 2, _lib.ERR_DTYPE), ("q", 4, _lib.ERR_ALIGN),
                                 ("length", 1 << 33, _lib.ERR_SHAPE)):
        bad = _lib.HeadNorm.from_buffer_copy(heads)
        setattr(bad, field, value)
        assert lib.meep2b_head_norm_rotate(ctypes.byref(bad), None) == status, field


@pytest.mark.parametrize("spoil", [lambda a: setattr(a, "sliding_window", 128),
                                   lambda a: setattr(a.k_norm, "variance_epsilon", 1e-5)], ids=["window", "epsilon"])
def test_a_refused_module_leaves_the_others_as_they_were(spoil):
    from test_model import tiny_qwen3_moe

    model = tiny_qwen3_moe(layers=3)
    found = [a for _, a in mb.model.attention_modules(model)]
    before = [a.forward for a in found]
    spoil(found[-1])
    with pytest.raises(NotImplementedError):
        mb.model.install_attention(model)
    assert [a.forward for a in found] == before


def plain_qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions=None, eps=1e-6):
    """qk_norm_rope in elementary operations, for what can be said of a patched attention without a GPU."""
    at = torch.arange(q.shape[1]).expand(q.shape[:2]) if positions is None else positions
    c, s, n = cos[at][:, :, None], sin[at][:, :, None], cos.shape[1]

    def heads(x, w):
        x = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w
        a, b = x[..., :n], x[..., n:2 * n]
        return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * n:]], -1)

    return heads(q, q_weight), heads(k, k_weight)


@pytest.mark.parametrize("implementation", ["flash_attention_2", "flex_attention", "paged|sdpa"])
def test_attention_that_separates_sequences_without_a_mask_is_refused(implementation):
    """A model for flash attention gets packed sequences without a mask: taken for causal attention, tokens would see other
    sequences."""
    from test_model import tiny_qwen3_moe

    model = tiny_qwen3_moe()
    model.config._attn_implementation = implementation
    with pytest.raises(NotImplementedError, match="attn_implementation"):
        mb.model.install_attention(model)
    model.config._attn_implementation = "sdpa"
    mb.model.install_attention(model)
    model.config._attn_implementation = implementation  # changed afterwards
    attention = next(mb.model.attention_modules(model))[1]
    x, angles = torch.zeros((1, 4, 256)), (torch.ones((1, 4, 64)), torch.zeros((1, 4, 64)))
    with pytest.raises(NotImplementedError, match="attn_implementation"):
        attention(x, position_embeddings=angles, attention_mask=None)


def test_packed_sequences_and_attention_weights(monkeypatch):
    from test_model import tiny_qwen3_moe

    model = tiny_qwen3_moe().eval()
    ids = torch.randint(0, 512, (1, 12), generator=torch.Generator().manual_seed(1))
    positions = torch.tensor([[0, 1, 2, 3, 4, 0, 1, 2, 0, 1, 2, 3]])
    packed = dict(input_ids=ids, position_ids=positions, use_cache=False)
    bounds = dict(cu_seq_lens_q=torch.tensor([0, 5, 8, 12]), cu_seq_lens_k=torch.tensor([0, 5, 8, 12]))
    with torch.no_grad():
        want = model(**packed).logits
    monkeypatch.setattr(mb.model, "qk_norm_rope", plain_qk_norm_rope)
    mb.model.install_attention(model)
    with torch.no_grad():  # the model gives a mask for sequences told by their positions, with the bounds or without
        for more in ({}, bounds):
            torch.testing.assert_close(model(**packed, **more).logits, want, atol=1e-4, rtol=0)
        with pytest.raises(NotImplementedError, match="packed"):
            model(input_ids=ids, use_cache=False, **bounds)
        model.set_attn_implementation("eager")
        torch.testing.assert_close(model(**packed).logits, want, atol=1e-4, rtol=0)
        with pytest.raises(NotImplementedError, match="output_attentions"):
            model(**packed, output_attentions=True)


def tiny(kind, **more):
    """A small Transformers causal language model of one kind, its attention within heads of 32."""
    import transformers

    sizes = dict(vocab_size=128, hidden_size=128, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
                 num_key_value_heads=2, head_dim=32, max_position_embeddings=64, pad_token_id=0)
    torch.manual_seed(0)
    model = getattr(transformers, kind + "ForCausalLM")(getattr(transformers, kind + "Config")(**{**sizes, **more})).eval()
    gen = torch.Generator().manual_seed(5)
    for n, p in model.named_parameters():
        if "_norm." in n:
            p.data += 0.2 * torch.randn(p.shape, generator=gen)
    return model


MOE = dict(moe_intermediate_size=64, num_experts=4, num_experts_per_tok=2)


@pytest.mark.parametrize("kind,more", [("Qwen3", {}), ("Qwen3Moe", MOE), ("Apertus", {}),
                                       ("Glm4Moe", dict(use_qk_norm=True, n_routed_experts=4, num_experts_per_tok=2,
                                                        moe_intermediate_size=64, partial_rotary_factor=0.5))],
                         ids=lambda x: x if isinstance(x, str) else "")
def test_attention_of_these_kinds_is_computed(monkeypatch, kind, more):
    from transformers import StaticCache

    model = tiny(kind, **more)
    before = [p.clone() for p in model.parameters()]
    ids = torch.randint(0, 128, (2, 9), generator=torch.Generator().manual_seed(1))
    mask = torch.ones_like(ids)
    mask[1, :4] = 0

    def run():
        with torch.no_grad():
            first = model(input_ids=ids, use_cache=True)
            static = StaticCache(config=model.config, max_cache_len=16)
            return [first.logits, model(input_ids=ids, attention_mask=mask).logits[:, 4:],
                    model(input_ids=ids[:, :1], past_key_values=first.past_key_values).logits,
                    model(input_ids=ids[:, :5], past_key_values=static).logits,
                    model(input_ids=ids[:, 5:6], past_key_values=static).logits]

    want = run()
    monkeypatch.setattr(mb.model, "qk_norm_rope", plain_qk_norm_rope)
    assert mb.model.install_attention(model) == 2
    assert mb.model.install_attention(model) == 2  # again
    for g, w in zip(run(), want):
        torch.testing.assert_close(g, w, atol=1e-4, rtol=0)
    assert all(torch.equal(p, q) for p, q in zip(model.parameters(), before)) and not model.training


@pytest.mark.parametrize("kind,more,why", [
    ("Olmoe", MOE, "over each head"),  # norms over all heads
    ("Afmoe", dict(MOE, layer_types=["full_attention"] * 2, num_dense_layers=1), "parameters of its own"),  # a gate
    ("Doge", {}, "parameters of its own"),  # a mask it learns
    ("Gemma3", None, "sliding window"),
], ids=lambda x: x if isinstance(x, str) else "")
def test_attention_of_other_kinds_is_refused(kind, more, why):
    if more is None:
        import transformers

        model = transformers.Gemma3ForCausalLM(transformers.Gemma3TextConfig(
            vocab_size=128, hidden_size=128, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
            num_key_value_heads=2, head_dim=32))
    else:
        model = tiny(kind, **more)
    with pytest.raises(NotImplementedError, match=why):
        mb.model.install_attention(model)


@pytest.mark.parametrize("kind", ["order", "gate", "one plus the weight", "no rotation", "pairs", "not causal", "scale"])
def test_attention_that_looks_alike_is_refused(kind):
    """Modules with every attribute of a Qwen3 attention that compute something else."""
    model = tiny("Qwen3")
    attention = [a for _, a in mb.model.attention_modules(model)][1]
    own = attention.forward

    def forward(hidden_states, position_embeddings, attention_mask=None, past_key_values=None, **kwargs):
        cos, sin = position_embeddings
        batch, length = hidden_states.shape[:2]
        q, k, v = (f(hidden_states).view(batch, length, -1, 32).transpose(1, 2)
                   for f in (attention.q_proj, attention.k_proj, attention.v_proj))

        def turn(x):
            half = torch.cat([-x[..., 16:], x[..., :16]], -1)
            if kind == "pairs":
                half = torch.stack([-x[..., 1::2], x[..., ::2]], -1).flatten(-2)
            return x * cos[:, None] + half * sin[:, None]

        norms = attention.q_norm, attention.k_norm
        if kind == "order":
            q, k = (n(turn(x)) for n, x in zip(norms, (q, k)))
        elif kind == "no rotation":
            q, k = (n(x) for n, x in zip(norms, (q, k)))
        elif kind == "one plus the weight":
            q, k = (turn(n(x) / n.weight * (1 + n.weight)) for n, x in zip(norms, (q, k)))
        else:
            q, k = (turn(n(x)) for n, x in zip(norms, (q, k)))
        out = torch.nn.functional.scaled_dot_product_attention(q, k, v, attn_mask=attention_mask, enable_gqa=True,
                                                               scale=0.5 if kind == "scale" else None)
        out = out.transpose(1, 2).reshape(batch, length, -1)
        return attention.o_proj(out.sigmoid() * out if kind == "gate" else out), None

    attention.forward = forward
    if kind == "not causal":
        attention.is_causal = False
    with pytest.raises(NotImplementedError, match=kind if kind == "not causal" else "not a Qwen3"):
        mb.model.install_attention(model)
    assert attention.forward is forward
    attention.forward, attention.is_causal = own, True
    assert mb.model.install_attention(model) == 2


def plain_loss(hidden, weight, targets, ignore_index=-100, reduction="mean"):
    logits = hidden.reshape(-1, hidden.shape[-1]).float() @ weight.float().t()
    return torch.nn.functional.cross_entropy(logits, targets.reshape(-1), ignore_index=ignore_index, reduction=reduction)


def trained_on():
    ids = torch.randint(1, 128, (2, 11), generator=torch.Generator().manual_seed(2))
    labels = ids.clone()
    labels[:, :4] = -100
    mask = torch.ones_like(ids)
    mask[1, 8:] = 0
    labels[mask == 0] = -100
    return ids, labels, mask


@pytest.mark.parametrize("kind,more", [("Qwen3Moe", MOE), ("GraniteMoe", dict(logits_scaling=6.0, num_local_experts=4)),
                                       ("GraniteMoe", dict(logits_scaling=0.25, num_local_experts=4)),
                                       ("Cohere", dict(logit_scale=0.0625)), ("Gemma2", dict(final_logit_softcapping=None)),
                                       ("Llama", dict(tie_word_embeddings=True))],
                         ids=lambda x: x if isinstance(x, str) else "")
def test_the_training_loss_is_the_models_own(monkeypatch, kind, more):
    """Models that scale their logits among them: the same loss and gradients in float32 as from the model's logits."""
    monkeypatch.setattr(mb.model, "linear_cross_entropy", plain_loss)
    model = tiny(kind, **more).train()
    for m in model.modules():
        if isinstance(m, torch.nn.Dropout):
            m.p = 0.0
    ids, labels, mask = trained_on()
    want = model(input_ids=ids, labels=labels, attention_mask=mask).loss
    params = [p for p in model.parameters() if p.requires_grad]
    grads = torch.autograd.grad(want, params, allow_unused=True)
    loss, counts = mb.model.training_loss(model, ids, labels, attention_mask=mask)
    assert counts is None
    torch.testing.assert_close(loss, want, atol=0, rtol=1e-5)
    for got, w in zip(torch.autograd.grad(loss, params, allow_unused=True), grads):
        assert (got is None) == (w is None)
        if w is not None:
            torch.testing.assert_close(got, w, atol=1e-5 * float(w.abs().max()), rtol=1e-3)
    with torch.inference_mode():
        again, _ = mb.model.training_loss(model, ids, labels, attention_mask=mask)
    torch.testing.assert_close(again, loss.detach(), atol=0, rtol=1e-6)


def test_models_that_do_more_to_their_logits_are_refused(monkeypatch):
    monkeypatch.setattr(mb.model, "linear_cross_entropy", plain_loss)
    ids, labels, mask = trained_on()

    def refused(model, match):
        with pytest.raises(NotImplementedError, match=match):
            mb.model.training_loss(model, ids, labels, attention_mask=mask)
        with torch.inference_mode(), pytest.raises(NotImplementedError, match=match):
            mb.model.training_loss(model, ids, labels, attention_mask=mask)

    refused(tiny("Gemma2", final_logit_softcapping=30.0), "after the head")
    model = tiny("Qwen3")
    hook = model.lm_head.register_forward_hook(lambda m, args, out: out + 1.0)
    refused(model, "after the head")
    hook.remove()
    hook = model.lm_head.register_forward_hook(lambda m, args, out: out.mul_(2.0))
    refused(model, "after the head")
    hook.remove()
    hook = model.lm_head.register_forward_pre_hook(lambda m, args: (args[0] * 0.5,))
    refused(model, "before the head")
    hook.remove()
    mb.model.training_loss(model, ids, labels, attention_mask=mask)
    assert not model.lm_head._forward_hooks and not model.model._forward_hooks

    class Adapted(torch.nn.Linear):
        def forward(self, x):
            return super().forward(x) * 2.0

    model.lm_head = Adapted(128, 128, bias=False)
    refused(model, "linear layer")
    model.lm_head = torch.nn.Linear(128, 128)
    refused(model, "bias")


def plain_balance(logits, top_k, mask=None, top_k_index=None):
    chosen = [torch.nn.functional.one_hot(i, x.shape[1]).sum(1) for x, i in zip(logits, top_k_index)]
    live = torch.ones(len(logits[0]), dtype=torch.bool) if mask is None else mask != 0
    n = len(logits) * int(live.sum())
    f = sum(c[live].sum(0) for c in chosen).float() / n
    m = sum(torch.softmax(x[live].float(), 1).sum(0) for x in logits) / n
    counts = torch.stack([c[live].sum(0) for c in chosen])
    return logits[0].shape[1] * (f * m).sum(), counts[0] if len(logits) == 1 else counts


@pytest.mark.parametrize("kind", ["Qwen3Moe", "Mixtral", "Olmoe", "Qwen2Moe"])
def test_the_balance_loss_of_these_routers(monkeypatch, kind):
    monkeypatch.setattr(mb.model, "linear_cross_entropy", plain_loss)
    monkeypatch.setattr(mb.model, "balance_loss", plain_balance)
    model = tiny(kind, **dict(MOE, num_local_experts=4))
    ids, labels, mask = trained_on()
    probabilities = []
    hooks = [r.register_forward_hook(lambda m, a, o: probabilities.append((o[0], o[2]))) for r in mb.model._routers(model)]
    plain, _ = mb.model.training_loss(model, ids, labels, attention_mask=mask)
    for h in hooks:
        h.remove()
    loss, counts = mb.model.training_loss(model, ids, labels, attention_mask=mask, balance=2.0)
    want, counted = plain_balance([p.log() for p, _ in probabilities], 2, mask.reshape(-1), [i for _, i in probabilities])
    torch.testing.assert_close(loss - plain, 2.0 * want, atol=1e-5, rtol=1e-5)
    assert torch.equal(counts, counted) and not any(r._forward_hooks for r in mb.model._routers(model))


@pytest.mark.parametrize("kind,more", [("Glm4Moe", dict(n_routed_experts=4, num_experts_per_tok=2, moe_intermediate_size=64)),
                                       ("Ernie4_5_Moe", dict(moe_num_experts=4, moe_k=2, moe_intermediate_size=64,
                                                             moe_layer_start_index=0)), ("GptOss", MOE), ("Qwen3", {}),
                                       ("DeepseekV2", dict(n_routed_experts=4, num_experts_per_tok=2, n_group=1, topk_group=1,
                                                           moe_intermediate_size=64, first_k_dense_replace=0, head_dim=16,
                                                           qk_rope_head_dim=16, qk_nope_head_dim=16, v_head_dim=16,
                                                           kv_lora_rank=32, q_lora_rank=None, num_key_value_heads=4))],
                         ids=lambda x: x if isinstance(x, str) else "")
def test_the_balance_loss_of_other_routers_is_refused(monkeypatch, kind, more):
    """Corrected, biased or grouped choices, gates that are not called as modules, and models without experts."""
    monkeypatch.setattr(mb.model, "linear_cross_entropy", plain_loss)
    monkeypatch.setattr(mb.model, "balance_loss", plain_balance)
    model = tiny(kind, **more)
    ids, labels, mask = trained_on()
    with pytest.raises(NotImplementedError, match="balance loss"):
        mb.model.training_loss(model, ids, labels, attention_mask=mask, balance=0.1)
    assert not any(m._forward_hooks for m in model.modules())
    mb.model.training_loss(model, ids, labels, attention_mask=mask)


def test_a_call_that_is_not_causal_is_refused(monkeypatch):
    monkeypatch.setattr(mb.model, "qk_norm_rope", plain_qk_norm_rope)
    model = tiny("Qwen3")
    mb.model.install_attention(model)
    attention = next(mb.model.attention_modules(model))[1]
    x, angles = torch.randn((1, 4, 128)), (torch.ones((1, 4, 32)), torch.zeros((1, 4, 32)))
    with pytest.raises(NotImplementedError, match="not causal"):
        attention(x, position_embeddings=angles, attention_mask=None, is_causal=False)
    attention(x, position_embeddings=angles, attention_mask=None, is_causal=True)


def test_nodes_built_for_another_torch_are_rebuilt_and_not_loaded(monkeypatch):
    """The compiled autograd nodes hold torch's class layouts: a file that another torch, ABI or interpreter built is stale,
    whatever its time."""
    build.build()
    assert not build.native_stale()
    tag = build.native_tag()
    assert torch.__version__ in tag
    monkeypatch.setattr(build, "native_tag", lambda: tag.replace(torch.__version__, "9.9.9"))
    assert build.native_stale()
    monkeypatch.setattr(_lib, "_native", None)
    with pytest.raises(RuntimeError, match="was built for torch"):
        _lib.native()


class Packed(torch.nn.Module):
    """A projection whose weight is stored in another form than it computes in, as quantised ones are."""

    def __init__(self, linear):
        super().__init__()
        self.in_features, self.out_features = linear.in_features, linear.out_features
        self.held = [linear]
        self.weight = torch.nn.Parameter(torch.zeros((linear.weight.numel() // 2, 1), dtype=torch.uint8), requires_grad=False)

    def forward(self, x):
        return torch.nn.functional.linear(x.float(), self.held[0].weight).to(x.dtype)


@pytest.mark.parametrize("norms", [torch.float32, torch.bfloat16])
def test_attention_with_quantised_projections_or_wider_norms_is_taken(norms):
    """Packed projections (QLoRA), and norms kept in float32 beside projections in bf16."""
    model = tiny("Qwen3")
    for _, a in mb.model.attention_modules(model):
        for n in ("q_proj", "k_proj", "v_proj", "o_proj"):
            setattr(a, n, Packed(getattr(a, n)))
        a.q_norm.to(norms), a.k_norm.to(norms)
    assert mb.model.install_attention(model) == 2
    model = tiny("Qwen3").to(torch.bfloat16)
    for _, a in mb.model.attention_modules(model):
        a.q_norm.to(norms), a.k_norm.to(norms)
    assert mb.model.install_attention(model) == 2


@pytest.mark.parametrize("form", ["own", "float", "no logits_to_keep", "compiled", "float and capped"])
def test_the_training_loss_of_other_forms_of_models(monkeypatch, form):
    """Models that widen their logits (older Transformers), that know no logits_to_keep, that were compiled; in bf16."""
    import types

    from transformers import Qwen3ForCausalLM
    from transformers.modeling_outputs import CausalLMOutputWithPast

    monkeypatch.setattr(mb.model, "linear_cross_entropy", plain_loss)

    class Widening(Qwen3ForCausalLM):
        def forward(self, logits_to_keep=0, **kwargs):
            out = super().forward(logits_to_keep=logits_to_keep, **kwargs)
            logits = out.logits.float()
            return CausalLMOutputWithPast(logits=20 * torch.tanh(logits / 20) if "capped" in form else logits)

    class Plain(Qwen3ForCausalLM):
        def forward(self, input_ids=None, attention_mask=None, use_cache=None, return_dict=None):
            hidden = self.model(input_ids=input_ids, attention_mask=attention_mask, use_cache=use_cache)[0]
            return types.SimpleNamespace(logits=self.lm_head(hidden))

    model = tiny("Qwen3").to(torch.bfloat16)
    ids, labels, mask = trained_on()
    with torch.no_grad():
        hidden = model.model(input_ids=ids, attention_mask=mask, use_cache=False).last_hidden_state
        want = plain_loss(hidden[:, :-1], model.lm_head.weight, labels[:, 1:])
    if form.startswith("float"):
        model.__class__ = Widening
    elif form == "no logits_to_keep":
        model.__class__ = Plain
    elif form == "compiled":
        model = torch.compile(model, backend="eager")
    if form == "float and capped":
        with pytest.raises(NotImplementedError, match="after the head"):
            mb.model.training_loss(model, ids, labels, attention_mask=mask)
        return
    loss, _ = mb.model.training_loss(model, ids, labels, attention_mask=mask)
    torch.testing.assert_close(loss.detach(), want, atol=0, rtol=1e-6)
