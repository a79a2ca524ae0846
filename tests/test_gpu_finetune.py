"""A Transformers MoE model whose step runs the fine-tuning operators (model.install_attention, model.training_loss):
its loss and gradients against the same model on its own path."""

import pytest
import torch

import meepsquared_b200 as mb
from test_model import tiny_qwen3_moe

pytestmark = pytest.mark.gpu
DEV = "cuda"


def build(layers=1):
    model = tiny_qwen3_moe(layers=layers).to(DEV, torch.bfloat16)
    for p in model.parameters():
        p.requires_grad_(False)
    mb.model.install(model, rank=16, alpha=32, generator=torch.Generator().manual_seed(1))
    gen = torch.Generator().manual_seed(2)
    for p in mb.model.lora_parameters(model):
        with torch.no_grad():
            p.copy_((torch.randn(p.shape, generator=gen) * 0.02).to(p))
    for _, a in mb.model.attention_modules(model):
        for norm in (a.q_norm, a.k_norm):
            with torch.no_grad():
                norm.weight.copy_(1 + 0.1 * torch.randn(norm.weight.shape, generator=gen).to(norm.weight))
            norm.weight.requires_grad_()
    return model


def trained(model):
    return [p for p in model.parameters() if p.requires_grad]


def take(model):
    grads = [p.grad.float().clone() for p in trained(model)]
    for p in trained(model):
        p.grad = None
    return grads


def compare(got, want):
    """Two bf16 computations of a whole model that round at different points: each gradient within 3% of its norm and
    10% of its largest element (as the routed layer's model test)."""
    for i, (g, r) in enumerate(zip(got, want)):
        assert (g - r).norm() <= 3e-2 * r.norm(), i
        torch.testing.assert_close(g, r, atol=0.1 * r.abs().max().item(), rtol=0, msg=str(i))


def batch(padded):
    gen = torch.Generator().manual_seed(4)
    ids = torch.randint(0, 512, (3, 70), generator=gen).to(DEV)
    labels = ids.clone()
    labels[:, :20] = -100
    mask = None
    if padded:
        mask = torch.ones_like(ids)
        mask[1, 50:] = 0
        mask[2, 33:] = 0
        labels[mask == 0] = -100
    return ids, labels, mask


@pytest.mark.parametrize("padded", [False, True])
def test_the_loss_matches_the_models_own(padded):
    """Up to the last hidden states both run the same operations, so that every token meets the same experts."""
    model = build()
    ids, labels, mask = batch(padded)
    out = model(input_ids=ids, labels=labels, attention_mask=mask)
    out.loss.backward()
    want_loss, want = out.loss.detach().float(), take(model)
    loss, counts = mb.model.training_loss(model, ids, labels, attention_mask=mask)
    loss.backward()
    assert counts is None and abs(loss.item() - want_loss.item()) <= 1e-2 * want_loss.item()
    compare(take(model), want)


@pytest.mark.parametrize("padded,own_positions", [(False, False), (True, False), (False, True)])
def test_attention_matches_the_models_own(padded, own_positions):
    """Each attention module alone, on the inputs that the model gives it (in the whole model the two roundings send
    near-tied tokens to other experts, and the later layers then see other inputs)."""
    model = build(layers=2)
    ids, _, mask = batch(padded)
    calls = []
    modules = [m for _, m in mb.model.attention_modules(model)]
    hooks = [m.register_forward_hook(lambda m, a, k, o: calls.append(k), with_kwargs=True) for m in modules]
    positions = None
    if own_positions:  # every sequence at positions of its own: one row of angles for every token
        positions = torch.arange(ids.shape[1], device=DEV)[None] + torch.tensor([[0], [17], [400]], device=DEV)
    with torch.no_grad():
        model(input_ids=ids, attention_mask=mask, position_ids=positions, use_cache=False)
    for h in hooks:
        h.remove()
    assert calls[0]["position_embeddings"][0].shape[0] == (3 if own_positions else 1)

    def run(module, kwargs, dy):
        x = kwargs["hidden_states"].detach().requires_grad_()
        out = module(**dict(kwargs, hidden_states=x))[0]
        leaves = [x, module.q_norm.weight, module.k_norm.weight]
        return [out.detach(), *torch.autograd.grad(out, leaves, dy)]

    gen = torch.Generator().manual_seed(6)
    dys = [torch.randn(k["hidden_states"].shape, generator=gen).to(DEV, torch.bfloat16) for k in calls]
    want = [run(m, k, dy) for m, k, dy in zip(modules, calls, dys)]
    assert mb.model.install_attention(model) == 2
    live = slice(None) if mask is None else mask != 0
    for m, k, dy, w in zip(modules, calls, dys, want):
        got = run(m, k, dy)
        compare([got[0][live].float()], [w[0][live].float()])
        compare([g.float() for g in got[1:]], [x.float() for x in w[1:]])


def test_the_balance_loss_of_the_routers():
    """Against its definition on the routers' probabilities as the model's hooks see them."""
    model = build(layers=2)
    for _, layer in enumerate(model.model.layers):
        layer.mlp.gate.weight.requires_grad_()
    mb.model.install_attention(model)
    ids = torch.randint(0, 512, (2, 40), generator=torch.Generator().manual_seed(4)).to(DEV)
    mask = torch.ones_like(ids)
    mask[1, 25:] = 0
    seen = []
    hooks = [layer.mlp.gate.register_forward_hook(lambda m, a, o: seen.append((o[0], o[2]))) for layer in model.model.layers]
    plain, none = mb.model.training_loss(model, ids, ids, attention_mask=mask)
    for h in hooks:
        h.remove()
    live = mask.reshape(-1) != 0
    n = 2 * int(live.sum())
    f = sum(torch.nn.functional.one_hot(i, 8).sum(1)[live].sum(0) for _, i in seen).float() / n
    m = sum(p[live].sum(0) for p, _ in seen) / n
    want = 8 * (f * m).sum()
    want_grads = torch.autograd.grad(want, [layer.mlp.gate.weight for layer in model.model.layers], retain_graph=True)
    loss, counts = mb.model.training_loss(model, ids, ids, attention_mask=mask, balance=0.5)
    assert torch.equal(counts, torch.stack([torch.nn.functional.one_hot(i, 8).sum(1)[live].sum(0) for _, i in seen]))
    extra = loss - plain  # the routers' product runs in bf16 in both
    assert abs(extra.item() - 0.5 * want.item()) <= 1e-2 * want.item()
    got = torch.autograd.grad(loss - plain, [layer.mlp.gate.weight for layer in model.model.layers], retain_graph=True)
    for g, w in zip(got, want_grads):
        # the language-model part cancels between two equal graphs up to its own bf16 rounding
        assert torch.isfinite(g).all() and (g.float() - 0.5 * w.float()).norm() <= 0.1 * w.float().norm()


def test_decoding_behind_a_cache():
    model = build(layers=2).eval()
    ids = torch.randint(0, 512, (2, 9), generator=torch.Generator().manual_seed(4)).to(DEV)

    def run():
        with torch.no_grad():
            first = model(input_ids=ids, use_cache=True)
            nxt = model(input_ids=ids[:, :1], past_key_values=first.past_key_values, use_cache=True)
        return first.logits.float(), nxt.logits.float()

    want = run()
    mb.model.install_attention(model)
    for g, w in zip(run(), want):
        assert (g - w).norm() <= 3e-2 * w.norm()


@pytest.mark.parametrize("scaling", [6.0, 0.25])
def test_a_model_that_scales_its_logits(scaling):
    """GraniteMoe divides its logits: the loss within bf16's rounding of the logits (which the model's own path has), the
    gradients as the other whole-model comparisons."""
    from transformers import GraniteMoeConfig, GraniteMoeForCausalLM

    torch.manual_seed(0)
    model = GraniteMoeForCausalLM(GraniteMoeConfig(
        vocab_size=512, hidden_size=256, intermediate_size=128, num_hidden_layers=1, num_attention_heads=4,
        num_key_value_heads=2, num_local_experts=4, num_experts_per_tok=2, logits_scaling=scaling)).to(DEV, torch.bfloat16)
    for p in model.parameters():
        p.requires_grad_(False)
    model.model.norm.weight.requires_grad_()
    model.model.layers[0].input_layernorm.weight.requires_grad_()
    ids, labels, mask = batch(True)
    out = model(input_ids=ids, labels=labels, attention_mask=mask)
    out.loss.backward()
    want_loss, want = out.loss.detach().float(), take(model)
    loss, _ = mb.model.training_loss(model, ids, labels, attention_mask=mask)
    loss.backward()
    assert abs(loss.item() - want_loss.item()) <= 1e-2 * want_loss.item()
    compare(take(model), want)
