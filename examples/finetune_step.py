#!/usr/bin/env python
"""A LoRA fine-tuning step of a mixture-of-experts language model on one B200, with everything this package has for it:
the routed layer on every experts module, norms and rotation of the query and key heads in one pass, the loss without
the logits, the routers' balance loss and the tokens of every expert.

    python examples/finetune_step.py [--layers 4] [--tokens 16384] [--sequence 4096] [--vocab 131072] [--steps 5]

Random weights of a Qwen3-MoE-shaped model (hidden 2048, 128 experts of 768, 32 query and 4 key heads of 128) and random
token ids whose first quarter of each sequence is a prompt (no targets). The model's own step, with the routed layer
alone, is timed beside it. Prints one line for each: loss, milliseconds a step, tokens a second, peak memory."""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

import meepsquared_b200 as mb  # noqa: E402


def build(a):
    from transformers import Qwen3MoeConfig, Qwen3MoeForCausalLM

    cfg = Qwen3MoeConfig(vocab_size=a.vocab, hidden_size=2048, intermediate_size=8192, moe_intermediate_size=768,
                         num_hidden_layers=a.layers, num_attention_heads=32, num_key_value_heads=4, head_dim=128,
                         num_experts=128, num_experts_per_tok=8, decoder_sparse_step=1, mlp_only_layers=[],
                         norm_topk_prob=True, max_position_embeddings=a.sequence)
    torch.manual_seed(0)
    with torch.device("cuda"):
        model = Qwen3MoeForCausalLM(cfg).to(torch.bfloat16)
    for p in model.parameters():
        p.requires_grad_(False)
    mb.model.install(model, rank=16, alpha=32, generator=torch.Generator().manual_seed(0))
    return model


def timed(step, steps):
    for _ in range(2):
        loss = step()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(steps):
        loss = step()
    stop.record()
    torch.cuda.synchronize()
    return float(loss), start.elapsed_time(stop) / steps, torch.cuda.max_memory_allocated() / 2 ** 30


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=16384)
    ap.add_argument("--sequence", type=int, default=4096)
    ap.add_argument("--vocab", type=int, default=131072)
    ap.add_argument("--steps", type=int, default=5)
    a = ap.parse_args()
    model = build(a)
    params = mb.model.lora_parameters(model)
    optimizer = torch.optim.AdamW(params, lr=1e-4)
    batch = max(1, a.tokens // a.sequence)
    ids = torch.randint(0, a.vocab, (batch, a.sequence), generator=torch.Generator().manual_seed(1)).cuda()
    labels = ids.clone()
    labels[:, :a.sequence // 4] = -100
    counts = None

    def own():
        loss = model(input_ids=ids, labels=labels).loss
        loss.backward()
        optimizer.step()
        optimizer.zero_grad(set_to_none=True)
        return loss.detach()

    def operators():
        nonlocal counts
        loss, counts = mb.model.training_loss(model, ids, labels, balance=0.001)
        loss.backward()
        optimizer.step()
        optimizer.zero_grad(set_to_none=True)
        return loss.detach()

    def say(name, result):
        loss, ms, gib = result
        print(f"{name:28s} loss {loss:8.4f}  {ms:8.2f} ms a step  {batch * a.sequence / ms * 1e3:10.0f} tokens/s  "
              f"peak {gib:6.1f} GiB", flush=True)

    say("the model's own loss", timed(own, a.steps))
    mb.model.install_attention(model)
    say("with the operators", timed(operators, a.steps))
    spread = counts.double()
    print("tokens of an expert, by layer: " + "  ".join(
        f"{int(c.min())}..{int(c.max())} (mean {c.mean():.0f})" for c in spread))


if __name__ == "__main__":
    main()
