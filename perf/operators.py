"""Cases and plain forms of the operators a fine-tuning step needs around the expert layer.

Three operators, each with the forms a program calls:

* ``linear_cross_entropy``: the language-model loss of hidden states against a large vocabulary, without keeping the
  logits; alone (evaluation), with the gradient of the hidden states (frozen head: LoRA) or of the head as well;
* ``balance_loss``: the router's load-balancing loss and the tokens each expert got, over one layer or many, with
  the gradient of the router logits;
* ``qk_norm_rope``: RMS norm of every query and key head and the rotation by position, in one pass; with its
  gradients (training), or for the new token of every sequence (serving).

``run`` computes the plain form in float32 with elementary torch operations, or (``own``) makes the package's calls.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
IGNORE = -100


# ------------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # evaluation of one short answer: a few tokens' loss, no gradient (latency)
        dict(name="ce_short_loss", op="ce", tokens=37, hidden=2048, vocab=16384, grad="none", ignored=0.0,
             reduction="mean"),
        # per-token losses of a scored batch, its prompts masked out (evaluation, preference and distillation scores)
        dict(name="ce_masked_scores", op="ce", tokens=5000, hidden=2048, vocab=100003, grad="none", ignored=0.6,
             reduction="none"),
        # a fine-tuning step with a frozen head: loss and the hidden states' gradient, prompts masked out
        dict(name="ce_masked_step", op="ce", tokens=4093, hidden=2048, vocab=131072, grad="hidden", ignored=0.5,
             reduction="mean"),
        # the same at the benchmark's batch, every position a target: the largest case
        dict(name="ce_full_step", op="ce", tokens=16384, hidden=2048, vocab=131072, grad="hidden", ignored=0.0,
             reduction="mean"),
        # the head is trained too, with an odd vocabulary
        dict(name="ce_trained_head", op="ce", tokens=4096, hidden=4096, vocab=32003, grad="both", ignored=0.1,
             reduction="sum"),
        # one layer's routers on a small batch (latency), as a per-layer loss is called
        dict(name="balance_one_layer", op="balance", layers=1, tokens=2048, experts=128, top_k=8, dtype="bf16",
             masked=0.0, ids=False, train=True),
        # a whole model's routers at the benchmark's batch, padding masked out
        dict(name="balance_24_layers", op="balance", layers=24, tokens=16384, experts=128, top_k=8, dtype="bf16",
             masked=0.2, ids=False, train=True),
        # few experts, float32 logits, the selection the router already made, an odd token count
        dict(name="balance_8_experts", op="balance", layers=4, tokens=8191, experts=8, top_k=2, dtype="f32",
             masked=0.1, ids=True, train=True),
        # serving: the next token of each of 64 sequences, every one at a position of its own
        dict(name="qk_decode", op="qk", batch=64, length=1, q_heads=32, kv_heads=4, dim=128, rotated=128,
             dtype="bf16", train=False, fused=True, positions=True),
        # serving: one sequence's prompt, odd length
        dict(name="qk_prompt", op="qk", batch=1, length=1111, q_heads=32, kv_heads=4, dim=128, rotated=128,
             dtype="bf16", train=False, fused=True, positions=False),
        # the training step of the benchmark's model: four sequences of 4096
        dict(name="qk_step", op="qk", batch=4, length=4096, q_heads=32, kv_heads=4, dim=128, rotated=128,
             dtype="bf16", train=True, fused=False, positions=False),
        # packed sequences in float32, heads of 64 with half of them rotated, odd length
        dict(name="qk_packed_f32", op="qk", batch=3, length=1777, q_heads=10, kv_heads=5, dim=64, rotated=32,
             dtype="f32", train=True, fused=True, positions=True),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["ce", "ce", "balance", "qk"])
    if op == "ce":
        c = dict(op=op, tokens=_log(rng, 1, 16384), hidden=8 * _log(rng, 8, 512), vocab=_log(rng, 1000, 131072),
                 grad=rng.choice(["none", "hidden", "hidden", "both"]), ignored=rng.choice([0.0, 0.3, 0.7]),
                 reduction=rng.choice(["mean", "sum", "none"]))
        c["hidden"] += 8 if c["hidden"] == 3072 else 0
        most = 4 * 16384 * 2048 * 131072
        while 2 * (1 + _directions(c)) * c["tokens"] * c["hidden"] * c["vocab"] > most:
            c["tokens"] //= 2
        return c
    if op == "balance":
        c = dict(op=op, layers=_log(rng, 1, 24), tokens=_log(rng, 1, 16384), experts=_log(rng, 4, 512),
                 dtype=rng.choice(["bf16", "f32"]), masked=rng.choice([0.0, 0.25]), ids=rng.choice([False, True]),
                 train=rng.choice([False, True, True]))
        c["top_k"] = rng.randint(1, min(8, c["experts"]))
        while c["layers"] * c["tokens"] * c["experts"] > 24 * 16384 * 128 // (2 if c["dtype"] == "f32" else 1):
            c["tokens"] //= 2
        return c
    kv = rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 80, 96, 128, 256])
    c = dict(op=op, batch=rng.choice([1, 2, 5, 64]), length=_log(rng, 1, 16384), q_heads=kv * rng.choice([1, 2, 5, 8]),
             kv_heads=kv, dim=dim, rotated=rng.choice([dim, dim, 32]), dtype=rng.choice(["bf16", "bf16", "f32"]),
             train=rng.choice([False, True]), fused=rng.choice([False, True]), positions=rng.choice([False, True]))
    most = 16384 * 36 * 128 // (2 if c["dtype"] == "f32" else 1)
    while c["length"] > 1 and c["batch"] * c["length"] * (c["q_heads"] + c["kv_heads"]) * dim > most:
        c["length"] //= 2
    return c


def _directions(c):
    return {"none": 0, "hidden": 1, "both": 2}[c["grad"]]


def work(case):
    c = case
    if c["op"] == "ce":
        live = max(1, round(c["tokens"] * (1.0 - c["ignored"])))
        d = _directions(c)
        product = 2 * live * c["hidden"] * c["vocab"]
        nbytes = (live * c["hidden"] * 2 + c["vocab"] * c["hidden"] * 2 + c["tokens"] * 8
                  + (c["tokens"] * 4 if c["reduction"] == "none" else 4))
        nbytes += (c["tokens"] * c["hidden"] * 2 if d >= 1 else 0) + (c["vocab"] * c["hidden"] * 2 if d >= 2 else 0)
        return {"bytes": nbytes, "flops": (1 + d) * product}
    if c["op"] == "balance":
        size = 2 if c["dtype"] == "bf16" else 4
        n = c["layers"] * c["tokens"]
        live = n * (1.0 - c["masked"])
        nbytes = live * c["experts"] * size + (live * c["top_k"] * 8 if c["ids"] else 0) + 8 * c["experts"]
        nbytes += n * c["experts"] * size if c["train"] else 0
        return {"bytes": nbytes, "flops": live * c["experts"] * (10 if c["train"] else 5)}
    size = 2 if c["dtype"] == "bf16" else 4
    n = c["batch"] * c["length"] * (c["q_heads"] + c["kv_heads"]) * c["dim"]
    # training: x in, y out, then dy in, dx out (x is kept from the forward pass, but has to be read again: counted once)
    return {"bytes": n * size * (4 if c["train"] else 2) + c["length"] * c["rotated"] * 4,
            "flops": n * (20 if c["train"] else 7)}


# ------------------------------------------------------------------------------------------------------- the inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    gen = _generator(seed)
    c = case
    if c["op"] == "ce":
        T, H, V = c["tokens"], c["hidden"], c["vocab"]
        weight = torch.empty((V, H), dtype=torch.bfloat16, device="cuda").normal_(0.0, 0.02, generator=gen)
        targets = torch.randint(0, V, (T,), device="cuda", generator=gen)
        hidden = torch.randn((T, H), device="cuda", generator=gen)
        # a model that has learned something: the target's logit stands out, by up to 16 for some tokens
        rows = weight[targets].float()
        pull = 16.0 * torch.rand((T, 1), device="cuda", generator=gen) / rows.square().sum(1, keepdim=True).clamp_min(1e-6)
        hidden = (hidden + pull * rows).to(torch.bfloat16)
        # the ignored positions come in runs (prompts), about `ignored` of all
        if c["ignored"]:
            runs = torch.rand(((T + 63) // 64,), device="cuda", generator=gen) < c["ignored"]
            targets = torch.where(runs.repeat_interleave(64)[:T], IGNORE, targets)
        upstream = (torch.randn((T,), device="cuda", generator=gen) if c["reduction"] == "none"
                    else torch.ones((), device="cuda"))
        hidden.requires_grad_(c["grad"] != "none")
        weight.requires_grad_(c["grad"] == "both")
        return dict(case, hidden_states=hidden, weight=weight, targets=targets, upstream=upstream)
    if c["op"] == "balance":
        T, E, dt = c["tokens"], c["experts"], DTYPES[c["dtype"]]
        # every expert has a tendency of its own beside the tokens' differences
        def layer(_):
            bias = 0.5 * torch.randn((1, E), device="cuda", generator=gen)
            return (torch.randn((T, E), device="cuda", generator=gen) + bias).to(dt).requires_grad_(c["train"])
        logits = list(map(layer, range(c["layers"])))
        ids = None
        if c["ids"]:
            ids = [_largest(x.detach(), c["top_k"]) for x in logits]
        mask = torch.rand((T,), device="cuda", generator=gen) >= c["masked"] if c["masked"] else None
        return dict(case, logits=logits, index=ids, mask=mask, upstream=torch.full((), 0.001, device="cuda"))
    B, L, D, dt = c["batch"], c["length"], c["dim"], DTYPES[c["dtype"]]
    hq, hk = c["q_heads"], c["kv_heads"]
    if c["fused"]:  # slices of one projection of queries, keys and values
        qkv = torch.randn((B, L, (hq + 2 * hk) * D), device="cuda", generator=gen).to(dt)
        q, k = qkv[..., :hq * D].unflatten(-1, (hq, D)), qkv[..., hq * D:(hq + hk) * D].unflatten(-1, (hk, D))
    else:
        q = torch.randn((B, L, hq, D), device="cuda", generator=gen).to(dt)
        k = torch.randn((B, L, hk, D), device="cuda", generator=gen).to(dt)
    q, k = q.detach().requires_grad_(c["train"]), k.detach().requires_grad_(c["train"])
    wq = (1.0 + 0.1 * torch.randn((D,), device="cuda", generator=gen)).to(dt).requires_grad_(c["train"])
    wk = (1.0 + 0.1 * torch.randn((D,), device="cuda", generator=gen)).to(dt).requires_grad_(c["train"])
    rows = 32768 if c["positions"] else L
    half = c["rotated"] // 2
    angle = (torch.arange(rows, dtype=torch.float64)[:, None]
             * 1e6 ** (-torch.arange(half, dtype=torch.float64)[None] / half))
    cos, sin = angle.cos().float().cuda(), angle.sin().float().cuda()
    positions = torch.randint(0, rows, (B, L), device="cuda", generator=gen) if c["positions"] else None
    dq = torch.randn((B, L, hq, D), device="cuda", generator=gen).to(dt) if c["train"] else None
    dk = torch.randn((B, L, hk, D), device="cuda", generator=gen).to(dt) if c["train"] else None
    return dict(case, q=q, k=k, wq=wq, wk=wk, cos=cos, sin=sin, pos=positions, dq=dq, dk=dk)


def _largest(x, k):
    """The k largest of each row, the lower index first where values are equal."""
    return x.float().sort(dim=-1, descending=True, stable=True)[1][..., :k].contiguous()


# ------------------------------------------------------------------------------------------------------- the passes

def run(state):
    if own:
        return {"ce": _own_ce, "balance": _own_balance, "qk": _own_qk}[state["op"]](state)
    with torch.no_grad():
        return {"ce": _plain_ce, "balance": _plain_balance, "qk": _plain_qk}[state["op"]](state)


def _own_ce(s):
    import meepsquared_b200 as mb

    loss = mb.linear_cross_entropy(s["hidden_states"], s["weight"], s["targets"], ignore_index=IGNORE,
                                   reduction=s["reduction"])
    if s["grad"] == "none":
        return {"loss": loss}
    wanted = [s["hidden_states"]] + ([s["weight"]] if s["grad"] == "both" else [])
    grads = torch.autograd.grad(loss, wanted, s["upstream"])
    return {"loss": loss.detach(), "grads": list(grads)}


def _own_balance(s):
    import meepsquared_b200 as mb

    loss, counts = mb.balance_loss(s["logits"], s["top_k"], mask=s["mask"], top_k_index=s["index"])
    if not s["train"]:
        return {"loss": loss, "counts": counts}
    return {"loss": loss.detach(), "counts": counts, "grads": list(torch.autograd.grad(loss, s["logits"], s["upstream"]))}


def _own_qk(s):
    import meepsquared_b200 as mb

    q, k = mb.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], positions=s["pos"], eps=EPS)
    if not s["train"]:
        return {"q": q, "k": k}
    dq, dk, dwq, dwk = torch.autograd.grad([q, k], [s["q"], s["k"], s["wq"], s["wk"]], [s["dq"], s["dk"]])
    return {"q": q.detach(), "k": k.detach(), "grads": [dq, dk, dwq, dwk]}


def _plain_ce(s):
    hidden, weight, targets = s["hidden_states"].float(), s["weight"].float(), s["targets"]
    live = targets != IGNORE
    at = torch.where(live, targets, 0)[:, None]
    p = hidden @ weight.t()
    target_logit = p.gather(1, at)[:, 0]
    top = p.max(1, keepdim=True)[0]
    p.sub_(top).exp_()
    total = p.sum(1, keepdim=True)
    losses = torch.where(live, total.log()[:, 0] + top[:, 0] - target_logit, 0.0)
    count = live.sum().clamp_min(1)
    loss = {"none": losses, "sum": losses.sum(), "mean": losses.sum() / count}[s["reduction"]]
    if s["grad"] == "none":
        return {"loss": loss}
    g = s["upstream"] / count if s["reduction"] == "mean" else s["upstream"]
    g = torch.where(live, g, 0.0)[:, None]
    p.mul_(g / total)
    p.scatter_add_(1, at, -g)
    grads = [(p @ weight).to(torch.bfloat16)]
    if s["grad"] == "both":
        grads.append((p.t() @ hidden).to(torch.bfloat16))
    return {"loss": loss, "grads": grads}


def _plain_balance(s):
    x = torch.stack(s["logits"]).float()
    L, T, E = x.shape
    live = torch.ones(T, dtype=torch.bool, device=x.device) if s["mask"] is None else s["mask"]
    index = _largest(x, s["top_k"]) if s["index"] is None else torch.stack(s["index"])
    chosen = torch.zeros((L, T, E), dtype=torch.int64, device=x.device).scatter_(2, index, 1) * live[:, None]
    counts = chosen.sum(1)
    n = (live.sum() * L).clamp_min(1).float()
    p = (x - x.max(-1, keepdim=True)[0]).exp()
    p = p / p.sum(-1, keepdim=True)
    share = counts.sum(0) / n
    loss = E * (share * (p * live[:, None]).sum((0, 1)) / n).sum()
    said = counts[0] if L == 1 else counts
    if not s["train"]:
        return {"loss": loss, "counts": said}
    dp = s["upstream"] * E / n * share
    dx = p * (dp - (p * dp).sum(-1, keepdim=True)) * live[:, None]
    return {"loss": loss, "counts": said, "grads": list(dx.to(s["logits"][0].dtype))}


def _turn(x, cos, sin):
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _plain_qk(s):
    at = torch.arange(s["length"], device=s["q"].device)[None].expand(s["batch"], -1) if s["pos"] is None else s["pos"]
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    q, dq, dwq = _plain_heads(s["q"], s["wq"], cos, sin, s["dq"])
    k, dk, dwk = _plain_heads(s["k"], s["wk"], cos, sin, s["dk"])
    if not s["train"]:
        return {"q": q, "k": k}
    return {"q": q, "k": k, "grads": [dq, dk, dwq, dwk]}


def _plain_heads(x, w, cos, sin, dy):
    dt = x.dtype
    x, w = x.float(), w.float()
    r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    n = x * r
    y = _turn(n * w, cos, sin).to(dt)
    if dy is None:
        return y, None, None
    u = _turn(dy.float(), cos, -sin)
    dw = (u * n).sum((0, 1, 2))
    u = u * w
    dx = r * (u - n * (u * n).mean(-1, keepdim=True))
    return y, dx.to(dt), dw.to(dt)


# ------------------------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"ce": _exact_ce, "balance": _exact_balance, "qk": _exact_qk}[case["op"]](s)


def _exact_ce(s):
    hidden, weight = s["hidden_states"].detach().double(), s["weight"].detach().double()
    live = (s["targets"] != IGNORE).nonzero()[:, 0]
    losses = torch.zeros(s["tokens"], dtype=torch.float64, device="cuda")
    d_hidden = torch.zeros_like(hidden)
    d_weight = torch.zeros_like(weight) if s["grad"] == "both" else None
    scale = s["upstream"].double().expand(s["tokens"]) / (max(1, live.numel()) if s["reduction"] == "mean" else 1)
    for rows in live.split(2048):
        logits = hidden[rows] @ weight.t()
        want = s["targets"][rows]
        lse = torch.logsumexp(logits, 1)
        each = torch.arange(rows.numel(), device="cuda")
        losses[rows] = lse - logits[each, want]
        if s["grad"] == "none":
            continue
        soft = torch.exp(logits - lse[:, None])
        soft[each, want] -= 1.0
        soft *= scale[rows, None]
        d_hidden[rows] = soft @ weight
        if d_weight is not None:
            d_weight.addmm_(soft.t(), hidden[rows])
    loss = losses if s["reduction"] == "none" else losses.sum() / (max(1, live.numel()) if s["reduction"] == "mean" else 1)
    if s["grad"] == "none":
        return {"loss": loss}
    return {"loss": loss, "grads": [d_hidden] + ([d_weight] if d_weight is not None else [])}


def _exact_balance(s):
    L, T, E = s["layers"], s["tokens"], s["experts"]
    live = torch.arange(T, device="cuda") if s["mask"] is None else s["mask"].nonzero()[:, 0]
    n = max(1, L * live.numel())
    counts = torch.zeros((L, E), dtype=torch.int64, device="cuda")
    mass = torch.zeros(E, dtype=torch.float64, device="cuda")
    for i, x in enumerate(s["logits"]):
        if s["index"] is None:  # every logit and its index as one whole number, no two alike
            bits = x.detach().float().view(torch.int32).long()
            order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * 1024 - torch.arange(E, device="cuda")
            ids = order.topk(s["top_k"], dim=-1)[1]
        else:
            ids = s["index"][i]
        counts[i] = torch.bincount(ids[live].reshape(-1), minlength=E)
        mass += torch.softmax(x.detach()[live].double(), -1).sum(0)
    share = counts.sum(0).double() / n
    loss = E * torch.dot(share, mass / n)
    said = counts[0] if L == 1 else counts
    if not s["train"]:
        return {"loss": loss, "counts": said}
    grads = []
    for x in s["logits"]:
        soft = torch.softmax(x.detach()[live].double(), -1)
        d = torch.zeros((T, E), dtype=torch.float64, device="cuda")
        d[live] = soft * (share[None] - (soft @ share)[:, None]) * (s["upstream"].double() * E / n)
        grads.append(d)
    return {"loss": loss, "counts": said, "grads": grads}


def _exact_qk(s):
    B, L, D = s["batch"], s["length"], s["dim"]
    at = s["pos"].reshape(-1) if s["pos"] is not None else torch.arange(L, device="cuda").repeat(B)
    turn = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
    half = s["cos"].shape[1]

    def heads(x, w):
        v = x.double().reshape(B * L, -1, D)
        v = v / torch.sqrt((v * v).sum(-1, keepdim=True) / D + EPS) * w.double()
        z = torch.complex(v[..., :half], v[..., half:2 * half]) * turn
        return torch.cat([z.real, z.imag, v[..., 2 * half:]], -1).reshape(x.shape)

    if not s["train"]:
        return {"q": heads(s["q"], s["wq"]), "k": heads(s["k"], s["wk"])}
    leaves = [s[n].detach().double().requires_grad_() for n in ("q", "k", "wq", "wk")]
    q, k = heads(leaves[0], leaves[2]), heads(leaves[1], leaves[3])
    grads = torch.autograd.grad([q, k], leaves, [s["dq"].double(), s["dk"].double()])
    return {"q": q.detach(), "k": k.detach(), "grads": list(grads)}
