"""balance_loss against its definition in float64: the loss, the counts (exactly) and the logits' gradient.

Tolerances: a float32 softmax of E logits is off by about (E / 32 + 10) 2^-23 of each probability, below 1e-5 for
E <= 1024, and so is the loss, a sum of them; the gradient is p (f - sum p f), off by 1e-5 of p (|f| + sum p |f|) with f
less its mean, and rounded once to the logits' type."""

import pytest
import torch

import meepsquared_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda"


def choice(x, k):
    """The k largest, the lower index first where equal (float64 holds every float32 exactly)."""
    return torch.sort(x.double(), dim=-1, descending=True, stable=True)[1][..., :k]


def formula(logits, k, mask, ids, upstream):
    E = logits[0].shape[1]
    live = torch.ones(logits[0].shape[0], dtype=torch.bool, device=DEV) if mask is None else mask != 0
    n = max(1, len(logits) * int(live.sum()))
    ids = [choice(x, k) for x in logits] if ids is None else ids
    counts = torch.stack([torch.bincount(i[live].reshape(-1)[(i[live].reshape(-1) >= 0) & (i[live].reshape(-1) < E)],
                                         minlength=E) for i in ids])
    f = counts.sum(0).double() / n
    p = [torch.softmax(x.double(), -1) for x in logits]
    loss = E * (f * sum(q[live].sum(0) for q in p)).sum() / n
    centred = f - f.mean()
    grads, tols = [], []
    for x, q in zip(logits, p):
        q = torch.where(live[:, None], q, 0.0)
        scale = upstream * E / n
        want = scale * q * (centred - (q * centred).sum(1, keepdim=True))
        tol = 1e-5 * abs(scale) * q * (centred.abs() + (q * centred.abs()).sum(1, keepdim=True))
        grads.append(want)
        tols.append(tol + (1.01 * 2.0 ** -8 * want.abs() if x.dtype == torch.bfloat16 else 1e-38) + 1e-40)
    return loss, counts, grads, tols


def check(logits, k, mask=None, ids=None, upstream=0.01):
    loss, counts, grads, tols = formula(logits, k, mask, ids, upstream)
    leaves = [x.detach().requires_grad_() for x in logits]
    one = len(leaves) == 1
    got, said = mb.balance_loss(leaves[0] if one else leaves, k, mask=mask,
                                top_k_index=None if ids is None else (ids[0] if one else ids))
    assert torch.equal(said, counts[0] if one else counts)
    assert got.dtype == torch.float32 and abs(float(got.detach()) - float(loss)) <= 1e-5 * abs(float(loss))
    for x, want, tol in zip(torch.autograd.grad(got, leaves, torch.full((), upstream, device=DEV)), grads, tols):
        assert torch.isfinite(x).all() and bool(((x.double() - want).abs() <= tol).all())
    with torch.no_grad():
        again, counted = mb.balance_loss(leaves, k, mask=mask, top_k_index=ids)
    assert torch.equal(again, got.detach()) and torch.equal(counted, said)


def make(layers, tokens, experts, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn((tokens, experts), generator=gen) + torch.randn((1, experts), generator=gen)).to(DEV, dtype)
            for _ in range(layers)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("experts,k", [(1, 1), (3, 3), (8, 2), (9, 4), (16, 1), (30, 6), (60, 4), (64, 8), (128, 8),
                                       (130, 8), (256, 8), (300, 5), (512, 10), (1000, 33), (1024, 8)])
@pytest.mark.parametrize("layers,tokens", [(1, 1), (1, 515), (3, 77)])
def test_loss_counts_and_gradient(layers, tokens, experts, k, dtype):
    check(make(layers, tokens, experts, dtype), k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_many_layers(dtype):
    check(make(128, 300, 64, dtype), 8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_equal_logits_go_to_the_lower_expert(dtype):
    gen = torch.Generator().manual_seed(1)
    x = torch.randint(-2, 3, (400, 128), generator=gen).to(DEV, dtype)
    x[:, ::3] *= -1.0  # zeros of both signs
    x[5] = 0.0
    check([x], 8)
    check([x[:, :24].contiguous()], 24)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", [torch.bool, torch.int64, torch.float32])
def test_masked_tokens(dtype, kind):
    logits = make(2, 333, 40, dtype)
    mask = (torch.arange(333, device=DEV) % 5 != 2)
    clean = [x.clone() for x in logits]
    logits[0][2] = float("nan")
    logits[1][7] = float("inf")
    logits[1][12] = -float("inf")
    check(clean, 6, mask.to(kind))
    a = mb.balance_loss(clean, 6, mask=mask)
    b = mb.balance_loss(logits, 6, mask=mask)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    leaves = [x.requires_grad_() for x in logits]
    for x in torch.autograd.grad(mb.balance_loss(leaves, 6, mask=mask)[0], leaves):
        assert torch.isfinite(x).all() and not x[~mask].any()


def test_nothing_left_by_the_mask():
    x = make(1, 50, 16, torch.bfloat16)[0].requires_grad_()
    loss, counts = mb.balance_loss(x, 4, mask=torch.zeros(50, dtype=torch.bool, device=DEV))
    assert float(loss.detach()) == 0.0 and not counts.any()
    loss.backward()
    assert not x.grad.any()


def test_no_tokens():
    x = torch.zeros((0, 16), device=DEV, requires_grad=True)
    loss, counts = mb.balance_loss(x, 4)
    loss.backward()
    assert float(loss.detach()) == 0.0 and not counts.any() and x.grad.shape == x.shape


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_experts_ruled_out_by_minus_infinity(dtype):
    logits = make(1, 200, 64, dtype)
    logits[0][:, 10:30] = -float("inf")
    logits[0][:, 40] = torch.finfo(dtype).min
    check(logits, 8)
    check([logits[0][:, 8:34].contiguous()], 8)  # fewer are left than are chosen: the lowest of the ruled-out follow


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("index", [torch.int64, torch.int32])
def test_a_choice_already_made(dtype, index):
    logits = make(2, 257, 24, dtype)
    gen = torch.Generator().manual_seed(2)
    ids = [torch.rand((257, 24), generator=gen).argsort(1)[:, :3].to(DEV) for _ in logits]
    ids[0][4, 1], ids[1][9, 0] = 24, -1  # sentinels: no expert
    check(logits, 3, torch.arange(257, device=DEV) % 3 != 0, [i.to(index) for i in ids])


def test_near_balance_the_gradient_keeps_its_bits():
    """Every expert chosen equally often, one token aside: f is nearly constant and its mean drops out of the
    gradient."""
    x = torch.zeros((8192, 128), device=DEV)
    x.scatter_(1, (torch.arange(8192, device=DEV)[:, None] * 8 + torch.arange(8, device=DEV)) % 128, 1.0)
    x[0] = x[0].roll(1)
    check([x], 8)


def test_the_gradient_is_the_differences_slope():
    """The loss along a direction that changes no choice, in float32: its differences over steps of 2e-3 carry 1e-7
    of the loss over the change, below 1%."""
    x = make(1, 64, 16, torch.float32)[0].requires_grad_()
    loss, counts = mb.balance_loss(x, 4)
    grad, = torch.autograd.grad(loss, x)
    step = 2e-2 * grad / grad.norm() * 64 ** 0.5
    with torch.no_grad():
        up, c0 = mb.balance_loss(x + step, 4, top_k_index=choice(x, 4))
        down, c1 = mb.balance_loss(x - step, 4, top_k_index=choice(x, 4))
    assert torch.equal(c0, counts) and torch.equal(c1, counts)
    along = 2 * float((grad.double() * step.double()).sum())
    assert abs(float(up) - float(down) - along) <= 0.01 * along + 4e-7 * float(loss.detach())


def test_other_strides_streams_and_again():
    x = make(1, 300, 128, torch.bfloat16)[0]
    want = mb.balance_loss(x, 8)
    wide = torch.zeros((300, 200), dtype=torch.bfloat16, device=DEV)
    wide[:, 3:131] = x
    odd = torch.zeros((300 * 128 + 1,), dtype=torch.bfloat16, device=DEV)
    odd[1:] = x.reshape(-1)
    leaf = odd[1:].view(300, 128).detach().requires_grad_()
    base = x.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(mb.balance_loss(leaf, 8)[0], leaf)[0],
                       torch.autograd.grad(mb.balance_loss(base, 8)[0], base)[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = mb.balance_loss(x, 8)
    torch.cuda.synchronize()
    for got in (mb.balance_loss(wide[:, 3:131], 8), mb.balance_loss(x.t().contiguous().t(), 8), other):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_second_derivative_is_refused():
    xs = [x.requires_grad_() for x in make(2, 20, 16, torch.float32)]
    grads = torch.autograd.grad(mb.balance_loss(xs, 2)[0], xs, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable twice"):
        grads[0].sum().backward()


def test_some_layers_gradients_alone():
    xs = make(3, 20, 16, torch.float32)
    want = [x.detach().requires_grad_() for x in xs]
    mb.balance_loss(want, 2)[0].backward()
    some = [x.detach().requires_grad_(i != 1) for i, x in enumerate(xs)]
    mb.balance_loss(some, 2)[0].backward()
    assert some[1].grad is None and all(torch.equal(some[i].grad, want[i].grad) for i in (0, 2))


def test_refusals():
    x = make(1, 10, 16, torch.float32)[0]
    with pytest.raises(ValueError, match="top_k"):
        mb.balance_loss(x, 17)
    with pytest.raises(ValueError, match="top_k"):
        mb.balance_loss(x, 0)
    with pytest.raises(ValueError, match="logits"):
        mb.balance_loss([x, x[:5]], 2)
    with pytest.raises(ValueError, match="logits"):
        mb.balance_loss([], 2)
    with pytest.raises(TypeError, match="float32 or bf16"):
        mb.balance_loss(x.half(), 2)
    with pytest.raises(ValueError, match="mask"):
        mb.balance_loss(x, 2, mask=torch.ones(9, device=DEV))
    with pytest.raises(ValueError, match="top_k_index"):
        mb.balance_loss(x, 2, top_k_index=torch.zeros((10, 3), dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError, match="1024"):
        mb.balance_loss(torch.zeros((4, 1025), device=DEV), 2)
    with pytest.raises(ValueError, match="128"):
        mb.balance_loss([x] * 129, 2)


def test_offsets_past_32_bits():
    """More than 2^31 logits: the counts of all tokens against the choice in pieces, and the last rows' gradient."""
    tokens, experts = 17_000_003, 128
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = torch.empty((tokens, experts), dtype=torch.bfloat16, device=DEV).normal_(generator=gen).requires_grad_()
    loss, counts = mb.balance_loss(x, 4)
    grad, = torch.autograd.grad(loss, x)
    assert int(counts.sum()) == 4 * tokens
    want = torch.zeros(experts, dtype=torch.int64, device=DEV)
    mass = torch.zeros(experts, dtype=torch.float64, device=DEV)
    for rows in x.detach().split(1 << 20):
        key = rows.float().view(torch.int32).long()
        key = torch.where(key < 0, -(key & 0x7FFFFFFF), key) * 1024 - torch.arange(experts, device=DEV)
        want += torch.bincount(key.topk(4, dim=1)[1].reshape(-1), minlength=experts)
        mass += torch.softmax(rows.float(), 1).sum(0, dtype=torch.float64)
    assert torch.equal(counts, want)
    f = want.double() / tokens
    assert abs(float(loss.detach()) - float(experts * (f * mass).sum() / tokens)) <= 1e-5 * float(loss.detach())
    p = torch.softmax(x.detach()[-100:].double(), 1)
    f = f - f.mean()
    dx = experts / tokens * p * (f - (p * f).sum(1, keepdim=True))
    tol = 1e-5 * experts / tokens * p * (f.abs() + (p * f.abs()).sum(1, keepdim=True)) + 1.01 * 2.0 ** -8 * dx.abs()
    assert bool(((grad[-100:].double() - dx).abs() <= tol + 1e-38).all())


def test_recomputed_under_a_checkpoint():
    from torch.utils.checkpoint import checkpoint

    xs = make(2, 50, 16, torch.float32)
    a = [x.detach().requires_grad_() for x in xs]
    mb.balance_loss(a, 2)[0].backward()
    b = [x.detach().requires_grad_() for x in xs]
    checkpoint(lambda *y: mb.balance_loss(y, 2)[0], *b, use_reentrant=False).backward()
    assert all(torch.equal(x.grad, y.grad) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_rows_of_very_large_and_very_low_logits(dtype):
    """A row whose mask of the type's lowest value leaves nothing has equal probabilities; beside a logit of 1e10 or more
    only its equals have any."""
    x = make(1, 90, 24, dtype)[0]
    x[3] = torch.finfo(dtype).min
    x[7] = -1e10
    x[11] = 1e10
    x[12, 5:] = torch.finfo(dtype).min
    x[17] = torch.finfo(dtype).min
    x[17, 9] = torch.finfo(dtype).max
    x[23, ::2] = 3e12
    check([x], 5)
    check([x[:, :8].contiguous()], 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("gap", [10.0, 30.0, 45.0])
@pytest.mark.parametrize("tokens", [1, 700])
def test_unlikely_experts_chosen(tokens, gap, dtype):
    """A choice of experts that have hardly any probability (a given choice need not follow the logits): the loss is a sum
    of the small ones alone."""
    x = make(1, tokens, 16, dtype)[0]
    x[:, 0] += gap
    ids = torch.arange(tokens, device=DEV)[:, None] % 5 * 3 + torch.tensor([[1, 3]], device=DEV)
    check([x], 2, ids=[ids])


@pytest.mark.parametrize("experts,tokens", [(100, 1 << 26), (7, 1 << 27)])
def test_many_tokens_of_equal_probabilities(experts, tokens):
    """Every probability is 1 / E and the loss exactly top_k, whatever the choice: float32 sums of thousands of equal
    summands drift, all in one direction."""
    x = torch.zeros((tokens, experts), dtype=torch.bfloat16, device=DEV)
    loss, counts = mb.balance_loss(x, 3)
    assert counts[:3].tolist() == [tokens] * 3 and not counts[3:].any()
    assert abs(float(loss) - 3.0) <= 1e-5 * 3.0


@pytest.mark.parametrize("which", [0, 1])
def test_forward_mode_derivatives_are_refused(which):
    """An answer without the tangent would read as a derivative of zero."""
    import torch.autograd.forward_ad as forward

    inputs = make(2, 20, 16, torch.float32)

    def call(*x):
        return mb.balance_loss(x, 2)[0]

    with forward.dual_level():
        dual = [forward.make_dual(x, torch.ones_like(x)) if i == which else x for i, x in enumerate(inputs)]
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(*dual)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda x: call(*[x if i == which else y for i, y in enumerate(inputs)]), (inputs[which],),
                       (torch.ones_like(inputs[which]),))
    call(*inputs)  # and nothing is left behind


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_captured_in_a_graph(dtype):
    xs = [x.requires_grad_() for x in make(3, 200, 64, dtype)]
    mask = torch.arange(200, device=DEV) % 7 != 0

    def step():
        loss, counts = mb.balance_loss(xs, 6, mask=mask)
        return loss.detach(), counts, *torch.autograd.grad(loss, xs)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (5, 6):
        with torch.no_grad():
            for x, new in zip(xs, make(3, 200, 64, dtype, seed)):
                x.copy_(new)
        graph.replay()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)
