"""linear_cross_entropy against softmax cross entropy in float64: losses, the hidden states' gradient and the head's.

Tolerances, with d = (H / 16 + 16) 2^-23 max_tv sum_i |h_ti W_vi|, what a float32 sum of H products (in tensor-core
steps of 16, each rounded or cut) can be off, for a logit:
  loss   2 d for the logits that enter it, and 2^-20 of itself for its logarithm and its sum over the vocabulary;
  dh     the probabilities are rounded to bf16 (2^-8 of each, of which the sum over the vocabulary keeps at most
         2^-8 sum_v p_v |W_v|) and carry their logits' error (2 d); one bf16 rounding at the end;
  dW     the same with the sum over the tokens.
What float32 cannot hold is zero: probabilities below 2^-126, so that dh and dW may miss FLOOR."""

import pytest
import torch

import meepsquared_b200 as mb
from meepsquared_b200 import _lib, _loss

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_ULP = 1.1 * 2.0 ** -8  # of a bf16 rounding, and a tenth for the float32 arithmetic around it

FLOOR = 1e-35  # 2^-126 times a vocabulary's weights


def inputs(tokens, hidden, vocab, seed=0, scale=1.0, ignored=0.0):
    gen = torch.Generator().manual_seed(seed)
    h = (scale * torch.randn((tokens, hidden), generator=gen)).to(DEV, torch.bfloat16)
    w = (torch.randn((vocab, hidden), generator=gen) * hidden ** -0.5).to(DEV, torch.bfloat16)
    t = torch.randint(0, vocab, (tokens,), generator=gen).to(DEV)
    if ignored:
        t[(torch.rand((tokens,), generator=gen) < ignored).to(DEV)] = -100
    return h, w, t


def formula(h, w, t, upstream):
    """Losses, dh, dW in float64 for per-token upstream gradients, and the tolerances of each."""
    h, w, live = h.double(), w.double(), t != -100
    z = h[live] @ w.t()
    y = t[live]
    at = torch.arange(y.numel(), device=h.device)
    lse = torch.logsumexp(z, 1)
    losses = torch.zeros(t.numel(), dtype=torch.float64, device=h.device)
    losses[live] = lse - z[at, y]
    p = torch.exp(z - lse[:, None])
    g = upstream.double()[live, None]
    dz = p.clone()
    dz[at, y] -= 1.0
    dz *= g
    dh = torch.zeros_like(h)
    dh[live] = dz @ w
    dw = dz.t() @ h[live]
    d = (h.shape[1] / 16 + 16) * 2.0 ** -23 * float((h[live].abs() @ w.abs().t()).max()) if y.numel() else 0.0
    each = HALF_ULP + 2 * d
    tol_h = torch.zeros_like(h)
    mass = p * g.abs()
    mass[at, y] = dz[at, y].abs()
    tol_h[live] = each * (mass @ w.abs())
    tol_h += HALF_ULP * dh.abs() + FLOOR
    tol_w = each * (mass.t() @ h[live].abs()) + HALF_ULP * dw.abs() + FLOOR
    return losses, dh, dw, 2 * d + 2.0 ** -20 * losses.abs(), tol_h, tol_w


def within(got, want, tol, name):
    got = got.double()
    assert got.shape == want.shape, name
    over = (got - want).abs() - tol
    assert torch.isfinite(got).all() and float(over.detach().max()) <= 0, \
        f"{name}: {float(over.detach().max()):.3g} over, {int((over > 0).sum())} of {over.numel()}"


def check(h, w, t, reduction, head, seed=3):
    n = t.numel()
    up = torch.randn((n,), generator=torch.Generator().manual_seed(seed)).to(DEV) if reduction == "none" else None
    live = int((t != -100).sum())
    per = up if up is not None else torch.full((n,), 1.0 / max(1, live) if reduction == "mean" else 1.0, device=DEV)
    losses, dh, dw, tol, tol_h, tol_w = formula(h, w, t, per)
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_(head)
    loss = mb.linear_cross_entropy(h, w, t, reduction=reduction)
    if reduction == "none":
        within(loss, losses, tol, "losses")
        loss.backward(up)
    else:
        share = max(1, live) if reduction == "mean" else 1
        assert abs(float(loss.detach()) - float(losses.sum()) / share) <= float(tol.sum()) / share + 1e-7 * abs(float(loss.detach()))
        loss.backward()
    within(h.grad, dh, tol_h, "dh")
    if head:
        within(w.grad, dw, tol_w, "dw")
    else:
        assert w.grad is None
    with torch.no_grad():
        again = mb.linear_cross_entropy(h, w, t, reduction=reduction)
    assert torch.equal(again, loss.detach())
    assert _lib.device_error(0) == 0


@pytest.mark.parametrize("head", [False, True], ids=["frozen", "trained"])
@pytest.mark.parametrize("tokens,hidden,vocab", [(1, 8, 1), (1, 64, 7), (2, 72, 256), (37, 200, 257), (255, 64, 1000),
                                                 (257, 128, 513), (300, 512, 5003), (700, 264, 2048),
                                                 (70, 2048, 300), (70, 2056, 300), (300, 4104, 1000),
                                                 (5, 8200, 700), (128, 72, 600), (129, 72, 600), (384, 72, 600),
                                                 (385, 2056, 600), (640, 72, 900)])
def test_losses_and_gradients(tokens, hidden, vocab, head):
    h, w, t = inputs(tokens, hidden, vocab)
    check(h, w, t, "none", head)


@pytest.mark.parametrize("head", [False, True], ids=["frozen", "trained"])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("ignored", [0.3, 0.97, 1.1], ids=["some", "most", "all"])
def test_ignored_tokens(reduction, ignored, head):
    h, w, t = inputs(500, 136, 777, ignored=ignored)
    check(h, w, t, reduction, head)


@pytest.mark.parametrize("head", [False, True], ids=["frozen", "trained"])
def test_what_ignored_tokens_hold_does_not_matter(head):
    h, w, t = inputs(300, 64, 600, ignored=0.5)
    clean = [x.clone() for x in (h, w, t)]
    h[t == -100] = float("nan")
    h[int((t == -100).nonzero()[0])] = float("inf")
    outs = []
    for a, b in ((clean[0], clean[1]), (h, w)):
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_(head)
        loss = mb.linear_cross_entropy(a, b, t)
        loss.backward()
        outs.append((loss.detach(), a.grad, b.grad))
    for x, y in zip(*outs):
        assert x is None or torch.equal(x, y)


@pytest.mark.parametrize("head", [False, True], ids=["frozen", "trained"])
@pytest.mark.parametrize("planes", [1, 3, 16])
@pytest.mark.parametrize("piece_cols", [256, 768])
def test_pieces_and_planes(monkeypatch, piece_cols, planes, head):
    monkeypatch.setattr(_loss, "PLAN", (piece_cols, planes))
    h, w, t = inputs(600, 192, 2000, ignored=0.2)
    check(h, w, t, "none", head)


@pytest.mark.parametrize("tokens", [100, 350, 700])
@pytest.mark.parametrize("hidden", [64, 2104])
@pytest.mark.parametrize("pieces", [False, True], ids=["whole", "pieces"])
def test_targets_far_below_the_largest_logit(monkeypatch, pieces, hidden, tokens):
    """Logits hundreds above the target's: beyond the window of the target's own reference, in some rows of some
    tiles (the others keep theirs), and far below it."""
    if pieces:
        monkeypatch.setattr(_loss, "PLAN", (512, 2))
    h, w, t = inputs(tokens, hidden, 1500)
    far = torch.arange(tokens, device=DEV) % 97 == 5
    h[far] *= 200.0   # logits of +-600 or so
    h[tokens * 6 // 7:] *= 30.0   # around the window's edge
    check(h, w, t, "none", False)
    check(h, w, t, "none", True)


def test_a_target_far_above_the_others():
    h, w, t = inputs(64, 64, 300)
    h = (w[t].float() * 300.0).to(torch.bfloat16)
    check(h, w, t, "none", False)


@pytest.mark.parametrize("head", [False, True], ids=["frozen", "trained"])
def test_a_target_outside_the_vocabulary_is_nan_alone(head):
    h, w, t = inputs(40, 64, 100)
    t[3], t[17] = 100, -5
    h, w = h.requires_grad_(), w.requires_grad_(head)
    loss = mb.linear_cross_entropy(h, w, t, reduction="none")
    bad = torch.zeros(40, dtype=torch.bool, device=DEV)
    bad[[3, 17]] = True
    assert torch.equal(torch.isnan(loss), bad)
    loss.sum().backward()
    assert torch.equal(torch.isnan(h.grad).all(1), bad) and torch.equal(torch.isnan(h.grad).any(1), bad)


def test_infinite_hidden_states_make_their_own_token_nan():
    h, w, t = inputs(300, 64, 900)
    h[7, 3] = float("inf")
    h.requires_grad_()
    loss = mb.linear_cross_entropy(h, w, t, reduction="none")
    assert torch.isnan(loss).nonzero().flatten().tolist() == [7]
    loss.sum().backward()
    assert torch.isnan(h.grad).any(1).nonzero().flatten().tolist() == [7]


def test_strides_offsets_and_shapes():
    h, w, t = inputs(6 * 35, 64, 500, ignored=0.1)
    want = mb.linear_cross_entropy(h, w, t, reduction="none")
    wide = torch.zeros((210, 96), dtype=torch.bfloat16, device=DEV)
    wide[:, 16:80] = h
    head = torch.zeros((500, 72), dtype=torch.bfloat16, device=DEV)
    head[:, 8:] = w
    odd = torch.zeros((210 * 64 + 1,), dtype=torch.bfloat16, device=DEV)
    odd[1:] = h.reshape(-1)
    for a, b in ((wide[:, 16:80], head[:, 8:]), (odd[1:].view(210, 64), w), (h.t().contiguous().t(), w.t().contiguous().t())):
        assert torch.equal(mb.linear_cross_entropy(a, b, t, reduction="none"), want)
    shaped = mb.linear_cross_entropy(h.view(6, 35, 64), w, t.view(6, 35).int(), reduction="none")
    assert torch.equal(shaped, want.view(6, 35))
    x = wide[:, 16:80].detach().view(6, 35, 64).requires_grad_()
    mb.linear_cross_entropy(x, w, t.view(6, 35), reduction="sum").backward()
    y = h.detach().requires_grad_()
    mb.linear_cross_entropy(y, w, t, reduction="sum").backward()
    assert torch.equal(x.grad.reshape(210, 64), y.grad)


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_no_tokens(reduction):
    h = torch.zeros((0, 64), dtype=torch.bfloat16, device=DEV, requires_grad=True)
    w = torch.ones((10, 64), dtype=torch.bfloat16, device=DEV, requires_grad=True)
    loss = mb.linear_cross_entropy(h, w, torch.zeros((0,), dtype=torch.int64, device=DEV), reduction=reduction)
    assert loss.dtype == torch.float32 and tuple(loss.shape) == ((0,) if reduction == "none" else ())
    loss.sum().backward()
    assert h.grad.shape == h.shape and not w.grad.any()


@pytest.mark.parametrize("head", [False, True], ids=["frozen", "trained"])
def test_the_gradient_is_the_differences_slope(head):
    """(f(h + e d) - f(h - e d)) / 2e along a direction, every point exact in bf16. The third-order term of a log-sum
    along steps of e |logit change| ~ 0.05 is below 0.1%, the gradient's bf16 roundings 2^-8 of its terms."""
    gen = torch.Generator().manual_seed(5)
    h = (torch.randint(-64, 64, (32, 64), generator=gen) / 64.0).to(DEV, torch.bfloat16)
    w = (torch.randint(-32, 32, (200, 64), generator=gen) / 64.0).to(DEV, torch.bfloat16)
    t = torch.randint(0, 200, (32,), generator=gen).to(DEV)
    h.requires_grad_(), w.requires_grad_(head)
    mb.linear_cross_entropy(h, w, t, reduction="sum").backward()
    x = w if head else h
    sign = torch.sign(x.grad.float())
    e = 2.0 ** -7
    step = (sign * e).to(torch.bfloat16)
    with torch.no_grad():
        up, down = x + step, x - step
        assert torch.equal(up.float(), x.float() + sign * e) and torch.equal(down.float(), x.float() - sign * e)
        f = [mb.linear_cross_entropy(*((h, v) if head else (v, w)), t, reduction="none").double().sum() for v in (up, down)]
    slope = float(f[0] - f[1]) / (2 * e)
    along = float((x.grad.double() * sign).sum())
    assert abs(slope - along) <= 0.01 * abs(along)


def test_again_and_on_another_stream():
    h, w, t = inputs(900, 128, 3001, ignored=0.2)
    first = None
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), torch.cuda.current_stream(), side):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            a, b = h.detach().requires_grad_(), w.detach().requires_grad_()
            loss = mb.linear_cross_entropy(a, b, t)
            loss.backward(retain_graph=True)
            kept = a.grad.clone(), b.grad.clone()
            a.grad = b.grad = None
            loss.backward()
            got = loss.detach(), a.grad, b.grad
        torch.cuda.synchronize()
        assert torch.equal(kept[0], got[1]) and torch.equal(kept[1], got[2])
        if first is None:
            first = got
        assert all(torch.equal(x, y) for x, y in zip(first, got))


@pytest.mark.parametrize("head", [False, True], ids=["frozen", "trained"])
def test_a_second_derivative_is_refused(head):
    h, w, t = inputs(20, 64, 70)
    h, w = h.requires_grad_(), w.requires_grad_(head)
    grad, = torch.autograd.grad(mb.linear_cross_entropy(h, w, t), h, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable twice"):
        grad.float().sum().backward()
    loss = mb.linear_cross_entropy(h, w, t)
    loss.backward()
    with pytest.raises(RuntimeError, match="second time"):
        loss.backward()


def test_one_gradient_without_the_other():
    h, w, t = inputs(300, 64, 700)
    both = [h.detach().requires_grad_(), w.detach().requires_grad_()]
    mb.linear_cross_entropy(*both, t).backward()
    alone = w.detach().requires_grad_()
    mb.linear_cross_entropy(h, alone, t).backward()
    assert torch.equal(alone.grad, both[1].grad)
    loss = mb.linear_cross_entropy(*both, t)
    assert torch.equal(torch.autograd.grad(loss, both[0], retain_graph=True)[0], both[0].grad)
    assert torch.equal(torch.autograd.grad(loss, both[1])[0], both[1].grad)


def test_captured_in_a_graph():
    h, w, t = inputs(300, 64, 700, ignored=0.2)
    h.requires_grad_()

    def step():
        loss = mb.linear_cross_entropy(h, w, t)
        return loss.detach(), torch.autograd.grad(loss, h)[0]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals():
    h, w, t = inputs(8, 64, 20)
    with pytest.raises(ValueError, match="targets"):
        mb.linear_cross_entropy(h, w, t[:7])
    with pytest.raises(ValueError, match="head"):
        mb.linear_cross_entropy(h, w[:, :56], t)
    with pytest.raises(ValueError, match="reduction"):
        mb.linear_cross_entropy(h, w, t, reduction="max")
    with pytest.raises(ValueError, match="multiple of 8"):
        mb.linear_cross_entropy(h[:, :60], w[:, :60], t)
    with pytest.raises(TypeError, match="bf16"):
        mb.linear_cross_entropy(h.float(), w, t)
    with pytest.raises(TypeError, match="targets"):
        mb.linear_cross_entropy(h, w, t.float())
    with pytest.raises(ValueError, match="devices"):
        mb.linear_cross_entropy(h, w.cpu(), t)


@pytest.mark.parametrize("long", ["rows", "head"])
def test_offsets_past_32_bits(long):
    """More than 2^31 values of hidden states (an odd number of tokens, two in three ignored) or of the head: losses and
    gradients of the first and the last rows against the formula on those rows alone."""
    tokens, vocab, hidden = (1100001, 300, 2048) if long == "rows" else (40, 1100001, 2048)
    gen = torch.Generator(device=DEV).manual_seed(1)
    h = torch.empty((tokens, hidden), dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
    w = torch.empty((vocab, hidden), dtype=torch.bfloat16, device=DEV).normal_(0.0, hidden ** -0.5, generator=gen)
    t = torch.randint(0, vocab, (tokens,), device=DEV, generator=gen)
    t[:2], t[-2:] = 0, vocab - 1
    if long == "rows":
        t[1000:-1000][torch.arange(tokens - 2000, device=DEV) % 3 != 0] = -100
    up = torch.ones((tokens,), device=DEV)
    h.requires_grad_()
    loss = mb.linear_cross_entropy(h, w, t, reduction="none")
    loss.backward(up)
    ends = torch.cat([torch.arange(20, device=DEV), torch.arange(tokens - 20, tokens, device=DEV)])
    part = h.detach()[ends].double()
    z = torch.cat([part @ w[i:i + 65536].double().t() for i in range(0, vocab, 65536)], 1)
    lse = torch.logsumexp(z, 1)
    at = torch.arange(40, device=DEV)
    d = (hidden / 16 + 16) * 2.0 ** -23 * float((part[:2].abs() @ w[:20000].double().abs().t()).max()) * 2
    want = lse - z[at, t[ends]]
    assert float((loss.detach()[ends].double() - want).abs().max()) <= 2 * d + 2.0 ** -20 * float(want.max())
    p = torch.exp(z - lse[:, None])
    p[at, t[ends]] -= 1.0
    dh = sum(p[:, i:i + 65536] @ w[i:i + 65536].double() for i in range(0, vocab, 65536))
    assert float((h.grad[ends].double() - dh).norm()) <= 2.0 ** -8 * float(dh.norm())
    assert not h.grad[t == -100].any() if long == "rows" else True
    assert torch.isfinite(loss).all() and _lib.device_error(0) == 0


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_under_a_checkpoint(reentrant):
    from torch.utils.checkpoint import checkpoint

    h, w, t = inputs(200, 64, 500, ignored=0.2)
    for head in (False, True):
        a, b = h.detach().requires_grad_(), w.detach().requires_grad_(head)
        mb.linear_cross_entropy(a, b, t).backward()
        c, d = h.detach().requires_grad_(), w.detach().requires_grad_(head)
        checkpoint(lambda x, y: mb.linear_cross_entropy(x, y, t), c, d, use_reentrant=reentrant).backward()
        assert torch.equal(a.grad, c.grad) and (not head or torch.equal(b.grad, d.grad))


def test_saved_on_the_host_in_between():
    h, w, t = inputs(200, 64, 500, ignored=0.2)
    a, b, c, d = (x.detach().requires_grad_() for x in (h, w, h, w))
    mb.linear_cross_entropy(a, b, t).backward()
    with torch.autograd.graph.save_on_cpu():
        loss = mb.linear_cross_entropy(c, d, t)
    loss.backward()
    assert torch.equal(a.grad, c.grad) and torch.equal(b.grad, d.grad)


def test_two_streams_at_once():
    cases = [inputs(700, 256, 4001, seed=i, ignored=0.2) for i in range(2)]

    def step(case):
        a, b = case[0].detach().requires_grad_(), case[1].detach().requires_grad_()
        loss = mb.linear_cross_entropy(a, b, case[2])
        loss.backward()
        c = case[0].detach().requires_grad_()
        mb.linear_cross_entropy(c, case[1], case[2]).backward()
        return loss.detach(), a.grad, b.grad, c.grad

    want = [step(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for stream, case in zip(streams, cases):
            with torch.cuda.stream(stream):
                got.append(step(case))
    torch.cuda.synchronize()
    for i, result in enumerate(got):
        assert all(torch.equal(x, y) for x, y in zip(result, want[i % 2]))
    assert _lib.device_error(0) == 0


def test_a_small_upstream_gradient_on_far_targets():
    """Logits near, but within, the window above the target (about 2^90), times an upstream gradient of 1e-15 or so: the
    row's scale times the gradient alone would be below float32's normal range, the hidden states' gradient is not."""
    gen = torch.Generator().manual_seed(11)
    vocab, hidden = 600, 64
    w = (torch.randn((vocab, hidden), generator=gen) * 0.02).to(DEV, torch.bfloat16)
    w[:, 0] = 0.0
    w[-1, 0] = 1.0  # its logit is the first component of the hidden state
    h = torch.randn((40, hidden), generator=gen).to(DEV, torch.bfloat16)
    h[:, 0] = torch.linspace(58.0, 64.0, 40)
    t = torch.randint(0, vocab - 1, (40,), generator=gen).to(DEV)
    for g in (1e-12, 1e-15, 1e-17, 1e-20):
        up = torch.full((40,), g, device=DEV)
        losses, dh, _, tol, tol_h, _ = formula(h, w, t, up)
        leaf = h.detach().requires_grad_()
        loss = mb.linear_cross_entropy(leaf, w, t, reduction="none")
        within(loss, losses, tol, "losses")
        loss.backward(up)
        within(leaf.grad, dh, tol_h, f"dh at {g}")


@pytest.mark.parametrize("which", [0, 1])
def test_forward_mode_derivatives_are_refused(which):
    """An answer without the tangent would read as a derivative of zero."""
    import torch.autograd.forward_ad as forward

    h, w, t = inputs(20, 64, 100)
    given = (h, w)

    def call(*x):
        return mb.linear_cross_entropy(*x, t)

    with forward.dual_level():
        dual = [forward.make_dual(x, torch.ones_like(x)) if i == which else x for i, x in enumerate(given)]
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(*dual)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda x: call(*[x if i == which else y for i, y in enumerate(given)]), (given[which],),
                       (torch.ones_like(given[which]),))
    call(*given)  # and nothing is left behind


def test_the_first_calls_of_a_process_from_several_threads():
    """Every kernel is set up at its first launch, here by threads that come at once (in a process of its own)."""
    import os
    import subprocess
    import sys

    code = """
import threading, torch
import meepsquared_b200 as mb
gen = torch.Generator().manual_seed(0)
h, w = (torch.randn(s, generator=gen).to("cuda", torch.bfloat16) for s in ((300, 72), (600, 72)))
t = torch.randint(0, 600, (300,), generator=gen).cuda()
start, results = threading.Barrier(6), [None] * 6
def one(i):
    a, b = h.detach().requires_grad_(), w.detach().requires_grad_(i % 2 == 1)
    with torch.cuda.stream(torch.cuda.Stream()):
        start.wait()
        loss = mb.linear_cross_entropy(a, b, t)
        loss.backward()
        torch.cuda.current_stream().synchronize()
    results[i] = loss.detach(), a.grad
torch.cuda.synchronize()
threads = [threading.Thread(target=one, args=(i,)) for i in range(6)]
[x.start() for x in threads], [x.join() for x in threads]
for i in range(2, 6):
    assert torch.equal(results[i][0], results[i % 2][0]) and torch.equal(results[i][1], results[i % 2][1])
print("alike")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(mb.__file__)))  # of the package
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=240)
    assert done.returncode == 0 and "alike" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("hidden", [2048, 4096])
def test_the_mean_loss_is_not_cut_off(hidden):
    """A tensor core cuts every step's sum off toward zero, which shrinks every logit alike: 1.1e-6 of the mean loss over
    the 256 steps of 4,096 products, half of it over the 128 steps that are summed at a time. Over 4,000 tokens what is
    not systematic averages out; 7e-7 lies between the two."""
    gen = torch.Generator(device=DEV).manual_seed(21)
    tokens, vocab = 4000, 32003
    w = torch.empty((vocab, hidden), dtype=torch.bfloat16, device=DEV).normal_(0.0, 0.02, generator=gen)
    t = torch.randint(0, vocab, (tokens,), device=DEV, generator=gen)
    h = torch.randn((tokens, hidden), device=DEV, generator=gen)
    rows = w[t].float()  # the target's logit stands out by up to 16
    h += 16.0 * torch.rand((tokens, 1), device=DEV, generator=gen) / rows.square().sum(1, keepdim=True) * rows
    h = h.to(torch.bfloat16)
    want = 0.0
    for a, b in zip(h.split(1000), t.split(1000)):
        z = a.double() @ w.double().t()
        want += float((torch.logsumexp(z, 1) - z.gather(1, b[:, None])[:, 0]).sum())
    got = float(mb.linear_cross_entropy(h, w, t).double())
    assert abs(got * tokens - want) <= 7e-7 * want


@pytest.mark.parametrize("tokens,hidden,vocab", [(16384, 512, 600), (300, 2048, 600), (70000, 2048, 300)])
def test_what_a_frozen_heads_graph_holds(tokens, hidden, vocab):
    """Between forward and backward: the gradient's planes, 512 MB or one of tokens (up to a multiple of 256) x hidden in
    float32 where that is more, and 40 bytes or so a token."""
    h = torch.zeros((tokens, hidden), dtype=torch.bfloat16, device=DEV).requires_grad_()
    w = torch.zeros((vocab, hidden), dtype=torch.bfloat16, device=DEV)
    t = torch.zeros((tokens,), dtype=torch.int64, device=DEV)
    before = torch.cuda.memory_allocated()
    loss = mb.linear_cross_entropy(h, w, t)
    held = torch.cuda.memory_allocated() - before
    assert held <= max(1 << 29, (tokens + 255) // 256 * 256 * hidden * 4) + 64 * tokens + (1 << 16)
    loss.backward()
    del loss
    assert torch.cuda.memory_allocated() - before <= tokens * hidden * 2 + (1 << 16)
