"""qk_norm_rope against its formula in float64, forward and backward.

Tolerances, u = 2^-24: a value of the result is the sum of two products of x, r, w and a cosine or sine, with r off by
a few u (a sum of D squares in a tree, rsqrt): 32 u of the absolute terms; the gradient of x has two such steps and a
mean over D: 64 u of r (|v| + |n| mean |v n|); a weight's gradient sums its rows in runs of at most 2,048 (a group's,
then the CTA's, then over CTAs): (64 + rows up to 2,048) u of the absolute terms. One rounding to the type at the end
(2^-8 in bf16)."""

import pytest
import torch

import meepsquared_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
ULP = {torch.float32: U, torch.bfloat16: 2.0 ** -8}


def turn(x, c, s):
    n = c.shape[-1]
    a, b = x[..., :n], x[..., n:2 * n]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * n:]], -1)


def turn_abs(x, c, s):
    n = c.shape[-1]
    a, b = x[..., :n].abs(), x[..., n:2 * n].abs()
    return torch.cat([a * c.abs() + b * s.abs(), b * c.abs() + a * s.abs(), x[..., 2 * n:].abs()], -1)


def formula(x, w, c, s, eps, dy):
    """y, dx, dw in float64 and their tolerances, for x (B, T, heads, D) and c, s (B, T, 1, n)."""
    kind = x.dtype
    x, w = x.double(), w.double()
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x * r
    y = turn(n * w, c, s)
    tol = 32 * U * turn_abs(n * w, c, s) + 1.01 * ULP[kind] * y.abs() + 1e-38
    if dy is None:
        return (y, tol),
    dy = dy.double()
    u, ua = turn(dy, c, -s), turn_abs(dy, c, s)
    rows = x.numel() // x.shape[-1]
    dw = (u * n).sum((0, 1, 2))
    tol_w = (64 + min(rows, 2048)) * U * (ua * n.abs()).sum((0, 1, 2)) + 1.01 * ULP[kind] * dw.abs() + 1e-38
    v, va = u * w, ua * w.abs()
    dx = r * (v - n * (v * n).mean(-1, keepdim=True))
    tol_x = 64 * U * r * (va + n.abs() * (va * n.abs()).mean(-1, keepdim=True)) + 1.01 * ULP[kind] * dx.abs() + 1e-38
    return (y, tol), (dx, tol_x), (dw, tol_w)


def angles(rows, half, dtype=torch.float32):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(half, dtype=torch.float64) / max(1, half))
    return a.cos().to(DEV, dtype), a.sin().to(DEV, dtype)


def make(b, t, hq, hk, d, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.randn(shape, generator=gen).to(DEV, dtype)

    return rand(b, t, hq, d), rand(b, t, hk, d), 1 + 0.2 * rand(d), 1 + 0.2 * rand(d), rand(b, t, hq, d), rand(b, t, hk, d)


def near(got, want, name):
    value, tol = want
    assert got.shape == value.shape, name
    over = (got.double() - value).abs() - tol
    assert torch.isfinite(got).all() and float(over.max()) <= 0, f"{name}: {float(over.max()):.3g} over"


def check(q, k, wq, wk, dq, dk, cos, sin, positions=None, eps=1e-6):
    at = torch.arange(q.shape[1], device=DEV).expand(q.shape[:2]) if positions is None else positions.long()
    c, s = cos.double()[at][:, :, None], sin.double()[at][:, :, None]
    leaves = [x.detach().requires_grad_() for x in (q, k, wq, wk)]
    out = mb.qk_norm_rope(*leaves, cos, sin, positions=positions, eps=eps)
    grads = torch.autograd.grad(out, leaves, [dq, dk])
    for i, (x, w, dy) in enumerate(((q, wq, dq), (k, wk, dk))):
        y, dx, dw = formula(x, w, c, s, eps, dy)
        near(out[i].detach(), y, f"out {i}")
        near(grads[i], dx, f"dx {i}")
        near(grads[2 + i], dw, f"dw {i}")
        assert out[i].is_contiguous() and out[i].dtype == x.dtype
    with torch.no_grad():
        again = mb.qk_norm_rope(q, k, wq, wk, cos, sin, positions=positions, eps=eps)
    assert torch.equal(again[0], out[0]) and torch.equal(again[1], out[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("dim,half", [(16, 8), (32, 16), (48, 24), (64, 32), (64, 16), (80, 40), (96, 24), (112, 56),
                                      (128, 64), (128, 0), (160, 16), (192, 96), (256, 128), (256, 32)])
def test_every_head_size(dim, half, dtype):
    cos, sin = angles(40, half)
    check(*make(2, 33, 3, 2, dim, dtype), cos, sin)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("b,t,hq,hk", [(1, 1, 1, 1), (64, 1, 32, 4), (1, 1, 40, 8), (5, 7, 1, 1), (1, 1111, 32, 4),
                                       (3, 257, 17, 5), (2, 2048, 16, 2)])
def test_lengths_and_heads(b, t, hq, hk, dtype):
    cos, sin = angles(t, 64)
    check(*make(b, t, hq, hk, 128, dtype), cos, sin)


@pytest.mark.parametrize("index", [torch.int64, torch.int32])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_positions_and_angle_types(kind, index):
    cos, sin = angles(5000, 32, kind)
    gen = torch.Generator().manual_seed(3)
    pos = torch.randint(0, 5000, (4, 19), generator=gen).to(DEV, index)
    check(*make(4, 19, 6, 3, 64, torch.bfloat16), cos, sin, pos)
    wide = torch.cat([cos, cos], 1), torch.cat([sin, sin], 1)  # the halves repeated, as Transformers keeps them
    check(*make(4, 19, 6, 3, 64, torch.float32), wide[0][:, :32], wide[1][:, :32], pos)
    shifted = torch.zeros((5000, 33), dtype=kind, device=DEV)
    shifted[:, 1:] = cos
    check(*make(4, 19, 6, 3, 64, torch.bfloat16), shifted[:, 1:], sin, pos)


def test_positions_without_angles_are_nan():
    cos, sin = angles(10, 16)
    q, k, wq, wk, _, _ = make(1, 4, 2, 1, 64, torch.bfloat16)
    pos = torch.tensor([[0, 10, -1, 9]], device=DEV)
    for out in mb.qk_norm_rope(q, k, wq, wk, cos, sin, positions=pos):
        assert torch.isnan(out[0, 1:3, :, :32]).all()
        assert torch.isfinite(out[0, 1:3, :, 32:]).all() and torch.isfinite(out[0, [0, 3]]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_slices_transposes_and_offsets(dtype):
    q, k, wq, wk, dq, dk = make(2, 21, 4, 2, 64, dtype)
    cos, sin = angles(21, 32)
    want = mb.qk_norm_rope(q, k, wq, wk, cos, sin)
    fused = torch.zeros((2, 21, 8, 64), dtype=dtype, device=DEV)
    fused[:, :, :4], fused[:, :, 4:6] = q, k
    check(fused[:, :, :4], fused[:, :, 4:6], wq, wk, dq, dk, cos, sin)
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k)]
    check(*heads_first, wq, wk, dq.transpose(1, 2).contiguous().transpose(1, 2), dk, cos, sin)
    odd = torch.zeros(q.numel() + 1, dtype=dtype, device=DEV)
    odd[1:] = q.reshape(-1)
    odd_w = torch.zeros(65, dtype=dtype, device=DEV)
    odd_w[1:] = wq
    inner = torch.zeros((2, 21, 4, 128), dtype=dtype, device=DEV)[..., ::2]
    inner.copy_(q)
    for a, w in ((odd[1:].view(q.shape), odd_w[1:]), (inner, wq)):
        got = mb.qk_norm_rope(a, k, w, wk, cos, sin)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check(q, k, wq, wk, dq[:, :, :1].expand_as(dq), dk, cos, sin)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_small_large_and_zero_heads(dtype):
    q, k, wq, wk, dq, dk = make(1, 9, 3, 2, 128, dtype)
    cos, sin = angles(9, 64)
    q[0, 0] *= 1e-4
    q[0, 1] *= 1e4
    q[0, 2] = 0.0
    check(q, k, wq, wk, dq, dk, cos, sin, eps=1e-5)


def test_an_infinite_head_is_its_own():
    q, k, wq, wk, _, _ = make(1, 9, 3, 2, 128, torch.bfloat16)
    cos, sin = angles(9, 64)
    q[0, 4, 1, 0] = float("inf")
    out = mb.qk_norm_rope(q, k, wq, wk, cos, sin)
    bad = torch.isnan(out[0]).any(-1)
    assert bad[0, 4, 1] and int(bad.sum()) == 1 and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("needed", [(0,), (1,), (2,), (3,), (0, 1)])
def test_some_gradients_alone(needed):
    parts = make(1, 40, 4, 2, 64, torch.bfloat16)
    cos, sin = angles(40, 32)
    every = [x.detach().requires_grad_() for x in parts[:4]]
    want = torch.autograd.grad(mb.qk_norm_rope(*every, cos, sin), every, list(parts[4:]))
    some = [x.detach().requires_grad_(i in needed) for i, x in enumerate(parts[:4])]
    got = torch.autograd.grad(mb.qk_norm_rope(*some, cos, sin), [some[i] for i in needed], list(parts[4:]))
    assert all(torch.equal(g, want[i]) for g, i in zip(got, needed))


def test_one_output_used():
    q, k, wq, wk, dq, _ = make(1, 40, 4, 2, 64, torch.bfloat16)
    cos, sin = angles(40, 32)
    leaves = [x.detach().requires_grad_() for x in (q, k, wq, wk)]
    out = mb.qk_norm_rope(*leaves, cos, sin)[0]
    grads = torch.autograd.grad(out, leaves, dq)
    assert not grads[1].any() and not grads[3].any() and grads[0].any() and grads[2].any()


def test_float32_weights_of_bf16_heads():
    q, k, wq, wk, dq, dk = make(1, 40, 4, 2, 64, torch.bfloat16)
    cos, sin = angles(40, 32)
    want = mb.qk_norm_rope(q, k, wq, wk, cos, sin)
    w = wq.float().requires_grad_()
    got = mb.qk_norm_rope(q, k, w, wk.float(), cos, sin)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got[0].float().sum().backward()
    assert w.grad.dtype == torch.float32 and w.grad.any()


def test_the_gradient_is_the_differences_slope():
    """In float32 with steps of 1e-2 of a norm-1 direction per head: the differences' third order is below 1e-3."""
    q, k, wq, wk, dq, dk = make(1, 8, 2, 1, 64, torch.float32)
    cos, sin = angles(8, 32)
    leaves = [x.detach().requires_grad_() for x in (q, k, wq, wk)]

    def f(*a):
        out = mb.qk_norm_rope(*a, cos, sin)
        return (out[0].double() * dq).sum() + (out[1].double() * dk).sum()

    grads = torch.autograd.grad(f(*leaves), leaves)
    for i, g in enumerate(grads):
        step = 1e-2 * g / g.norm()
        with torch.no_grad():
            ends = [f(*[x + sign * step if j == i else x for j, x in enumerate(leaves)]) for sign in (1, -1)]
        along = 2e-2 * float(g.norm())
        assert abs(float(ends[0] - ends[1]) - along) <= 2e-3 * along


def test_again_on_another_stream_and_empty():
    parts = make(2, 300, 8, 2, 128, torch.bfloat16)
    cos, sin = angles(300, 64)
    first = None
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            leaves = [x.detach().requires_grad_() for x in parts[:4]]
            out = mb.qk_norm_rope(*leaves, cos, sin)
            got = [*out, *torch.autograd.grad(out, leaves, list(parts[4:]))]
        torch.cuda.synchronize()
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))
    empty = [x[:0].detach().requires_grad_() for x in parts[:2]] + [x.detach().requires_grad_() for x in parts[2:4]]
    out = mb.qk_norm_rope(*empty, cos, sin)
    grads = torch.autograd.grad(out, empty, [x[:0] for x in parts[4:]])
    assert out[0].shape[0] == 0 and not grads[2].any() and not grads[3].any()


def test_a_second_derivative_is_refused():
    q, k, wq, wk, dq, dk = make(1, 8, 2, 1, 64, torch.float32)
    cos, sin = angles(8, 32)
    q.requires_grad_()
    grad, = torch.autograd.grad(mb.qk_norm_rope(q, k, wq, wk, cos, sin), q, [dq, dk], create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable twice"):
        grad.sum().backward()


def test_an_input_changed_in_place_is_noticed():
    q, k, wq, wk, dq, dk = make(1, 8, 2, 1, 64, torch.float32)
    cos, sin = angles(8, 32)
    leaf = q.requires_grad_()
    x = leaf * 1.0
    out = mb.qk_norm_rope(x, k, wq, wk, cos, sin)
    x.mul_(2.0)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(out, leaf, [dq, dk])


def test_refusals():
    q, k, wq, wk, _, _ = make(1, 4, 2, 1, 64, torch.bfloat16)
    cos, sin = angles(4, 32)
    cases = [(ValueError, (q[0], k, wq, wk, cos, sin)), (ValueError, (q, k[:, :3], wq, wk, cos, sin)),
             (ValueError, (q[..., :56], k[..., :56], wq[:56], wk[:56], cos, sin)),
             (ValueError, (q, k, wq[:32], wk, cos, sin)), (ValueError, (q, k, wq, wk, cos[:3], sin[:3])),
             (ValueError, (q, k, wq, wk, cos[:, :12], sin[:, :12])),
             (ValueError, (q, k, wq, wk, torch.cat([cos, cos], 1), torch.cat([sin, sin], 1))),
             (TypeError, (q.half(), k.half(), wq, wk, cos, sin)), (TypeError, (q, k.float(), wq, wk, cos, sin)),
             (TypeError, (q, k, wq, wk, cos.half(), sin.half())), (ValueError, (q, k, wq, wk, cos.cpu(), sin.cpu()))]
    for error, args in cases:
        with pytest.raises(error):
            mb.qk_norm_rope(*args)
    with pytest.raises(ValueError, match="positions"):
        mb.qk_norm_rope(q, k, wq, wk, cos, sin, positions=torch.zeros(4, dtype=torch.int64, device=DEV))
    with pytest.raises(TypeError, match="positions"):
        mb.qk_norm_rope(q, k, wq, wk, cos, sin, positions=torch.zeros((1, 4), device=DEV))


def test_offsets_past_32_bits():
    """More than 2^31 values of queries, in a slice of a fused projection: the last tokens against the formula."""
    tokens, d = 530_001, 128
    gen = torch.Generator(device=DEV).manual_seed(1)
    fused = torch.empty((1, tokens, 34, d), dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
    q, k = fused[:, :, :33].requires_grad_(), fused[:, :, 33:].detach()
    wq, wk = (1 + 0.1 * torch.randn(d, device=DEV, generator=gen)).bfloat16(), torch.ones(d, device=DEV).bfloat16()
    cos, sin = angles(1000, 64)
    pos = (torch.arange(tokens, device=DEV) % 1000)[None]
    out = mb.qk_norm_rope(q, k, wq, wk, cos, sin, positions=pos)
    dy = torch.empty_like(out[0]).normal_(generator=gen)
    grad, = torch.autograd.grad(out[0], q, dy)
    for at in (slice(0, 10), slice(tokens - 10, tokens)):
        c, s = cos.double()[pos[:, at]][:, :, None], sin.double()[pos[:, at]][:, :, None]
        y, dx, _ = formula(q.detach()[:, at], wq, c, s, 1e-6, dy[:, at])
        near(out[0].detach()[:, at], y, "out")
        near(grad[:, at], dx, "dx")


def test_recomputed_under_a_checkpoint():
    from torch.utils.checkpoint import checkpoint

    parts = make(1, 40, 4, 2, 64, torch.bfloat16)
    cos, sin = angles(40, 32)
    a = [x.detach().requires_grad_() for x in parts[:4]]
    want = torch.autograd.grad(mb.qk_norm_rope(*a, cos, sin), a, list(parts[4:]))
    b = [x.detach().requires_grad_() for x in parts[:4]]
    out = checkpoint(lambda *y: mb.qk_norm_rope(*y, cos, sin), *b, use_reentrant=False)
    got = torch.autograd.grad(out, b, list(parts[4:]))
    assert all(torch.equal(x, y) for x, y in zip(want, got))


@pytest.mark.parametrize("kinds", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                                   (torch.bfloat16, torch.float16), (torch.float16, torch.float32)],
                         ids=["f32-f32", "f32-bf16", "bf16-f16", "f16-f32"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("dim,half", [(16, 8), (64, 16), (80, 40), (128, 64), (256, 128)])
def test_weights_of_their_own_type(dim, half, dtype, kinds):
    """Norm weights that the heads' type cannot hold: used as they are, and each gradient rounded to its weight's type
    alone (float16 has 11 significant bits, normal from 2^-14)."""
    bits = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
    q, k, _, _, dq, dk = make(3, 37, 5, 2, dim, dtype)
    gen = torch.Generator().manual_seed(9)
    ws = [(1 + 0.2 * torch.randn((dim,), generator=gen)).to(DEV, kind) for kind in kinds]
    assert dtype == torch.float32 or any(bool((w.to(dtype) != w).any()) for w in ws)
    cos, sin = angles(37, half)
    at = torch.arange(37, device=DEV).expand(3, 37)
    c, s = cos.double()[at][:, :, None], sin.double()[at][:, :, None]
    leaves = [x.detach().requires_grad_() for x in (q, k, *ws)]
    out = mb.qk_norm_rope(*leaves, cos, sin)
    grads = torch.autograd.grad(out, leaves, [dq, dk])
    for i, (x, w, dy) in enumerate(((q, ws[0], dq), (k, ws[1], dk))):
        y, dx, (dw, tol) = formula(x, w, c, s, 1e-6, dy)
        near(out[i].detach(), y, f"out {i}")
        near(grads[i], dx, f"dx {i}")
        tol = tol + 1.01 * (bits[w.dtype] - ULP[dtype]) * dw.abs() + (2.0 ** -24 if w.dtype == torch.float16 else 0.0)
        near(grads[2 + i], (dw, tol), f"dw {i}")
        assert out[i].dtype == dtype and grads[2 + i].dtype == w.dtype
    with torch.no_grad():
        again = mb.qk_norm_rope(q, k, *ws, cos, sin)
    assert torch.equal(again[0], out[0]) and torch.equal(again[1], out[1])


@pytest.mark.parametrize("which", range(6))
def test_forward_mode_derivatives_are_refused(which):
    """An answer without the tangent would read as a derivative of zero."""
    import torch.autograd.forward_ad as forward

    q, k, wq, wk, _, _ = make(1, 6, 2, 1, 64, torch.bfloat16)
    inputs = (q, k, wq, wk, *angles(6, 32))

    def call(*x):
        return mb.qk_norm_rope(*x)[0]

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
    q, k, wq, wk, dq, dk = make(2, 30, 4, 2, 64, dtype)
    leaves = [x.detach().requires_grad_() for x in (q, k, wq, wk)]
    cos, sin = angles(30, 32)

    def step():
        out = mb.qk_norm_rope(*leaves, cos, sin)
        return *(x.detach() for x in out), *torch.autograd.grad(out, leaves, [dq, dk])

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
            for x, new in zip(leaves, make(2, 30, 4, 2, 64, dtype, seed)):
                x.copy_(new)
        graph.replay()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)
