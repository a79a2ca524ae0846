"""Norms of the query and key heads with the rotation by position in the same pass, and their gradients: what stands
between the attention's projections and the attention itself in models that norm their heads (Transformers'
``Qwen3MoeAttention``: q_norm, k_norm, apply_rotary_pos_emb)."""

import ctypes

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


def _heads(t):
    """(B, T, heads, dim) that 16-byte loads can address: itself, or a copy."""
    vec = 16 // t.element_size()
    s = t.stride()
    if s[3] == 1 and not (s[0] % vec or s[1] % vec or s[2] % vec) and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _vector(w, dtype):
    w = w.detach().to(dtype).contiguous()
    return w if w.data_ptr() % 16 == 0 else w.clone()


def _struct(q, k, q_weight, k_weight, cos, sin, positions, eps):
    b, t, hq, d = q.shape
    return _lib.HeadNorm(q=q.data_ptr(), k=k.data_ptr(), batch=b, length=t, q_heads=hq, kv_heads=k.shape[2], dim=d,
                         half=cos.shape[1], q_stride=q.stride()[:3], k_stride=k.stride()[:3], dtype=_DTYPES[q.dtype],
                         angle_dtype=_DTYPES[cos.dtype], q_weight=q_weight.data_ptr(), k_weight=k_weight.data_ptr(),
                         cos=cos.data_ptr(), sin=sin.data_ptr(), ld_cos=cos.stride(0), ld_sin=sin.stride(0),
                         angles=cos.shape[0], positions=None if positions is None else positions.data_ptr(), eps=eps)


def _forward(q, k, q_weight, k_weight, cos, sin, positions, eps):
    q, k = _heads(q), _heads(k)
    wq, wk = _vector(q_weight, q.dtype), _vector(k_weight, q.dtype)
    q_out, k_out = torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype,
                                                                                     device=q.device)
    a = _struct(q, k, wq, wk, cos, sin, positions, eps)
    a.q_out, a.k_out = q_out.data_ptr(), k_out.data_ptr()
    _lib.check(_lib.load().meep2b_head_norm_rotate(ctypes.byref(a), _lib.stream_of(q)), "meep2b_head_norm_rotate")
    return q_out, k_out


class _QKNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.eps = eps
        return _forward(q.detach(), k.detach(), q_weight, k_weight, cos, sin, positions, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        q, k, dq_out, dk_out = _heads(q.detach()), _heads(k.detach()), _heads(dq_out), _heads(dk_out)
        lib = _lib.load()
        wq, wk = _vector(q_weight, q.dtype), _vector(k_weight, q.dtype)
        dq, dk = torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype,
                                                                                  device=q.device)
        a = _struct(q, k, wq, wk, cos, sin, positions, ctx.eps)
        a.q_out, a.k_out, a.dq_out, a.dk_out = dq.data_ptr(), dk.data_ptr(), dq_out.data_ptr(), dk_out.data_ptr()
        a.dq_out_stride, a.dk_out_stride = dq_out.stride()[:3], dk_out.stride()[:3]
        dwq = dwk = None
        if ctx.needs_input_grad[2] or ctx.needs_input_grad[3]:
            dwq, dwk = torch.empty_like(wq), torch.empty_like(wk)
            partial = torch.empty(lib.meep2b_head_norm_partials() * q.shape[3], dtype=torch.float32, device=q.device)
            a.dq_weight, a.dk_weight, a.partial = dwq.data_ptr(), dwk.data_ptr(), partial.data_ptr()
        _lib.check(lib.meep2b_head_norm_rotate_backward(ctypes.byref(a), _lib.stream_of(q)),
                   "meep2b_head_norm_rotate_backward")
        need = ctx.needs_input_grad
        return (dq if need[0] else None, dk if need[1] else None, dwq.to(q_weight.dtype) if need[2] else None,
                dwk.to(k_weight.dtype) if need[3] else None, None, None, None, None)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor,
                 sin: torch.Tensor, positions=None, eps: float = 1e-6):
    """Every head of q (B, T, q_heads, D) and k (B, T, kv_heads, D) normed and turned by its position: (q', k').

    y = R(pos) (x / sqrt(mean(x^2) + eps) * weight), float32 inside and one rounding at the end. bf16 or float32 (both
    alike), any strides (slices of a fused projection are read in place where they start on 16 bytes); D a multiple of
    16 up to 256. q_weight, k_weight (D). cos, sin (P, n), float32 or bf16: row p holds the angles of position p; the
    first 2n dimensions turn in pairs (i, i + n), the others stay (n a multiple of 8, 2n <= D). positions (B, T)
    integers, or None: 0 .. T - 1 in every sequence (P >= T). A position outside the angles makes its turned values
    NaN. The results are contiguous (B, T, heads, D). Differentiable in q, k and the weights (once)."""
    if not q.is_cuda:
        raise RuntimeError("qk_norm_rope runs on a CUDA GPU")
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"queries {tuple(q.shape)} and keys {tuple(k.shape)}: (B, T, heads, D) expected")
    d = q.shape[3]
    if d % 16 or not 16 <= d <= 256 or not q.shape[2] or not k.shape[2]:
        raise ValueError(f"{q.shape[2]} and {k.shape[2]} heads of {d}: heads of a multiple of 16 up to 256 expected")
    if q.dtype not in _DTYPES or k.dtype != q.dtype:
        raise TypeError(f"queries in {q.dtype} and keys in {k.dtype}: float32 or bf16 expected, both alike")
    if tuple(q_weight.shape) != (d,) or tuple(k_weight.shape) != (d,):
        raise ValueError(f"norm weights {tuple(q_weight.shape)} and {tuple(k_weight.shape)}: ({d},) expected")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] % 8 or 2 * cos.shape[1] > d:
        raise ValueError(f"cos {tuple(cos.shape)} and sin {tuple(sin.shape)}: (positions, n) expected, n a multiple of "
                         f"8 up to {d // 2}")
    if cos.dtype not in _DTYPES or sin.dtype != cos.dtype:
        raise TypeError(f"cos in {cos.dtype} and sin in {sin.dtype}: float32 or bf16 expected, both alike")
    if any(t.device != q.device for t in (k, q_weight, k_weight, cos, sin)):
        raise ValueError("queries, keys, weights and angles are on different devices")
    cos, sin = (x if x.stride(1) == 1 else x.contiguous() for x in (cos.detach(), sin.detach()))
    if positions is None:
        if cos.shape[0] < q.shape[1]:
            raise ValueError(f"angles of {cos.shape[0]} positions for sequences of {q.shape[1]}")
    else:
        if positions.shape != q.shape[:2] or positions.device != q.device:
            raise ValueError(f"positions {tuple(positions.shape)}: {tuple(q.shape[:2])} on the queries' device expected")
        if positions.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"positions in {positions.dtype}: int64 or int32 expected")
        positions = positions.to(torch.int64).contiguous()
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _QKNormRope.apply(q, k, q_weight, k_weight, cos, sin, positions, eps)
    return _forward(q.detach(), k.detach(), q_weight, k_weight, cos, sin, positions, eps)
