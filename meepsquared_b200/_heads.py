"""Norms of the query and key heads with the rotation by position in the same pass, and their gradients: what stands
between the attention's projections and the attention itself in models that norm their heads (Transformers'
``Qwen3MoeAttention``: q_norm, k_norm, apply_rotary_pos_emb)."""

import torch

from . import _lib

_DTYPES = (torch.float32, torch.bfloat16)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor,
                 sin: torch.Tensor, positions=None, eps: float = 1e-6):
    """Every head of q (B, T, q_heads, D) and k (B, T, kv_heads, D) normed and turned by its position: (q', k').

    y = R(pos) (x / sqrt(mean(x^2) + eps) * weight), float32 inside and one rounding at the end. bf16 or float32 (both
    alike), any strides (slices of a fused projection are read in place where they start on 16 bytes); D a multiple of
    16 up to 256. q_weight, k_weight (D): both of the heads' type, or read as float32; a weight's gradient is rounded
    once, to the weight's type. cos, sin (P, n), float32 or bf16: row p holds the angles of position p; the first 2n
    dimensions turn in pairs (i, i + n), the others stay (n a multiple of 8, 2n <= D). positions (B, T) integers, or
    None: 0 .. T - 1 in every sequence (P >= T). A position outside the angles makes its turned values NaN. The results
    are contiguous (B, T, heads, D). Differentiable in q, k and the weights (once)."""
    if not q.is_cuda:
        raise RuntimeError("qk_norm_rope runs on a CUDA GPU")
    qs, ks, cs = q.shape, k.shape, cos.shape
    if len(qs) != 4 or len(ks) != 4 or qs[:2] != ks[:2] or qs[3] != ks[3]:
        raise ValueError(f"queries {tuple(qs)} and keys {tuple(ks)}: (B, T, heads, D) expected")
    d = qs[3]
    if d % 16 or not 16 <= d <= 256 or not qs[2] or not ks[2]:
        raise ValueError(f"{qs[2]} and {ks[2]} heads of {d}: heads of a multiple of 16 up to 256 expected")
    if q.dtype not in _DTYPES or k.dtype != q.dtype:
        raise TypeError(f"queries in {q.dtype} and keys in {k.dtype}: float32 or bf16 expected, both alike")
    if q_weight.shape != (d,) or k_weight.shape != (d,):
        raise ValueError(f"norm weights {tuple(q_weight.shape)} and {tuple(k_weight.shape)}: ({d},) expected")
    if len(cs) != 2 or cs != sin.shape or cs[1] % 8 or 2 * cs[1] > d:
        raise ValueError(f"cos {tuple(cs)} and sin {tuple(sin.shape)}: (positions, n) expected, n a multiple of 8 up to "
                         f"{d // 2}")
    if cos.dtype not in _DTYPES or sin.dtype != cos.dtype:
        raise TypeError(f"cos in {cos.dtype} and sin in {sin.dtype}: float32 or bf16 expected, both alike")
    dev = q.device
    if k.device != dev or q_weight.device != dev or k_weight.device != dev or cos.device != dev or sin.device != dev:
        raise ValueError("queries, keys, weights and angles are on different devices")
    if cos.stride(1) != 1 or sin.stride(1) != 1:
        cos, sin = cos.contiguous(), sin.contiguous()
    if positions is None:
        if cs[0] < qs[1]:
            raise ValueError(f"angles of {cs[0]} positions for sequences of {qs[1]}")
    else:
        if positions.shape != qs[:2] or positions.device != dev:
            raise ValueError(f"positions {tuple(positions.shape)}: {tuple(qs[:2])} on the queries' device expected")
        if positions.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"positions in {positions.dtype}: int64 or int32 expected")
        positions = positions.to(torch.int64).contiguous()
    return _lib.native().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps)
