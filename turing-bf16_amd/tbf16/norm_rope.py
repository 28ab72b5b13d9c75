"""RMS norm of every query and key head and rotation by position, in one pass over both: what stands
between a model's projections and its attention. No counterpart in the reference.

    angles = torch.arange(n, dtype=torch.float64)[:, None] * base ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    cos, sin = angles.cos().float().cuda(), angles.sin().float().cuda()      # (n, R / 2), once
    q, k = tbf16.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions)

tbf16.autograd.qk_norm_rope is the same with gradients.
"""
from __future__ import annotations

import torch

from ._ext import launch, ptr, same_device, ws_bytes

MAX_HEAD_DIM = 256
_CONTIGUOUS = torch.contiguous_format


def _heads(x):
    """(x, its address, its (b, s, h) strides) with heads the kernels read in place: x itself or a copy."""
    st, at = x.stride(), x.data_ptr()
    if len(st) == 3:
        sb, (ss, sh, step) = 0, st
    else:
        sb, ss, sh, step = st
    if step != 1 or (sb | ss | sh) & 7 or at & 15:
        return _heads(x.clone(memory_format=_CONTIGUOUS))
    return x, at, (sb, ss, sh)


def _table(t):
    return t if t.is_contiguous() and not t.data_ptr() & 15 else t.clone(memory_format=_CONTIGUOUS)


def _checked(q, k, wq, wk, cos, sin, positions, eps, interleaved):
    """(sizes, tail, kept): the arguments of the entry points that are alike for both directions, around the
    heads, and the tensors that their addresses belong to. Raises for what the kernels do not take."""
    shape, kshape = q.shape, k.shape
    D, n = shape[-1] if len(shape) else 0, len(shape)
    if ((n != 3 and n != 4) or len(kshape) != n or shape[0] != kshape[0] or shape[n - 3] != kshape[n - 3] or kshape[-1] != D
            or not shape[-2] or not kshape[-2]):
        raise ValueError(f"tbf16.qk_norm_rope: q {tuple(shape)} and k {tuple(kshape)} are not ((B,) S, H, D) and "
                         "((B,) S, Hkv, D)")
    if D & 15 or not 0 < D <= MAX_HEAD_DIM:
        raise ValueError(f"tbf16.qk_norm_rope: head dim {D} is not a multiple of 16 up to {MAX_HEAD_DIM}")
    if q.dtype is not torch.bfloat16 or k.dtype is not torch.bfloat16:
        raise TypeError("tbf16.qk_norm_rope: expected bf16 q and k")
    if wq.shape != (D,) or wk.shape != (D,):
        raise ValueError(f"tbf16.qk_norm_rope: weights {tuple(wq.shape)} and {tuple(wk.shape)} are not ({D},)")
    wide = wq.dtype is torch.float32
    if wq.dtype is not wk.dtype or not (wide or wq.dtype is torch.bfloat16):
        raise TypeError("tbf16.qk_norm_rope: expected weights both bf16 or both fp32")
    table = cos.shape
    if len(table) != 2 or table != sin.shape or table[0] == 0:
        raise ValueError(f"tbf16.qk_norm_rope: cos {tuple(table)} and sin {tuple(sin.shape)} are not tables of one "
                         "shape (positions, rotated dims / 2)")
    if cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
        raise TypeError("tbf16.qk_norm_rope: expected fp32 cos and sin")
    R = 2 * table[1]
    if R & 15 or not 0 < R <= D:
        raise ValueError(f"tbf16.qk_norm_rope: {R} rotated dims are not a multiple of 16 up to the head dim {D}")
    if positions.dtype is not torch.int32:
        raise TypeError("tbf16.qk_norm_rope: expected int32 positions")
    B, S = (1, shape[0]) if n == 3 else shape[:2]
    p, p_st = positions.shape, positions.stride()
    if p == (S,):
        p_st = 0, p_st[0]
    elif n == 3 or p != (B, S):
        raise ValueError(f"tbf16.qk_norm_rope: positions {tuple(p)} for tokens {tuple(shape[:-2])}")
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"tbf16.qk_norm_rope: eps {eps}")
    if B * S >= 2 ** 31:
        raise ValueError(f"tbf16.qk_norm_rope: {B * S} tokens")
    same_device("qk_norm_rope", q, k, wq, wk, cos, sin, positions)
    wq, wk, cos, sin = _table(wq), _table(wk), _table(cos), _table(sin)
    return ((B, S, shape[-2], kshape[-2], D),
            (wq.data_ptr(), wk.data_ptr(), wide, cos.data_ptr(), sin.data_ptr(), table[0], R, positions.data_ptr(), *p_st, eps,
             bool(interleaved)), (wq, wk, cos, sin))


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps=1e-6, interleaved=False):
    """(q', k'): with u = x / sqrt(mean(x^2) + eps) over a head and z = u * weight, the first R
    elements of z rotated by the token's position p in pairs (i, i + R / 2), or neighbours (2 i, 2 i + 1) where
    `interleaved`: (z_i cos[p, i] - z_j sin[p, i], z_j cos[p, i] + z_i sin[p, i]); elements from R on as they are.

    q bf16 (S, H, D) or (B, S, H, D), k the same with Hkv heads, any strides (views of one projection's
    output); weights (D,) bf16 or fp32; cos, sin fp32 (positions, R / 2); positions int32 (S,), or (B, S).
    D and R multiples of 16, D up to 256, R up to D. Returns contiguous bf16 tensors, rounded once from
    fp32. Tokens of a negative position are padding and give zeros; a position past the tables has no
    angle and gives NaN, as does a head of zeros without an eps. Inference only; gradients:
    tbf16.autograd.qk_norm_rope."""
    sizes, tail, kept = _checked(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    yq = torch.empty_like(q, memory_format=_CONTIGUOUS)
    yk = torch.empty_like(k, memory_format=_CONTIGUOUS)
    q, at_q, q_st = _heads(q)
    k, at_k, k_st = _heads(k)
    launch("tbf16_qk_norm_rope", q, at_q, at_k, *sizes, *q_st, *k_st, *tail, yq.data_ptr(), yk.data_ptr())
    return yq, yk


def backward(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, dyq, dyk, wanted):
    """Gradients of q, k and both weights (None where wanted says so) from those of the outputs."""
    sizes, tail, kept = _checked(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    dev = same_device("qk_norm_rope", q, dyq, dyk)
    if dyq.shape != q.shape or dyk.shape != k.shape or dyq.dtype is not torch.bfloat16 or dyk.dtype is not torch.bfloat16:
        raise ValueError(f"tbf16.qk_norm_rope: gradients {tuple(dyq.shape)} {dyq.dtype} and {tuple(dyk.shape)} {dyk.dtype}")
    want_q, want_k, want_wq, want_wk = wanted
    dq = torch.empty_like(q, memory_format=_CONTIGUOUS) if want_q else None
    dk = torch.empty_like(k, memory_format=_CONTIGUOUS) if want_k else None
    dwq = torch.empty_like(kept[0]) if want_wq else None
    dwk = torch.empty_like(kept[1]) if want_wk else None
    ws, wsb = None, 0
    if want_wq or want_wk:
        wsb = ws_bytes(dev, "tbf16_qk_norm_rope_bwd_ws_bytes", *sizes)
        ws = q.new_empty(wsb, dtype=torch.uint8)
    q, at_q, q_st = _heads(q)
    k, at_k, k_st = _heads(k)
    dyq, at_dyq, dyq_st = _heads(dyq)
    dyk, at_dyk, dyk_st = _heads(dyk)
    launch("tbf16_qk_norm_rope_bwd", q, at_q, at_k, at_dyq, at_dyk, *sizes, *q_st, *k_st, *dyq_st, *dyk_st, *tail,
           ptr(dq), ptr(dk), ptr(dwq), ptr(dwk), ptr(ws), wsb)
    return dq, dk, dwq, dwk
