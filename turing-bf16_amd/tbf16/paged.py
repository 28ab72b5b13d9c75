"""A paged key/value cache: writing new tokens into it, and attention of one new token per
sequence over it (what a decoding loop runs between its linears; the calls convert() and
patch() leave to torch, tbf16/convert.py:29-30 of the reference, which has no cache).

The cache is two bf16 tensors k_cache, v_cache (pages, Hkv, page, D) that the caller
allocates and keeps; a page holds `page` consecutive positions of one sequence. Position j of
sequence b lives in page page_table[b, j // page], row j % page, so its slot is
page_table[b, j // page] * page + j % page. Any strides with a contiguous D work: a cache kept
as (pages, page, Hkv, D) is passed as its transpose(1, 2).

    k_cache, v_cache = (torch.empty(pages, Hkv, 16, D, device="cuda", dtype=torch.bfloat16) for _ in "kv")
    tbf16.paged_write(k_cache, v_cache, k, v, slots)               # k, v (T, Hkv, D), slots int32 (T,)
    o = tbf16.paged_sdpa(q, k_cache, v_cache, page_table, lengths)  # q, o (B, H, D)

Both run on the current stream without waiting for the GPU and can be captured into a graph:
what changes from step to step (slots, page_table, lengths) is read on the device. Inference
only: no gradients. Keys and values stay bf16 and are multiplied as such (bf16 MFMA), so no
power-of-two scales are needed and any bf16 magnitude is taken.
"""
from __future__ import annotations

import ctypes
import math

import torch

from ._ext import launch, lib, ptr

MAX_HEAD_DIM = 256


def _strides(t, n) -> ctypes.Array:
    return (ctypes.c_int64 * n)(*t.stride()[:n])


def _rows_ok(t) -> bool:
    """Contiguous, 16-byte aligned rows along the last dimension."""
    *outer, last = t.stride()
    return last == 1 and t.data_ptr() % 16 == 0 and not any(s % 8 for s in outer)


def _check_cache(fn, k_cache, v_cache, *others):
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError(f"tbf16.{fn}: expected k_cache and v_cache of one shape (pages, Hkv, page, D), got "
                         f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    _, Hkv, page, D = k_cache.shape
    if D % 8 or not 0 < D <= MAX_HEAD_DIM:
        raise ValueError(f"tbf16.{fn}: head dim {D} is not a multiple of 8 up to {MAX_HEAD_DIM}")
    if Hkv == 0 or page == 0:
        raise ValueError(f"tbf16.{fn}: cache of shape {tuple(k_cache.shape)} holds nothing")
    if k_cache.dtype != torch.bfloat16 or v_cache.dtype != torch.bfloat16:
        raise TypeError(f"tbf16.{fn}: expected a bf16 cache")
    if not (_rows_ok(k_cache) and _rows_ok(v_cache)):
        raise ValueError(f"tbf16.{fn}: cache rows must be contiguous and 16-byte aligned (strides multiples of 8)")
    dev = k_cache.device
    if dev.type != "cuda":
        raise ValueError("tbf16: expected tensors on a ROCm (cuda) device")
    for t in (v_cache, *others):
        if t.device != dev:
            raise ValueError(f"tbf16.{fn}: tensors on {t.device} and {dev}")


def _index(fn, name, t, dim):
    if t.dtype != torch.int32 or t.dim() != dim:
        raise TypeError(f"tbf16.{fn}: expected {name} as an int32 tensor of {dim} dimension(s)")
    return t if t.stride(-1) == 1 or t.shape[-1] < 2 else t.contiguous()


def paged_write(k_cache, v_cache, k, v, slots) -> None:
    """k_cache[s // page, :, s % page] = k[t], v_cache likewise, for s = slots[t] of every
    token t. k, v bf16 (T, Hkv, D), any strides; slots int32 (T,). Slots outside the cache
    (negative: a padded batch) leave it as it is; where slots repeat, the last token's rows
    stay. In place; k and v must not lie in the cache's own storage."""
    _check_cache("paged_write", k_cache, v_cache, k, v, slots)
    pages, Hkv, page, D = k_cache.shape
    if k.dim() != 3 or k.shape != v.shape or k.shape[1:] != (Hkv, D):
        raise ValueError(f"tbf16.paged_write: k {tuple(k.shape)} and v {tuple(v.shape)} are not (T, {Hkv}, {D})")
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise TypeError("tbf16.paged_write: expected bf16 k and v")
    slots = _index("paged_write", "slots", slots, 1)
    T = k.shape[0]
    if slots.shape[0] != T:
        raise ValueError(f"tbf16.paged_write: {slots.shape[0]} slots for {T} tokens")
    if pages * page >= 2 ** 31:
        raise ValueError("tbf16.paged_write: the cache has more slots than int32 counts")
    for c in (k_cache, v_cache):
        if any(st == 0 and n > 1 for st, n in zip(c.stride(), c.shape)):
            raise ValueError("tbf16.paged_write: the cache is an expanded view")
    if k_cache.data_ptr() == v_cache.data_ptr() and pages:
        raise ValueError("tbf16.paged_write: k_cache and v_cache are the same memory")
    held = {c.untyped_storage().data_ptr() for c in (k_cache, v_cache)}
    if T and (k.untyped_storage().data_ptr() in held or v.untyped_storage().data_ptr() in held):
        raise ValueError("tbf16.paged_write: k and v lie in the cache's storage")
    torch.autograd.graph.increment_version((k_cache, v_cache))
    if T == 0 or pages == 0:
        return
    k, v = (t if _rows_ok(t) else t.contiguous() for t in (k, v))
    k, v = (t if t.data_ptr() % 16 == 0 else t.clone() for t in (k, v))
    launch("tbf16_paged_write", k_cache, ptr(k), ptr(v), T, Hkv, D, _strides(k, 2), _strides(v, 2), ptr(slots),
           ptr(k_cache), ptr(v_cache), pages, page, _strides(k_cache, 3), _strides(v_cache, 3))


def paged_sdpa(q, k_cache, v_cache, page_table, lengths, scale=None):
    """softmax(scale q k^T) v of one new token per sequence: q bf16 (B, H, D) -> bf16 (B, H, D),
    query head h over key/value head h // (H / Hkv), positions j < lengths[b] of the cache.
    page_table int32 (B, n), lengths int32 (B,) (at most n * page positions are looked at; the
    new token's own is among them once paged_write has put it there). A sequence of length 0
    gives zeros. Entries of page_table outside [0, pages) hold no keys: their positions are
    left out. scale: 1 / sqrt(D) if None. Logits, softmax statistics and sums in fp32, one
    rounding to bf16."""
    _check_cache("paged_sdpa", k_cache, v_cache, q, page_table, lengths)
    pages, Hkv, page, D = k_cache.shape
    if q.dim() != 3 or q.shape[2] != D:
        raise ValueError(f"tbf16.paged_sdpa: q {tuple(q.shape)} is not (B, H, {D})")
    if q.dtype != torch.bfloat16:
        raise TypeError("tbf16.paged_sdpa: expected bf16 q")
    B, H, _ = q.shape
    if H == 0 or H % Hkv:
        raise ValueError(f"tbf16.paged_sdpa: {H} query heads over {Hkv} key/value heads")
    page_table = _index("paged_sdpa", "page_table", page_table, 2)
    lengths = _index("paged_sdpa", "lengths", lengths, 1)
    if page_table.shape[0] != B or lengths.shape[0] != B:
        raise ValueError(f"tbf16.paged_sdpa: page_table for {page_table.shape[0]} and lengths for {lengths.shape[0]} "
                         f"sequences, q has {B}")
    if not _rows_ok(q):
        q = q.contiguous() if q.data_ptr() % 16 == 0 else q.clone(memory_format=torch.contiguous_format)
    o = torch.empty((B, H, D), device=q.device, dtype=torch.bfloat16)
    if B == 0:
        return o
    sc = 1.0 / math.sqrt(D) if scale is None else float(scale)
    ws = torch.empty((max(lib().tbf16_paged_attn_ws_bytes(B, H, Hkv, D), 16),), device=q.device, dtype=torch.uint8)
    launch("tbf16_paged_attn", q, ptr(q), B, H, Hkv, D, _strides(q, 2), ptr(k_cache), ptr(v_cache), pages, page,
           _strides(k_cache, 3), _strides(v_cache, 3), ptr(page_table), page_table.stride(0), page_table.shape[1],
           ptr(lengths), sc, ptr(o), ptr(ws), ws.numel())
    return o
