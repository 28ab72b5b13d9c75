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
power-of-two scales are needed.
"""
from __future__ import annotations

import torch

from ._ext import launch, lib

MAX_HEAD_DIM = 256


def _cache(fn, k_cache, v_cache):
    """(shape, k_cache's strides and address, v_cache's) of a cache the kernels take; raises for
    any other."""
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError(f"tbf16.{fn}: expected k_cache and v_cache of one shape (pages, Hkv, page, D), got "
                         f"{tuple(shape)} and {tuple(v_cache.shape)}")
    _, Hkv, page, D = shape
    if D & 7 or not 0 < D <= MAX_HEAD_DIM:
        raise ValueError(f"tbf16.{fn}: head dim {D} is not a multiple of 8 up to {MAX_HEAD_DIM}")
    if Hkv == 0 or page == 0:
        raise ValueError(f"tbf16.{fn}: cache of shape {tuple(shape)} holds nothing")
    if k_cache.dtype is not torch.bfloat16 or v_cache.dtype is not torch.bfloat16:
        raise TypeError(f"tbf16.{fn}: expected a bf16 cache")
    k_st, v_st, kc, vc = k_cache.stride(), v_cache.stride(), k_cache.data_ptr(), v_cache.data_ptr()
    if (k_st[3] != 1 or v_st[3] != 1 or (k_st[0] | k_st[1] | k_st[2] | v_st[0] | v_st[1] | v_st[2]) & 7
            or (kc | vc) & 15):
        raise ValueError(f"tbf16.{fn}: cache rows must be contiguous and 16-byte aligned (strides multiples of 8)")
    return shape, k_st, kc, v_st, vc


def _same_device(fn, first, *others):
    dev = first.get_device()
    if dev < 0:
        raise ValueError("tbf16: expected tensors on a ROCm (cuda) device")
    for t in others:
        if t.get_device() != dev:
            raise ValueError(f"tbf16.{fn}: tensors on {t.device} and {first.device}")


def _index(fn, name, t, dim):
    if t.dtype is not torch.int32 or t.dim() != dim:
        raise TypeError(f"tbf16.{fn}: expected {name} as an int32 tensor of {dim} dimension(s)")
    return t if t.stride(-1) == 1 or t.shape[-1] < 2 else t.contiguous()


def _rows(t):
    """(t, its strides) with contiguous, 16-byte aligned rows of its last of three dimensions: t
    itself or a copy."""
    st = t.stride()
    if st[2] == 1 and not (st[0] | st[1]) & 7 and not t.data_ptr() & 15:
        return t, st
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride()


def _span(t):
    """The addresses from a bf16 tensor's first element to behind its last one."""
    at = t.data_ptr()
    return at, at + 2 * (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride())))


def paged_write(k_cache, v_cache, k, v, slots) -> None:
    """k_cache[s // page, :, s % page] = k[t], v_cache likewise, for s = slots[t] of every
    token t. k, v bf16 (T, Hkv, D), any strides; slots int32 (T,). Slots outside the cache
    (negative: a padded batch) leave it as it is; where slots repeat, the last token's rows
    stay. In place; k and v must not lie between the cache's first and last element."""
    (pages, Hkv, page, D), kc_st, kc, vc_st, vc = _cache("paged_write", k_cache, v_cache)
    _same_device("paged_write", k_cache, v_cache, k, v, slots)
    shape = k.shape
    T = shape[0] if len(shape) else 0
    if v.shape != shape or shape != (T, Hkv, D):
        raise ValueError(f"tbf16.paged_write: k {tuple(shape)} and v {tuple(v.shape)} are not (T, {Hkv}, {D})")
    if k.dtype is not torch.bfloat16 or v.dtype is not torch.bfloat16:
        raise TypeError("tbf16.paged_write: expected bf16 k and v")
    slots = _index("paged_write", "slots", slots, 1)
    if slots.shape[0] != T:
        raise ValueError(f"tbf16.paged_write: {slots.shape[0]} slots for {T} tokens")
    if pages * page >= 2 ** 31:
        raise ValueError("tbf16.paged_write: the cache has more slots than int32 counts")
    if 0 in kc_st or 0 in vc_st:
        for c in (k_cache, v_cache):
            if any(st == 0 and n > 1 for st, n in zip(c.stride(), c.shape)):
                raise ValueError("tbf16.paged_write: the cache is an expanded view")
    if kc == vc and pages:
        raise ValueError("tbf16.paged_write: k_cache and v_cache are the same memory")
    held = k_cache.untyped_storage().data_ptr(), v_cache.untyped_storage().data_ptr()
    if T and pages and (k.untyped_storage().data_ptr() in held or v.untyped_storage().data_ptr() in held):
        # one allocation for all of them: fine where they lie apart in it
        for t in (k, v):
            for c in (k_cache, v_cache):
                (t0, t1), (c0, c1) = _span(t), _span(c)
                if t0 < c1 and c0 < t1:
                    raise ValueError("tbf16.paged_write: k and v lie in the cache's storage, within its rows")
    torch.autograd.graph.increment_version((k_cache, v_cache))
    if T == 0 or pages == 0:
        return
    (k, k_st), (v, v_st) = _rows(k), _rows(v)
    launch("tbf16_paged_write", k_cache, k.data_ptr(), v.data_ptr(), T, Hkv, D, k_st[0], k_st[1], v_st[0], v_st[1],
           slots.data_ptr(), kc, vc, pages, page, kc_st[0], kc_st[1], kc_st[2], vc_st[0], vc_st[1], vc_st[2])


# tbf16_paged_attn's workspace bytes per (device, B, H, Hkv, D, positions a table row covers): its
# blocks are counted by the device's CUs, so it is asked on the tensors' device, once
_WS_BYTES: dict = {}


def _ws_bytes(dev: int, *sizes: int) -> int:
    key = (dev, sizes)
    n = _WS_BYTES.get(key)
    if n is None:
        if len(_WS_BYTES) > 4096:
            _WS_BYTES.clear()
        with torch.cuda.device(dev):
            n = _WS_BYTES[key] = int(lib().tbf16_paged_attn_ws_bytes(*sizes))
    return n


def paged_sdpa(q, k_cache, v_cache, page_table, lengths, scale=None):
    """softmax(scale q k^T) v of one new token per sequence: q bf16 (B, H, D) -> bf16 (B, H, D),
    query head h over key/value head h // (H / Hkv), positions j < lengths[b] of the cache.
    page_table int32 (B, n), lengths int32 (B,) (at most n * page positions are looked at; the
    new token's own is among them once paged_write has put it there). A sequence of length 0
    gives zeros. Entries of page_table outside [0, pages) hold no keys: their positions are
    left out. scale: 1 / sqrt(D) if None. Logits, softmax statistics and sums in fp32, one
    rounding to bf16 (weights relative to the row's largest, the sum of weighted values may reach
    8e40, 256 times bf16's largest value). An infinite value makes its element infinite; where its
    key's weight is below 2^-90 of the row's largest the weight may count as zero, and the element
    is NaN."""
    (pages, Hkv, page, D), k_st, kc, v_st, vc = _cache("paged_sdpa", k_cache, v_cache)
    _same_device("paged_sdpa", k_cache, v_cache, q, page_table, lengths)
    if q.dim() != 3 or q.shape[2] != D:
        raise ValueError(f"tbf16.paged_sdpa: q {tuple(q.shape)} is not (B, H, {D})")
    if q.dtype is not torch.bfloat16:
        raise TypeError("tbf16.paged_sdpa: expected bf16 q")
    B, H, _ = q.shape
    if H == 0 or H % Hkv:
        raise ValueError(f"tbf16.paged_sdpa: {H} query heads over {Hkv} key/value heads")
    page_table = _index("paged_sdpa", "page_table", page_table, 2)
    lengths = _index("paged_sdpa", "lengths", lengths, 1)
    rows, n = page_table.shape
    if rows != B or lengths.shape[0] != B:
        raise ValueError(f"tbf16.paged_sdpa: page_table for {rows} and lengths for {lengths.shape[0]} sequences, q has {B}")
    q, q_st = _rows(q)
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    if B == 0:
        return o
    wsb = _ws_bytes(q.get_device(), B, H, Hkv, D, n * page)
    ws = q.new_empty(wsb, dtype=torch.uint8) if wsb else o  # (o: nothing is written there)
    launch("tbf16_paged_attn", q, q.data_ptr(), B, H, Hkv, D, q_st[0], q_st[1], kc, vc, pages, page, k_st[0], k_st[1],
           k_st[2], v_st[0], v_st[1], v_st[2], page_table.data_ptr(), page_table.stride(0), n, lengths.data_ptr(),
           D ** -0.5 if scale is None else float(scale), o.data_ptr(), ws.data_ptr(), wsb)
    return o
