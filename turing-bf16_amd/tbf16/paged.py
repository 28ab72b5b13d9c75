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

from ._ext import launch, lib, ptr
from ._ext import same_device as _same_device, ws_bytes as _ws_bytes

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


def _index(fn, name, t, dim):
    st = t.stride()
    if t.dtype is not torch.int32 or len(st) != dim:
        raise TypeError(f"tbf16.{fn}: expected {name} as an int32 tensor of {dim} dimension(s)")
    return t if st[-1] == 1 or t.shape[-1] < 2 else t.contiguous()


def _rows(t):
    """(t, its strides) with contiguous, 16-byte aligned rows of its last of three dimensions: t
    itself or a copy."""
    st = t.stride()
    if st[2] == 1 and not (st[0] | st[1]) & 7 and not t.data_ptr() & 15:
        return t, st
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride()


def _span(t):
    """The addresses from a tensor's first element to behind its last one."""
    at = t.data_ptr()
    return at, at + t.element_size() * (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride())))


def paged_advance(page_table, lengths, counts, free_pages, n_free, page, tokens, prefix_length=None):
    """Makes sequences of a paged cache longer by counts[b] tokens, or shorter by -counts[b], and
    says where the new tokens belong: (slots, positions, starts), int32 (tokens,), (tokens,) and
    (B + 1,). All on the device, in place, without waiting for it:

      page_table  int32 (B, n): sequence b's pages, each of which no other entry names (a page that
                  two entries give back goes on the stack twice); lengths int32 (B,): its tokens so far
      counts      int32 (B,): new tokens (0: none); negative: the last -counts[b] tokens are taken
                  back, all of them where there are fewer (a request that ends: -lengths[b])
      free_pages  int32 (pages,): a stack of the pages that nobody has, n_free int32 (1,) of them, the
                  next one taken last; pages is also the number of the cache's pages
      page        positions a page has; tokens: new tokens there is room for in this call

    First, pages that no position below the shortened lengths uses go back on the stack and
    their table entries become -1 (entries that name no page are not given back). Then sequences
    get their new tokens in order of b. One whose tokens do not fit its table row or `tokens`, or
    that needs pages that are no longer there after what the sequences before it asked for, gets
    none: its length stays. (What one asked for and did not get counts too: behind a prompt that finds
    too few pages nobody gets one. Sequences that decode belong before prompts in the batch.) The new
    tokens of all sequences lie one after the other, those of b from starts[b] on (at most `tokens`):
    slots for paged_write, positions from the sequence's old length on, plus prefix_length int32 (1,) where one is given (the tokens of a prefix that all
    sequences share, which the tables do not hold). Tokens that were not granted, and those past
    the last one, have slot and position -1, which paged_write leaves out and qk_norm_rope gives
    zeros. Taking all granted tokens back leaves lengths, table and the stack's n_free pages as they
    were, if lengths and n_free were in range, entries past a sequence's pages -1 and the stack's entries
    pages of the cache (other entries become -1, and an id that is no page does not go back).

    The attentions' rows are sequences, not tokens. Where a step has at most one new token for each of them and none for
    some, the tokens' slots and positions go into the order of sequences before anything is computed by them:

        new, at = starts[1:] > starts[:-1], starts[:-1].clamp(max=tokens - 1)
        slots, positions = torch.where(new, slots[at], -1), torch.where(new, positions[at], -1)

    Lengths outside [0, n * page] count as the nearest there is, n_free likewise."""
    shape, row = page_table.shape, page_table.stride()
    others = (lengths, counts, free_pages, n_free) if prefix_length is None else (lengths, counts, free_pages, n_free, prefix_length)
    if len(shape) != 2:
        raise ValueError(f"tbf16.paged_advance: page_table {tuple(shape)} is not (B, n)")
    B, n = shape
    sizes = [t.numel() for t in others]
    if sizes[:2] != [B, B] or sizes[3] != 1 or sizes[-1] != 1:
        raise ValueError(f"tbf16.paged_advance: {sizes[0]} lengths and {sizes[1]} counts for {B} sequences; n_free and "
                         f"prefix_length are one number each, got {sizes[3:]}")
    at = page_table.data_ptr()
    spans = [(at, at + 4 * ((B - 1) * row[0] + n))] if B and n else []
    for t, size in zip(others, sizes):
        if t.dtype is not torch.int32:
            raise TypeError(f"tbf16.paged_advance: expected int32, got {t.dtype} {tuple(t.shape)}")
        if t.dim() > 1 or not t.is_contiguous():
            raise ValueError(f"tbf16.paged_advance: lengths, counts and free_pages must be contiguous, of one dimension, got {tuple(t.shape)}")
        if size:
            at = t.data_ptr()
            spans.append((at, at + 4 * size))
    if page_table.dtype is not torch.int32:
        raise TypeError(f"tbf16.paged_advance: expected page_table as int32, got {page_table.dtype}")
    if (n > 1 and row[1] != 1) or (B > 1 and row[0] < n):
        raise ValueError("tbf16.paged_advance: page_table's rows must be contiguous and apart")
    _same_device("paged_advance", page_table, *others)
    spans.sort()
    end = 0
    for span in spans:
        if span[0] < end:
            raise ValueError("tbf16.paged_advance: two of its arguments lie in the same memory")
        end = span[1]
    pages, page, tokens = sizes[2], int(page), int(tokens)
    if page < 1 or pages * page >= 2 ** 31 - 1:
        raise ValueError(f"tbf16.paged_advance: {pages} pages of {page} positions")
    if not 0 <= tokens < 2 ** 31 - 1024 or B * max(n, 2) >= 2 ** 31:
        raise ValueError(f"tbf16.paged_advance: room for {tokens} tokens, page_table {tuple(shape)}")
    torch.autograd.graph.increment_version((page_table, lengths, free_pages, n_free))
    slots, positions, starts = page_table.new_empty(tokens), page_table.new_empty(tokens), page_table.new_empty(B + 1)
    wsb = lib().tbf16_paged_advance_ws_bytes(B, tokens)
    ws = page_table.new_empty(wsb, dtype=torch.uint8) if wsb else None
    launch("tbf16_paged_advance", page_table, page_table.data_ptr(), max(row[0], n), B, n, lengths.data_ptr(),
           counts.data_ptr(), free_pages.data_ptr(), pages, n_free.data_ptr(), page, tokens, ptr(prefix_length),
           slots.data_ptr(), positions.data_ptr(), starts.data_ptr(), ptr(ws), wsb)
    return slots, positions, starts


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


def _queries(fn, q, Hkv, D, page_table, lengths):
    """(q, its strides, B, H, page_table, its entries a sequence, lengths), checked."""
    shape = q.shape
    if len(shape) != 3 or shape[2] != D:
        raise ValueError(f"tbf16.{fn}: q {tuple(shape)} is not (B, H, {D})")
    if q.dtype is not torch.bfloat16:
        raise TypeError(f"tbf16.{fn}: expected bf16 q")
    B, H, _ = shape
    if H == 0 or H % Hkv:
        raise ValueError(f"tbf16.{fn}: {H} query heads over {Hkv} key/value heads")
    page_table = _index(fn, "page_table", page_table, 2)
    lengths = _index(fn, "lengths", lengths, 1)
    rows, n = page_table.shape
    if rows != B or lengths.shape[0] != B:
        raise ValueError(f"tbf16.{fn}: page_table for {rows} and lengths for {lengths.shape[0]} sequences, q has {B}")
    q, q_st = _rows(q)
    return q, q_st, B, H, page_table, n, lengths


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
    q, q_st, B, H, page_table, n, lengths = _queries("paged_sdpa", q, Hkv, D, page_table, lengths)
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    if B == 0:
        return o
    wsb = _ws_bytes(q.get_device(), "tbf16_paged_attn_ws_bytes", B, H, Hkv, D, n * page)
    ws = q.new_empty(wsb, dtype=torch.uint8) if wsb else o  # (o: nothing is written there)
    launch("tbf16_paged_attn", q, q.data_ptr(), B, H, Hkv, D, q_st[0], q_st[1], kc, vc, pages, page, k_st[0], k_st[1],
           k_st[2], v_st[0], v_st[1], v_st[2], page_table.data_ptr(), page_table.stride(0), n, lengths.data_ptr(),
           D ** -0.5 if scale is None else float(scale), o.data_ptr(), ws.data_ptr(), wsb)
    return o


def paged_sdpa_prefix(q, k_cache, v_cache, prefix_table, prefix_length, page_table, lengths, scale=None):
    """paged_sdpa where all sequences begin with the same tokens (a system prompt, a document that
    all of them ask about): positions j < prefix_length[0] of prefix_table int32 (m,), int32 (1,), come
    before each sequence's own positions j < lengths[b] of page_table. The prefix's keys and values
    are read once for the whole batch and multiplied with all its queries. One softmax over both:
    the result is paged_sdpa's on sequences that hold the prefix's tokens before their own.

    Arguments, results and limits as paged_sdpa's; a sequence without any key gives zeros. Weights of
    prefix keys below 2^-80 of the row's largest may count as zero (an infinite value then gives NaN)."""
    (pages, Hkv, page, D), k_st, kc, v_st, vc = _cache("paged_sdpa_prefix", k_cache, v_cache)
    _same_device("paged_sdpa_prefix", k_cache, v_cache, q, prefix_table, prefix_length, page_table, lengths)
    q, q_st, B, H, page_table, n, lengths = _queries("paged_sdpa_prefix", q, Hkv, D, page_table, lengths)
    prefix_table = _index("paged_sdpa_prefix", "prefix_table", prefix_table, 1)
    if prefix_length.dtype is not torch.int32 or prefix_length.numel() != 1:
        raise TypeError(f"tbf16.paged_sdpa_prefix: expected prefix_length as one int32, got {tuple(prefix_length.shape)}")
    m = prefix_table.shape[0]
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    if B == 0:
        return o
    wsb = _ws_bytes(q.get_device(), "tbf16_paged_attn_prefix_ws_bytes", B, H, Hkv, D, m * page, n * page)
    ws = q.new_empty(wsb, dtype=torch.uint8)
    launch("tbf16_paged_attn_prefix", q, q.data_ptr(), B, H, Hkv, D, q_st[0], q_st[1], kc, vc, pages, page, k_st[0],
           k_st[1], k_st[2], v_st[0], v_st[1], v_st[2], prefix_table.data_ptr(), m, prefix_length.data_ptr(),
           page_table.data_ptr(), page_table.stride(0), n, lengths.data_ptr(), D ** -0.5 if scale is None else float(scale),
           o.data_ptr(), ws.data_ptr(), wsb)
    return o
