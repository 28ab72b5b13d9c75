"""Training: backward passes on fp16 MFMA.

Linear: dX = dY @ W and dW = dY^T @ X are scaled fp16 GEMMs too. The contraction
dimension changes, so dY, W and X are scaled per column (exact powers of two)
where the forward pass scaled per row (tbf16/autograd.py:58-90 of the reference).
The column-scaled operands are written transposed by their quantisation pass,
so every GEMM reads both operands contraction-contiguous.

Attention: a fused flash-style backward with dO multiplied by a power of two
2^G picked so dS stays in fp16's normal range. If any gradient would overflow
fp16 the backward is redone with a smaller G: per-op loss scaling decided
immediately, so no step is ever skipped (same policy and retry as the reference,
tbf16/autograd.py:166-193). By default the retry is decided on the device: a
second, gated kernel call redoes the backward at the retried scale only when the
first one overflowed, so the host never waits for the GPU inside backward().
"""
from __future__ import annotations

import functools
import math
import os

import torch
import torch.nn.functional as F

from . import attention, norm_rope, ops, routing
from ._ext import launch, lib, ptr, strides3

# How the attention backward applies the overflow retry (TBF16_ATTN_CHECK):
#   "device" (default): a gated second call redoes the backward on the device at the
#       retried scale only if the first overflowed, so no host sync inside the
#       attention backward. The one case the device cannot settle, an overflow that
#       persists through every retry (non-finite dO), is checked once per
#       backward() call by a callback queued on the autograd engine: it waits for
#       the attention backwards' overflow words and raises FloatingPointError before
#       backward() returns, i.e. before an optimizer step can use the gradients (one
#       host sync per backward() call, not one per attention layer). Under HIP-graph
#       capture nothing can be waited for: the check is left to check_pending();
#   "deferred": as "device" without the end-of-backward callback: the error is
#       raised by a later backward or by check_pending(), once the GPU has got there;
#   "sync" (or "1"): the reference's host loop, one host sync per attention
#       backward, the error raised at once;
#   "off" (or "0"): one attempt, unchecked.
CHECK_OVERFLOW = {"0": "off", "off": "off", "1": "sync", "sync": "sync", "deferred": "deferred"}.get(
    os.environ.get("TBF16_ATTN_CHECK", "device").lower(), "device")
ATTN_RETRIES = 6
# An attempt's overflow word is the bit pattern of its largest fp16 intermediate
# magnitude (+inf if not finite); at 65520.0f = 0x477FF000 and above fp16 overflows.
_OVF_BITS = 0x477FF000


def _pad8(n: int) -> int:
    return n + (-n) % 8


def _quantize_cols_t(x: torch.Tensor, target_exp: int = 0, row_mul=None):
    """Column quantisation with the fp16 result transposed: (yT (K, R8), s_inv (K,)),
    R8 = R rounded up to 8, zero-filled past R."""
    x = ops._pad_cols(x) if not ops._ok_rows(x) else x
    R, K = x.shape
    R8 = _pad8(R)
    yT = torch.empty((K, R8), device=x.device, dtype=torch.float16)
    s_inv = torch.empty((K,), device=x.device, dtype=torch.float32)
    rm = None if row_mul is None else row_mul.float().contiguous()
    wsb = lib().tbf16_quantize_cols_ws_bytes(R, K)
    ws = torch.empty(max(wsb, 16), device=x.device, dtype=torch.uint8)
    launch("tbf16_quantize_cols_t", x, ptr(x), R, K, x.stride(0), int(target_exp), ptr(rm), ptr(yT), yT.stride(0),
           ptr(s_inv), ptr(ws), ws.numel())
    return yT, s_inv


def quantize_cols(x: torch.Tensor, target_exp: int = 0, row_mul=None):
    """bf16 (R, K) -> (fp16 (R, K), fp32 (K,) inverse scales), one power-of-two scale per column.
    row_mul (R,) powers of two, optional: quantize x * row_mul[:, None] instead (exact)
    (tbf16/autograd.py:26-36). The fp16 result is a transposed view of a K-major buffer."""
    if x.dtype != torch.bfloat16:
        raise TypeError("tbf16.quantize_cols: expected bf16")
    R, K = x.shape
    yT, s_inv = _quantize_cols_t(x, target_exp, row_mul)
    return yT[:K, :R].t(), s_inv


def _gemm_nt(a16, sa, bT16, sb, bias=None):
    """bf16((a16 @ bT16^T) * sa[:, None] * sb[None, :] + bias), both operands K-contiguous."""
    return ops.linear_q(a16, sa, bT16, sb, bias)


@torch.autocast("cuda", enabled=False)
def _scaled_mm(a16, sa, b16, sb):
    """(a16 @ b16) * sa[:, None] * sb[None, :] as bf16 (tbf16/autograd.py:49-55)."""
    a = a16 if a16.stride(-1) == 1 else a16.contiguous()
    bT = b16.t()
    bT = bT if bT.stride(-1) == 1 else bT.contiguous()
    return _gemm_nt(a, sa, bT, sb)


def _quantize_rows_t(x2: torch.Tensor, t: int):
    """(x16T (K, M8), sx (M,), exps (M,)): max row scales at t, fp16 written transposed."""
    x2 = ops._pad_cols(x2) if not ops._ok_rows(x2) else x2
    M, K = x2.shape
    M8 = _pad8(M)
    x16T = torch.empty((K, M8), device=x2.device, dtype=torch.float16)
    sx = torch.empty((M,), device=x2.device, dtype=torch.float32)
    exps = torch.empty((M,), device=x2.device, dtype=torch.int32)
    launch("tbf16_quantize_rows_t", x2, ptr(x2), M, K, x2.stride(0), int(t), ptr(x16T), x16T.stride(0), ptr(sx),
           ptr(exps))
    return x16T, sx, exps


def _one_call(w, *others) -> bool:
    """Whether the native halves of the training linear take these operands as they are:
    bf16 matrices with 16-byte rows (both dimensions multiples of 8), not empty, and no
    pinned tile configuration. Everything else goes pass by pass, with the same values."""
    return (ops._GEMM_CFG < 0 and w.shape[0] % 8 == 0 and w.numel() > 0
            and all(m.dtype == torch.bfloat16 and m.shape[0] > 0 and ops._ok_rows(m) for m in (w, *others)))


def _linear_forward(x2, w, bias, t, transposed=True):
    """(y, (x16T, sx)) in one native call, or (y, None): without `transposed`, for the
    further layers of one x. x's fp16 rows last for the call only."""
    ops._dev_check(x2, w)
    N, K = w.shape
    M, dev = x2.shape[0], x2.device
    L = lib()
    y = torch.empty((M, N), device=dev, dtype=torch.bfloat16)
    x16 = torch.empty((M, K), device=dev, dtype=torch.float16)
    sx = torch.empty((M,), device=dev, dtype=torch.float32)
    x16T = exps = None
    if transposed:
        x16T = torch.empty((K, _pad8(M)), device=dev, dtype=torch.float16)
        exps = torch.empty((M,), device=dev, dtype=torch.int32)
    ws = torch.empty((L.tbf16_train_linear_fwd_ws_bytes(N, K),), device=dev, dtype=torch.uint8)
    b = ops._bias_bf16(bias, N, dev)
    launch("tbf16_train_linear_fwd", x2, ptr(x2), M, K, x2.stride(0), ptr(w), N, w.stride(0), ptr(b), int(t), ptr(x16),
           ptr(x16T), _pad8(M), ptr(sx), ptr(exps), ptr(y), N, ptr(ws), ws.numel())
    return y, ((x16T, sx) if transposed else None)


class ScaledLinearFn(torch.autograd.Function):
    """tbf16/autograd.py:58-90: x rows max-scaled at target_exp(K) (their transposed fp16
    copy is saved instead of x, same size), w via prepare_weight, fp32 accumulation."""

    @staticmethod
    def forward(ctx, x, w, bias):
        N, K = w.shape
        x2 = x.reshape(-1, K)
        t = ops._target_exp(K)
        # x's transposed fp16 rows, which dW needs, are made once for every layer that x
        # feeds (Q/K/V, gate/up); the rows of this product are made for each, beside those
        # of w: kept, they would be a second copy of every live activation
        if _one_call(w, x2):
            made = []

            def build():
                y, rows_t = _linear_forward(x2, w, bias, t)
                made.append(y)
                return rows_t

            x16T, sx = routing.activations.get(x, ("rows_t", t, K), build)
            y = made[0] if made else _linear_forward(x2, w, bias, t, transposed=False)[0]
        else:
            x16T, sx = routing.activations.get(x, ("rows_t", t, K), lambda: _quantize_rows_t(x2, t)[:2])
            x16, _ = ops.quantize_rows(x2 if ops._ok_rows(x2) else ops._pad_cols(x2), t)
            y = _gemm_nt(x16[:, :K], sx, *ops.prepare_weight(w), bias)
        ctx.save_for_backward(x16T, sx, w)
        ctx.has_bias = bias is not None
        ctx.x_shape = x.shape
        return y.reshape(*x.shape[:-1], N)

    @staticmethod
    def backward(ctx, dy):
        x16T, sx, w = ctx.saved_tensors
        ops._dev_check(dy, x16T, sx, w)
        N, K = w.shape
        dy2 = dy.reshape(-1, N).to(torch.bfloat16).contiguous()
        M = dy2.shape[0]
        want_x, want_w, want_b = ctx.needs_input_grad
        want_b = want_b and ctx.has_bias
        t_w = ops._target_exp(N)
        t_dy = min(0, 15 - math.ceil(math.log2(max(M, 1))))
        # (x16T may have been unpacked by a saved-tensor hook, in any layout)
        if (_one_call(w, dy2) and x16T.shape[1] == _pad8(M) and x16T.is_contiguous() and x16T.data_ptr() % 16 == 0
                and sx.dtype == torch.float32 and sx.is_contiguous()):
            dev = dy2.device
            dx = torch.empty((M, K), device=dev, dtype=torch.bfloat16) if want_x else None
            dw = torch.empty((N, K), device=dev, dtype=torch.bfloat16) if want_w else None
            db = torch.empty((N,), device=dev, dtype=torch.bfloat16) if want_b and dy.dtype == torch.bfloat16 else None
            wsb = lib().tbf16_train_linear_bwd_ws_bytes(M, N, K, dx is not None, dw is not None, db is not None)
            ws = torch.empty((wsb,), device=dev, dtype=torch.uint8)
            launch("tbf16_train_linear_bwd", dy2, ptr(dy2), M, N, dy2.stride(0), ptr(w), K, w.stride(0), ptr(x16T),
                   x16T.stride(0), ptr(sx), int(t_w), int(ops.L1_TARGET), int(t_dy), ptr(dx), ptr(dw), ptr(db), ptr(ws),
                   ws.numel())
            if want_b and db is None:
                db = dy2.float().sum(0).to(dy.dtype)
            return (None if dx is None else dx.reshape(ctx.x_shape)), dw, db
        dx = dw = db = None
        if want_x:  # contraction over N
            w16cT, swc = _quantize_cols_t(w.contiguous(), t_w)
            # dY rows L1-scaled (|w16c| <= 1 bounds dX16 by 2^15), padded to w16cT's length
            dyp = dy2 if ops._ok_rows(dy2) else ops._pad_cols(dy2)
            dy16, sdy = ops.quantize_rows(dyp, ops.L1_TARGET, l1=True)
            dx = _gemm_nt(dy16, sdy, w16cT, swc)[:, :K].reshape(ctx.x_shape)
        if want_w:  # contraction over M
            # dW[n, k] = sum_m dy[m, n] * sx[m] * x16[m, k]: fold sx into dY, column-scale per n.
            dy16cT, sdyc = _quantize_cols_t(dy2, t_dy, sx)
            # (both operands have the columns that pad N and K to multiples of 8)
            dw = _gemm_nt(dy16cT, sdyc, x16T, _unit_scales(x16T.shape[0], dy2.device))[:N, :K]
        if want_b:
            db = dy2.float().sum(0).to(dy.dtype)
        return dx, dw, db


@functools.lru_cache(maxsize=32)
def _unit_scales(n: int, device: torch.device) -> torch.Tensor:
    """fp32 ones (n,): the inverse scales of an operand that is not scaled (dW's x16^T
    carries its row scales in dY)."""
    return torch.ones(n, device=device)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t as a 2-D (rows, last dim) view."""
    return t.reshape(-1, t.shape[-1])


class FP32LinearFn(torch.autograd.Function):
    """Linear layer computed in fp32 for bf16 tensors (tbf16/autograd.py:93-112): the
    route for skinny layers (LoRA adapters), whose shapes the scaled kernels would
    not fill. Only the bf16 operands are saved; each product is upcast on use."""

    @staticmethod
    @torch.autocast("cuda", enabled=False)
    def forward(ctx, x, w, bias):
        ctx.save_for_backward(x, w)
        ctx.bias_dtype = None if bias is None else bias.dtype
        y = torch.matmul(x.float(), w.float().t())
        if bias is not None:
            y = y + bias.float()
        return y.to(x.dtype)

    @staticmethod
    @torch.autocast("cuda", enabled=False)
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad
        g = _rows(dy).float()
        dx = torch.matmul(dy.float(), w.float()).to(x.dtype) if want_x else None
        dw = torch.matmul(g.t(), _rows(x).float()).to(w.dtype) if want_w else None
        db = g.sum(dim=0).to(dy.dtype) if (want_b and ctx.bias_dtype is not None) else None
        return dx, dw, db


def linear(x, w, bias=None):
    """Differentiable F.linear for bf16 x and w on fp16 MFMA (tbf16/autograd.py:115-117)."""
    return ScaledLinearFn.apply(x, w, bias)


def _attn_backward_once(q, k, v, o16, lse, dout, exps_fwd, bias, scale, causal, t_do, dropout_p=0.0, seed=0,
                        overflow=None, gate=None, outs=None, ws=None):
    """One backward attempt at dO target exponent t_do: (dq, dk, dv, exps_out, overflow, ws).
    overflow: the device int32 word the attempt writes (allocated if None); gate and
    outs / ws: an earlier attempt's word, outputs and workspace for a gated retry."""
    B, H, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    dev = q.device
    if outs is None:
        outs = (torch.empty(B, H, Sq, D, device=dev, dtype=torch.bfloat16),
                torch.empty(B, Hkv, Sk, D, device=dev, dtype=torch.bfloat16),
                torch.empty(B, Hkv, Sk, D, device=dev, dtype=torch.bfloat16),
                torch.empty(2, device=dev, dtype=torch.int32))
    dq, dk, dv, exps_out = outs
    if overflow is None:
        overflow = torch.zeros(1, device=dev, dtype=torch.int32)
    if ws is None:
        wsb = lib().tbf16_attn_bwd_ws_bytes(B, H, Hkv, Sq, Sk, D)
        ws = torch.empty(max(wsb, 16), device=dev, dtype=torch.uint8)
    bst = strides3(bias) if bias is not None else None
    launch("tbf16_attn_bwd", dev, ptr(q), ptr(k), ptr(v), ptr(o16), ptr(lse), ptr(dout), ptr(exps_fwd), B, H, Hkv, Sq, Sk,
           D, strides3(q), strides3(k), strides3(v), strides3(dout), ptr(bias), bst, float(scale), int(bool(causal)),
           int(t_do), float(dropout_p), int(seed), ptr(dq), ptr(dk), ptr(dv), ptr(exps_out), ptr(overflow), ptr(gate),
           ptr(ws), ws.numel())
    return dq, dk, dv, exps_out, overflow, ws


def _overflowed(word) -> bool:
    """An attempt's overflow word (non-negative float bits) at or above 65520.0f."""
    return int(word) >= _OVF_BITS


# device-mode backwards not yet checked for a persistent overflow: (event, pinned words)
_pending: list = []
_side: dict = {}


def _side_stream(device: torch.device) -> torch.cuda.Stream:
    """A default-priority stream per device for the overflow words' copies to the host."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    if idx not in _side:
        _side[idx] = torch.cuda.Stream(device=idx)
    return _side[idx]


def check_pending(block: bool = False) -> None:
    """Raises FloatingPointError if a device-mode attention backward overflowed fp16
    in its first attempt and again in its device-side retry (its gradients are then
    not finite). Only backwards the GPU has finished are looked at, unless block."""
    keep, failed = [], False
    for ev, words in _pending:
        if block:
            ev.synchronize()
        elif not ev.query():
            keep.append((ev, words))
            continue
        failed |= _overflowed(words[0]) and _overflowed(words[1])
    _pending[:] = keep
    if failed:
        raise FloatingPointError("tbf16 attention backward overflowed fp16 even after rescaling "
                                 "(its gradients are not finite)")


_warned_capture = False


def queue_overflow_check() -> None:
    """From inside an autograd backward: check every device-mode attention backward
    enqueued so far once the engine has run the whole backward() call, raising
    FloatingPointError from that call. Each attention layer queues one; the first to
    run waits for all pending words (one host sync), the rest find nothing left."""
    global _warned_capture
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        if not _warned_capture:
            _warned_capture = True
            import warnings
            warnings.warn("tbf16: attention backward captured in a HIP graph; the retry runs in the graph, "
                          "but an fp16 overflow that persists through every retry is not reported")
        return
    torch.autograd.Variable._execution_engine.queue_callback(lambda: check_pending(block=True))


def attn_backward(q, k, v, o16, lse, dout, exps_fwd, bias, scale, causal, check=None, attempt_fn=None,
                  dropout_p=0.0, seed=0, head_dim=None):
    """Retry policy of tbf16/autograd.py:173-189: G = t_do - e with t_do = 12 - ceil(log2 D);
    on fp16 overflow t_do -= 8, at most ATTN_RETRIES attempts, then FloatingPointError.
    D is the caller's head dim (head_dim, before any zero padding of q/k/v).
    `attempt_fn` replaces the kernel call (tests inject overflowing attempts)."""
    mode = CHECK_OVERFLOW if check is None else {True: "sync", False: "off"}.get(check, check)
    D = head_dim or q.shape[-1]
    t_do = 12 - math.ceil(math.log2(D))
    args = (q, k, v, o16, lse, dout, exps_fwd, bias, scale, causal)
    if attempt_fn is None and mode in ("device", "deferred") and q.numel() and k.numel():
        if not torch.cuda.is_current_stream_capturing():
            check_pending()  # earlier device-mode backwards the GPU has finished
        words = torch.empty(2, device=q.device, dtype=torch.int32)
        dq, dk, dv, exps_out, _, ws = _attn_backward_once(*args, t_do, dropout_p=dropout_p, seed=seed,
                                                          overflow=words[0:1])
        # the retry, run by the kernels only if the first attempt overflowed
        _attn_backward_once(*args, t_do, dropout_p=dropout_p, seed=seed, overflow=words[1:2], gate=words[0:1],
                            outs=(dq, dk, dv, exps_out), ws=ws)
        if torch.cuda.is_current_stream_capturing():
            # inside a graph capture nothing may leave the captured stream: the retry
            # runs in the graph, the persistent-overflow report is not available
            return dq, dk, dv, exps_out
        # the two words go to pinned host memory on a side stream, off the compute stream
        host = torch.empty(2, dtype=torch.int32, pin_memory=True)
        side = _side_stream(q.device)
        side.wait_stream(torch.cuda.current_stream(q.device))
        with torch.cuda.stream(side):
            host.copy_(words, non_blocking=True)
            ev = torch.cuda.Event()
            ev.record(side)
        words.record_stream(side)
        _pending.append((ev, host))
        return dq, dk, dv, exps_out
    if attempt_fn is not None:
        run = attempt_fn
    else:
        def run(*a):
            return _attn_backward_once(*a, dropout_p=dropout_p, seed=seed)[:5]
    for _ in range(ATTN_RETRIES):
        dq, dk, dv, exps_out, overflow = run(*args, t_do)
        if mode == "off":
            break
        if not _overflowed(overflow.item()):  # host sync, once per attention backward
            break
        t_do -= 8
    else:
        raise FloatingPointError("tbf16 attention backward overflowed fp16 even after rescaling")
    return dq, dk, dv, exps_out


class ScaledSDPAFn(torch.autograd.Function):
    """Fused fp16 attention forward/backward with everything in save_for_backward, so
    activation checkpointing can drop and recompute it (tbf16/autograd.py:149-193)."""

    @staticmethod
    @torch.autocast("cuda", enabled=False)
    def forward(ctx, q, k, v, attn_mask, dropout_p, is_causal, scale, enable_gqa, head_dim=None):
        attention._check_qkv(q, k, v, enable_gqa)
        attention._check_dropout(dropout_p)
        seed = attention.dropout_seed() if dropout_p else 0
        B, H, Sq, D = q.shape
        bias = attention.mask_to_bias(attn_mask, B, H, Sq, k.shape[2], q.device)
        qv, kv, vv = attention._kernel_view(q), attention._kernel_view(k), attention._kernel_view(v)
        sc = (1.0 / math.sqrt(D)) if scale is None else float(scale)
        o, lse, o16, exps = attention.attn_forward(qv, kv, vv, bias, is_causal, sc, v_exp=0, want_lse=True,
                                                   want_o16=True, dropout_p=dropout_p, seed=seed)
        ctx.save_for_backward(qv, kv, vv, o16, lse, exps, bias)
        ctx.args = (sc, bool(is_causal), float(dropout_p), seed, head_dim or D)
        return o

    @staticmethod
    @torch.autocast("cuda", enabled=False)
    def backward(ctx, dout):
        q, k, v, o16, lse, exps, bias = ctx.saved_tensors
        sc, causal, dropout_p, seed, head_dim = ctx.args
        dout = attention._kernel_view(dout.to(torch.bfloat16))
        dq, dk, dv, _ = attn_backward(q, k, v, o16, lse, dout, exps, bias, sc, causal, dropout_p=dropout_p, seed=seed,
                                      head_dim=head_dim)
        if CHECK_OVERFLOW == "device":
            queue_overflow_check()  # raises from this backward() call on a persistent overflow
        return dq, dk, dv, None, None, None, None, None, None


def sdpa(q, k, v, attn_mask=None, dropout_p=0.0, is_causal=False, scale=None, enable_gqa=False):
    """Differentiable bf16 scaled_dot_product_attention on fp16 MFMA (tbf16/autograd.py:196-198).
    Head dims that are not a multiple of 8 are zero-padded around the kernels (the pad
    and the slice are differentiable, so the gradients come back unpadded)."""
    qp, kp, vp, sc, D = attention.pad_head_dim(q, k, v, scale)
    out = ScaledSDPAFn.apply(qp, kp, vp, attn_mask, dropout_p, is_causal, sc, enable_gqa, D)
    return out if out.shape[-1] == D else out[..., :D]


class QKNormRopeFn(torch.autograd.Function):
    """tbf16.qk_norm_rope with its gradients: the norms are computed again in the backward pass from the
    saved inputs."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.how = eps, interleaved
        return norm_rope.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)

    @staticmethod
    def backward(ctx, dyq, dyk):
        if torch.is_grad_enabled():  # create_graph: the gradients have none of their own
            return QKNormRopeFn._once(ctx, dyq, dyk)
        return (*norm_rope.backward(*ctx.saved_tensors, *ctx.how, dyq, dyk, ctx.needs_input_grad[:4]), None, None, None, None, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def _once(ctx, dyq, dyk):
        return QKNormRopeFn.backward(ctx, dyq, dyk)


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps=1e-6, interleaved=False):
    """Differentiable tbf16.qk_norm_rope: gradients of q, k (bf16) and both weights (their own type), sums
    over tokens and heads in fp32 in a fixed order. Tokens of a negative position have no share in
    any. cos, sin and positions are constants. Can be captured into a graph with its backward pass, as
    long as no autograd graph made outside of the capture still holds the same leaves: torch would
    add up their gradients on the stream that one came from."""
    if cos.requires_grad or sin.requires_grad:
        raise ValueError("tbf16.autograd.qk_norm_rope: no gradients of cos and sin")
    return QKNormRopeFn.apply(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
