"""The operators of a serving step, as cases that can be timed and compared.

A case is a dict of plain values; `prepare` makes what a program has in hand before
the call, `run` is one pass, `exact` the same results in 64 bits, `work` the bytes and
operations a pass cannot do without. With `own` set, `run` makes the calls of tbf16's
public entry points; otherwise it computes the same in elementary torch operations.

Kinds:
  attend  attention of one new token per sequence over a paged key/value cache
          (tbf16.paged_sdpa)
  write   new tokens' keys and values into such a cache (tbf16.paged_write)
  linear  a linear in 8-bit integers, one scale per token and per output channel
          (tbf16.int8_linear on a weight prepared once)
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"


def _tbf16():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "turing-bf16_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tbf16
    return tbf16


def listed():
    return [
        # one conversation of a few hundred tokens, a head of keys per query head: latency counts
        {"name": "attend_one", "kind": "attend", "B": 1, "H": 16, "Hkv": 16, "D": 128, "page": 16, "shortest": 700,
         "longest": 700},
        # a serving batch of requests of every age, four query heads to a key head
        {"name": "attend_batch", "kind": "attend", "B": 32, "H": 32, "Hkv": 8, "D": 128, "page": 16, "shortest": 1,
         "longest": 4096},
        # one very long document
        {"name": "attend_long", "kind": "attend", "B": 1, "H": 32, "Hkv": 8, "D": 128, "page": 64, "shortest": 131072,
         "longest": 131072},
        # a full server: many requests, places of the batch that nobody has among them (length 0)
        {"name": "attend_many", "kind": "attend", "B": 128, "H": 32, "Hkv": 8, "D": 128, "page": 16, "shortest": 0,
         "longest": 8192},
        # a small model with an odd head dim, group and page size
        {"name": "attend_odd", "kind": "attend", "B": 7, "H": 20, "Hkv": 4, "D": 80, "page": 48, "shortest": 3,
         "longest": 2999},
        # a decoding batch's one token each
        {"name": "write_decode", "kind": "write", "T": 64, "Hkv": 8, "D": 128, "page": 16, "run": 1, "pad": 0},
        # prompts of 2048 tokens, the batch padded
        {"name": "write_prefill", "kind": "write", "T": 8192, "Hkv": 8, "D": 128, "page": 16, "run": 2048, "pad": 37},
        # one token through an MLP up-projection
        {"name": "linear_1", "kind": "linear", "M": 1, "K": 2560, "N": 10240, "bias": False},
        # sixteen sequences decoding together through the same layer
        {"name": "linear_16", "kind": "linear", "M": 16, "K": 2560, "N": 10240, "bias": False},
        # a short prompt through a square projection
        {"name": "linear_256", "kind": "linear", "M": 256, "K": 4096, "N": 4096, "bias": True},
        # an odd number of tokens through a vocabulary head with an added token
        {"name": "linear_odd", "kind": "linear", "M": 100, "K": 1000, "N": 32001, "bias": True},
        # a long prompt
        {"name": "linear_4096", "kind": "linear", "M": 4096, "K": 4096, "N": 4096, "bias": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer width: mostly a multiple of 64, sometimes only of 8."""
    m = rng.choice((64, 64, 64, 8))
    return max(lo, _log(rng, lo, hi) // m * m)


def draw(rng):
    while True:
        kind = rng.choice(("attend", "attend", "attend", "write", "linear", "linear", "linear"))
        if kind == "attend":
            Hkv = rng.choice((1, 2, 4, 5, 8, 8, 16))
            c = {"kind": kind, "B": _log(rng, 1, 128), "H": Hkv * rng.choice((1, 1, 2, 4, 4, 5, 8, 16)), "Hkv": Hkv,
                 "D": rng.choice((64, 64, 80, 96, 128, 128, 128, 256)), "page": rng.choice((8, 16, 16, 16, 32, 48, 64, 128)),
                 "longest": _log(rng, 1, 131072)}
            c["shortest"] = rng.choice((0, 1, c["longest"] // 2, c["longest"])) if c["B"] > 1 else c["longest"]
            if c["H"] <= 64 and work(c)["bytes"] <= 2.1e9:
                return c
        elif kind == "write":
            run = rng.choice((1, 1, _log(rng, 2, 4096)))
            c = {"kind": kind, "T": run * _log(rng, 1, 128), "Hkv": rng.choice((1, 2, 4, 8, 8, 16)),
                 "D": rng.choice((64, 80, 96, 128, 128, 256)), "page": rng.choice((8, 16, 16, 32, 48, 64, 128)), "run": run}
            c["pad"] = rng.choice((0, 0, rng.randrange(0, c["T"])))
            if c["T"] * c["Hkv"] * c["D"] <= 1 << 25:
                return c
        else:
            c = {"kind": kind, "M": _log(rng, 1, 8192), "K": _width(rng, 256, 8192), "N": _width(rng, 256, 16384),
                 "bias": rng.random() < 0.5}
            if rng.random() < 0.15:
                c["N"] += rng.randrange(1, 8)
            if 2 * c["M"] * c["K"] * c["N"] <= 1.38e11 and c["K"] * c["N"] <= 1 << 26:
                return c


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _lengths(case):
    """The sequences' lengths, evenly spread between the shortest and the longest."""
    B, lo, hi = case["B"], case["shortest"], case["longest"]
    return [hi if B == 1 else lo + (hi - lo) * i // (B - 1) for i in range(B)]


def _inputs(case, seed):
    g = _gen(seed)
    if case["kind"] == "attend":
        B, H, Hkv, D, page = (case[n] for n in ("B", "H", "Hkv", "D", "page"))
        lengths = _lengths(case)
        lengths = [lengths[i] for i in torch.randperm(B, generator=g, device=DEV).tolist()]
        need = [-(-n // page) for n in lengths]
        pages = sum(need) + 3  # a few that nobody has
        order = torch.randperm(pages, generator=g, device=DEV).int()
        table = torch.zeros(B, max(max(need), 1), dtype=torch.int32, device=DEV)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        # query heads from even to peaked weights, value heads of several sizes
        q = (_randn(g, B, H, D) * torch.exp2(2.0 * torch.rand(B, H, 1, generator=g, device=DEV))).bfloat16()
        k = _randn(g, pages, Hkv, page, D).bfloat16()
        v = (_randn(g, pages, Hkv, page, D) * torch.exp2(torch.randint(-4, 5, (Hkv, 1, 1), generator=g, device=DEV))).bfloat16()
        return {"q": q, "k_cache": k, "v_cache": v, "table": table, "lengths": lengths}
    if case["kind"] == "write":
        T, Hkv, D, page, run = (case[n] for n in ("T", "Hkv", "D", "page", "run"))
        seqs, each = -(-T // run), -(-run // page) + 1
        order = torch.randperm(seqs * each + 3, generator=g, device=DEV)
        t = torch.arange(T, device=DEV)
        start = torch.randint(0, page, (seqs,), generator=g, device=DEV)
        pos = start[t // run] + t % run
        slots = order[t // run * each + pos // page] * page + pos % page
        slots[T - case["pad"]:] = -1
        kv = _randn(g, T, 2, Hkv, D).bfloat16()  # both halves of one projection's output
        k = _randn(g, seqs * each + 3, Hkv, page, D).bfloat16()
        v = _randn(g, seqs * each + 3, Hkv, page, D).bfloat16()
        return {"k": kv[:, 0], "v": kv[:, 1], "slots": slots.int(), "k_cache": k, "v_cache": v}
    M, K, N = case["M"], case["K"], case["N"]
    x = _randn(g, M, K)
    # one channel in a hundred ten times the others, as activations have them
    x *= torch.where(torch.rand(K, generator=g, device=DEV) < 0.01, 10.0, 1.0)
    return {"x": x.bfloat16(), "w": (_randn(g, N, K) * K ** -0.5).bfloat16(),
            "b": _randn(g, N).bfloat16() if case["bias"] else None}


def _codes(x):
    """Rows as 8-bit codes rint(127 x / max |x|) and their scales max |x| / 127. The
    quotients are taken in 64 bits: many of a row's values lie on a border between two codes."""
    top = x.abs().amax(-1, keepdim=True).double()
    code = torch.round(127.0 * x.double() / torch.where(top > 0, top, 1.0))
    return code.to(torch.int8), (top / 127.0).float().squeeze(-1)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] == "attend":
        s["lengths_gpu"] = torch.tensor(s["lengths"], dtype=torch.int32, device=DEV)
    elif case["kind"] == "linear":
        w = s.pop("w")  # once per weight, kept by the program
        s["w8"], s["ws"] = _tbf16().prepare_weight_i8(w) if own else _codes(w)
    return s


def _attend(s):
    q, out = s["q"].float(), torch.zeros_like(s["q"])
    B, H, D = q.shape
    Hkv, page = s["k_cache"].shape[1:3]
    for b, n in enumerate(s["lengths"]):
        if n == 0:
            continue
        pages = s["table"][b, :-(-n // page)].long()
        k = s["k_cache"][pages].float().transpose(0, 1).reshape(Hkv, -1, D)[:, :n]
        v = s["v_cache"][pages].float().transpose(0, 1).reshape(Hkv, -1, D)[:, :n]
        logits = torch.matmul(q[b].view(Hkv, H // Hkv, D), k.transpose(1, 2)) * D ** -0.5
        p = torch.exp(logits - logits.amax(-1, keepdim=True))
        out[b] = (torch.matmul(p, v) / p.sum(-1, keepdim=True)).view(H, D).bfloat16()
    return out


def _write(s):
    page = s["k_cache"].shape[2]
    keep = s["slots"] >= 0
    slots = s["slots"][keep].long()
    s["k_cache"][slots // page, :, slots % page] = s["k"][keep]
    s["v_cache"][slots // page, :, slots % page] = s["v"][keep]
    return s["k_cache"], s["v_cache"]


def _linear(s):
    x8, sx = _codes(s["x"])
    y = (x8.float() @ s["w8"].float().t()) * sx[:, None] * s["ws"]
    if s["b"] is not None:
        y = y + s["b"].float()
    return y.bfloat16()


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"attend": _attend, "write": _write, "linear": _linear}[kind](state)
    tbf16 = _tbf16()
    if kind == "attend":
        return tbf16.paged_sdpa(state["q"], state["k_cache"], state["v_cache"], state["table"], state["lengths_gpu"])
    if kind == "write":
        tbf16.paged_write(state["k_cache"], state["v_cache"], state["k"], state["v"], state["slots"])
        return state["k_cache"], state["v_cache"]
    return tbf16.int8_linear(state["x"], state["w8"], state["ws"], state["b"])


def work(case):
    if case["kind"] == "attend":
        B, H, Hkv, D, page = (case[n] for n in ("B", "H", "Hkv", "D", "page"))
        keys = sum(_lengths(case))
        return {"bytes": 4 * Hkv * D * keys + 4 * B * H * D + 4 * B + 4 * sum(-(-n // page) for n in _lengths(case)),
                "flops": 4 * H * D * keys}
    if case["kind"] == "write":
        return {"bytes": 8 * (case["T"] - case["pad"]) * case["Hkv"] * case["D"] + 4 * case["T"], "flops": 0}
    M, K, N = case["M"], case["K"], case["N"]
    return {"bytes": 2 * M * K + N * K + 4 * N + (2 * N if case["bias"] else 0) + 2 * M * N, "flops": 2 * M * K * N}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "attend":
        B, H, Hkv, D, page = (case[n] for n in ("B", "H", "Hkv", "D", "page"))
        out = torch.zeros(B, H, D, dtype=torch.float64, device=DEV)
        for b, n in enumerate(s["lengths"]):
            if n:
                j = torch.arange(n, device=DEV)
                at, off = s["table"][b].long()[j // page], j % page
                for h in range(Hkv):
                    heads = slice(h * (H // Hkv), (h + 1) * (H // Hkv))
                    k, v = s["k_cache"][at, h, off].double(), s["v_cache"][at, h, off].double()
                    out[b, heads] = torch.softmax(s["q"][b, heads].double() @ k.t() / math.sqrt(D), -1) @ v
        return out
    if case["kind"] == "write":
        taken = torch.nonzero(s["slots"] >= 0).squeeze(1)
        for cache, rows in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])):
            flat = cache.transpose(1, 2).flatten(0, 1)  # a copy, one row a slot
            flat.index_copy_(0, s["slots"][taken].long(), rows[taken])
            cache.copy_(flat.unflatten(0, (-1, case["page"])).transpose(1, 2))
        return s["k_cache"].double(), s["v_cache"].double()

    def rows(t):  # (codes, scales) by the definition
        t = t.double()
        top = t.abs().max(1, keepdim=True).values
        return torch.where(top > 0, t * 127.0 / top, 0.0).round(), top / 127.0

    (x8, sx), (w8, sw) = rows(s["x"]), rows(s["w"])
    y = torch.mm(x8, w8.t()) * (sx * sw.t())
    return y if s["b"] is None else y + s["b"].double()
