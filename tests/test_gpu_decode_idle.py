"""A decoding loop some of whose places have no new token in a step: paged_advance packs the tokens, the attention's rows
are sequences, and the tokens' slots and positions are brought into the order of sequences between them. Eagerly and
from one captured graph, against 64 bits."""
import random

import pytest
import torch

import tbf16

from _operators64 import norm_rope64
from test_gpu_decode_loop import B, D, H, PAGE, PAGES, PREFIX, Hkv, Server, attend64, gen

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def step(s, room):
    """One step of up to one token a sequence, of `room` together."""
    slots, positions, starts = tbf16.paged_advance(s.table, s.lengths, s.counts, s.free, s.n_free, PAGE, room, s.far_length)
    new, at = starts[1:] > starts[:-1], starts[:-1].clamp(max=room - 1)
    slots, positions = torch.where(new, slots[at], -1), torch.where(new, positions[at], -1)
    q, k = tbf16.qk_norm_rope(s.qkv[:, :H], s.qkv[:, H:H + Hkv], *s.w, s.cos, s.sin, positions)
    tbf16.paged_write(s.k, s.v, k, s.qkv[:, H + Hkv:], slots)
    return tbf16.paged_sdpa_prefix(q, s.k, s.v, s.far[0], s.far_length, s.table, s.lengths), positions, slots


@pytest.mark.parametrize("room", [B, B - 2, B + 3])
@pytest.mark.parametrize("captured", [False, True])
def test_idle_places(dev, captured, room):
    s = Server(dev)
    g, r = gen(7), random.Random(room)
    qkv = torch.randn(PREFIX, H + 2 * Hkv, D, generator=g).to(BF).to(dev)
    _, k, _, _, _ = s.tokens(qkv, s.far, s.far_length, torch.tensor([PREFIX], dtype=torch.int32, device=dev), None)
    prefix = list(zip(k.cpu(), qkv[:, H + Hkv:].cpu()))
    state = s.table, s.lengths, s.free, s.n_free, s.k, s.v
    run = lambda: step(s, room)  # noqa: E731
    if captured:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        keep = [t.clone() for t in state]
        with torch.cuda.stream(side):
            step(s, room)
        torch.cuda.synchronize()
        for t, old in zip(state, keep):
            t.copy_(old)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(s, room)

        def run():
            graph.replay()
            return out
    own = [[] for _ in range(B)]
    for _ in range(40):
        # a place: idle, a token, or a request that ends (its pages go back before the others' come)
        counts = [r.choice((0, 1, 1, 1)) if r.random() < 0.95 else -len(own[b]) for b in range(B)]
        s.counts.copy_(torch.tensor(counts, dtype=torch.int32))
        s.qkv.copy_((torch.randn(B, H + 2 * Hkv, D, generator=g) * 2).to(BF))
        o, positions, slots = run()
        torch.cuda.synchronize()
        asked = 0
        for b, c in enumerate(counts):
            if c < 0:
                own[b] = []
            asked += c > 0
            new = c > 0 and asked <= room
            assert positions[b].item() == (PREFIX + len(own[b]) if new else -1) and (slots[b].item() >= 0) == new
            if not new:
                continue
            at = slots[b].long()
            k, v = (t[at // PAGE, :, at % PAGE].cpu() for t in (s.k, s.v))
            k64, bound = norm_rope64(s.qkv[b:b + 1, H:H + Hkv], s.w[1], s.cos, s.sin, positions[b:b + 1])
            assert ((k.double() - k64[0]).abs() <= bound[0]).all() and torch.equal(v, s.qkv[b, H + Hkv:].cpu())
            own[b].append((k, v))
            q, _ = tbf16.qk_norm_rope(s.qkv[b:b + 1, :H], s.qkv[b:b + 1, H:H + Hkv], *s.w, s.cos, s.sin, positions[b:b + 1])
            o64, top = attend64(s, q[0].cpu(), b, prefix + own[b])
            # half a bf16 step, and what fp32 logits of up to 64 |q k| <= 2^9 may be off
            assert ((o[b].cpu().double() - o64).abs() <= 2.0 ** -8 * o64.abs() + 2.0 ** -10 * top).all()
        assert s.lengths.tolist() == [len(t) for t in own]
        assert s.n_free.item() == PAGES - -(-PREFIX // PAGE) - sum(-(-len(t) // PAGE) for t in own)
