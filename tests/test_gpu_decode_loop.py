"""The operators around the paged cache together, as a serving loop runs them: pages, norm and rotation,
cache writes and attention behind a shared prefix, step by step, some requests ending and others coming, eagerly
and from one captured graph, against the same in 64 bits."""
import pytest
import torch

import tbf16

from _operators64 import norm_rope64

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
H, Hkv, D, R, PAGE, PAGES, B, WIDE, PREFIX = 8, 2, 64, 32, 16, 64, 5, 6, 40


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rope(dev):
    a = torch.arange(400, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    return a.cos().float().to(dev), a.sin().float().to(dev)


class Server:
    """The state a program keeps on the device, and one decoding step of one token a sequence."""

    def __init__(self, dev):
        i32 = lambda *s, v=0: torch.full(s, v, dtype=torch.int32, device=dev)  # noqa: E731
        self.k, self.v = (torch.full((PAGES, Hkv, PAGE, D), float("nan"), dtype=BF, device=dev) for _ in "kv")
        self.table, self.lengths, self.counts = i32(B, WIDE, v=-1), i32(B), i32(B)
        self.free = torch.randperm(PAGES, generator=gen(1)).int().to(dev)
        self.n_free, self.far, self.far_length = i32(1, v=PAGES), i32(1, 4, v=-1), i32(1)
        self.w = [(1 + 0.2 * torch.randn(D, generator=gen(2 + i))).to(BF).to(dev) for i in range(2)]
        self.cos, self.sin = rope(dev)
        self.qkv = torch.zeros(B, H + 2 * Hkv, D, dtype=BF, device=dev)

    def tokens(self, qkv, table, lengths, counts, prefix):
        """New tokens' heads into the cache; (q, k, positions, slots, starts)."""
        slots, positions, starts = tbf16.paged_advance(table, lengths, counts, self.free, self.n_free, PAGE, qkv.shape[0], prefix)
        q, k = tbf16.qk_norm_rope(qkv[:, :H], qkv[:, H:H + Hkv], *self.w, self.cos, self.sin, positions)
        tbf16.paged_write(self.k, self.v, k, qkv[:, H + Hkv:], slots)
        return q, k, positions, slots, starts

    def step(self):
        q, _, positions, slots, _ = self.tokens(self.qkv, self.table, self.lengths, self.counts, self.far_length)
        o = tbf16.paged_sdpa_prefix(q, self.k, self.v, self.far[0], self.far_length, self.table, self.lengths)
        return o, positions, slots


def attend64(server, q, b, kv):
    """o of sequence b from the keys and values that its tokens were given, in 64 bits."""
    k, v = (torch.stack([t[i] for t in kv]).double() for i in range(2))  # (n, Hkv, D)
    o = torch.empty(H, D, dtype=torch.float64)
    for h in range(H):
        p = torch.softmax(q[h].double() @ k[:, h // (H // Hkv)].t() * D ** -0.5, -1)
        o[h] = p @ v[:, h // (H // Hkv)]
    return o, v.abs().amax()


@pytest.mark.parametrize("captured", [False, True])
def test_decoding_with_a_shared_prefix(dev, captured):
    s = Server(dev)
    # the prefix: a sequence of its own, whose table the others' calls take
    g = gen(7)
    qkv = torch.randn(PREFIX, H + 2 * Hkv, D, generator=g).to(BF).to(dev)
    _, k, positions, slots, _ = s.tokens(qkv, s.far, s.far_length, torch.tensor([PREFIX], dtype=torch.int32, device=dev), None)
    assert positions.tolist() == list(range(PREFIX)) and (slots >= 0).all() and s.far_length.item() == PREFIX
    prefix = list(zip(k.cpu(), qkv[:, H + Hkv:].cpu()))
    own = [[] for _ in range(B)]
    # lengths at which requests have to end; the counts of a step are all 0 or 1: a token's row is its sequence's
    ends = {0: 20, 1: 7, 2: 33, 3: 12, 4: 90}
    run = s.step
    if captured:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        keep = [t.clone() for t in (s.table, s.lengths, s.free, s.n_free, s.k, s.v)]
        with torch.cuda.stream(side):
            s.step()
        torch.cuda.synchronize()
        for t, old in zip((s.table, s.lengths, s.free, s.n_free, s.k, s.v), keep):
            t.copy_(old)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = s.step()

        def run():
            graph.replay()
            return out
    none = torch.zeros(B, dtype=torch.int32, device=dev)
    for step in range(40):
        gone = [b for b in range(B) if len(own[b]) >= ends[b]]
        if gone:  # requests that end give their pages back, new ones take their places
            back = torch.tensor([-len(own[b]) if b in gone else 0 for b in range(B)], dtype=torch.int32, device=dev)
            tbf16.paged_advance(s.table, s.lengths, back, s.free, s.n_free, PAGE, 0)
            for b in gone:
                own[b] = []
            assert (s.table[gone] == -1).all()
        s.counts.copy_(none + 1)
        s.qkv.copy_((torch.randn(B, H + 2 * Hkv, D, generator=g) * 2).to(BF))
        o, positions, slots = run()
        torch.cuda.synchronize()
        assert positions.tolist() == [PREFIX + len(own[b]) for b in range(B)]
        used = [i for row, n in zip(s.table.tolist(), s.lengths.tolist()) for i in row[:-(-n // PAGE)]]
        used += s.far[0, :-(-PREFIX // PAGE)].tolist()
        assert len(set(used)) == len(used) == PAGES - s.n_free.item() and min(used) >= 0
        # what the step's own norms and rotations gave, from the cache; then the attention over all of it
        at = slots.long()
        k, v = (c[at // PAGE, :, at % PAGE].cpu() for c in (s.k, s.v))
        k64, bound = norm_rope64(s.qkv[:, H:H + Hkv], s.w[1], s.cos, s.sin, positions)
        assert ((k.double() - k64).abs() <= bound).all() and torch.equal(v, s.qkv[:, H + Hkv:].cpu())
        q, _ = tbf16.qk_norm_rope(s.qkv[:, :H], s.qkv[:, H:H + Hkv], *s.w, s.cos, s.sin, positions)
        for b in range(B):
            own[b].append((k[b], v[b]))
            o64, top = attend64(s, q[b].cpu(), b, prefix + own[b])
            # half a bf16 step, and what fp32 logits of up to 64 |q k| <= 2^9 and weights of 16 bits may be off
            assert ((o[b].cpu().double() - o64).abs() <= 2.0 ** -8 * o64.abs() + 2.0 ** -10 * top).all()
    back = -s.lengths
    tbf16.paged_advance(s.table, s.lengths, back, s.free, s.n_free, PAGE, 0)
    assert s.n_free.item() == PAGES - -(-PREFIX // PAGE) and not s.lengths.any()
