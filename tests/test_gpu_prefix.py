"""paged_sdpa_prefix on the GPU against 64 bits (tolerances: tests/_operators64.py)."""
import random

import pytest
import torch

import tbf16

from _operators64 import prefix_sdpa64

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make(dev, prefix, lengths, H, Hkv, D, page, seed=0, spare=3, kscale=1.0, junk=float("nan")):
    """(q, k_cache, v_cache, prefix_table, prefix_length, table, lengths), pages in random order; every row that
    no position uses holds `junk`, unused table entries point anywhere."""
    g = gen(seed)
    up = lambda n: -(-max(n, 0) // page)  # noqa: E731
    need = [up(prefix), *map(up, lengths)]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g)
    table = torch.randint(0, pages, (len(lengths), max(need[1:] + [1])), generator=g, dtype=torch.int32)
    far = torch.randint(0, pages, (need[0] + 2,), generator=g, dtype=torch.int32)
    k = (torch.randn(pages, Hkv, page, D, generator=g) * kscale).to(BF)
    v = (torch.randn(pages, Hkv, page, D, generator=g) * torch.exp2(torch.randint(-3, 4, (Hkv, 1, 1), generator=g))).to(BF)
    used = torch.zeros(pages, page, dtype=torch.bool)
    at = 0
    for i, (n, p) in enumerate(zip((prefix, *lengths), need)):
        mine = order[at:at + p]
        at += p
        (far if i == 0 else table[i - 1])[:p] = mine.int()
        j = torch.arange(max(n, 0))
        used[mine[j // page], j % page] = True
    for c in (k, v):
        c.masked_fill_(~used[:, None, :, None], junk)
    q = (torch.randn(len(lengths), H, D, generator=g) * 2).to(BF)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return [t.to(dev) for t in (q, k, v, far, i32([prefix]), table, i32(lengths))]


def check(a, scale=None, only=None):
    o = tbf16.paged_sdpa_prefix(*a, scale=scale)
    assert o.shape == a[0].shape and o.dtype == BF and o.is_contiguous()
    q, k, v, far, n, table, lengths = a
    got = o
    if only is not None:
        q, table, lengths, got = q[only], table[only], lengths[only], o[only]
    ref, bound = prefix_sdpa64(q, k, v, far, n.item(), table, lengths, scale)
    finite = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got.cpu()), finite)
    err = (got.cpu().double() - ref).abs()[finite]
    assert (err <= bound[finite]).all(), (err - bound[finite]).max()
    return o


SHAPES = [  # H, Hkv, D, page, prefix, lengths
    (1, 1, 8, 1, 1, [0]),
    (1, 1, 64, 16, 0, [0, 1, 5]),
    (4, 4, 64, 16, 33, [1, 0, 2]),
    (16, 16, 128, 16, 700, [1, 64, 17, 30]),
    (8, 2, 128, 16, 64, [1, 63, 64, 65, 100, 127, 0]),
    (32, 8, 128, 16, 1000, list(range(0, 320, 10))),
    (20, 4, 80, 48, 2999, [0, 3, 47, 48, 49, 333, 1, 2, 100, 200, 300, 7, 8]),
    (6, 3, 72, 24, 129, [25, 200, 0, 777]),
    (12, 12, 96, 7, 65, [1, 6, 7, 8, 333]),
    (16, 1, 256, 16, 300, [5, 300]),
    (16, 1, 256, 16, 191, [5, 30, 3, 0]),
    (16, 2, 256, 64, 1025, [1] * 9),
    (8, 4, 200, 16, 127, [3, 7, 0, 90]),
    (40, 1, 256, 8, 65, [9] * 8),
    (64, 1, 128, 16, 250, [1, 250, 7]),
    (71, 1, 64, 16, 400, [33, 400, 3]),
    (130, 2, 64, 100, 257, [40, 257]),
    (5, 1, 40, 16, 31, [18, 1]),
    (4, 1, 128, 128, 20000, [300]),
    (3, 3, 64, 16, 32, [5] * 40),
    (2, 1, 104, 5, 95, [0] * 100),
    (32, 8, 64, 16, 130, [b % 40 for b in range(70)]),
    (32, 4, 128, 32, 513, [b * 7 % 90 for b in range(75)]),
    (2, 2, 128, 3, 500, [2000, 1]),
]


@pytest.mark.parametrize("H,Hkv,D,page,prefix,lengths", SHAPES)
def test_shapes(dev, H, Hkv, D, page, prefix, lengths):
    check(make(dev, prefix, lengths, H, Hkv, D, page, seed=H + D + page))


@pytest.mark.parametrize("seed", range(40))
def test_random_batches(dev, seed):
    r = random.Random(seed)
    B, Hkv, D, page = r.choice((1, 2, 3, 9, 40, 150)), r.choice((1, 2, 5)), r.choice((8, 64, 72, 128, 248)), r.choice((1, 5, 16, 33, 64))
    top = r.choice((33, 200)) if B > 9 else r.choice((40, 700, 3000))
    prefix = r.choice((0, 1, r.randrange(1, 200), r.randrange(1, 3000), 64 * r.randrange(1, 30)))
    lengths = [r.choice((0, 1, r.randrange(top), 32 * r.randrange(1, top // 32 + 1))) for _ in range(B)]
    a = make(dev, prefix, lengths, Hkv * r.choice((1, 3, 4, 8)), Hkv, D, page, seed=seed)
    check(a)
    wide = torch.full((B, a[5].shape[1] + 5000 // page), -1, dtype=torch.int32, device=dev)  # room for long ones
    wide[:, :a[5].shape[1]] = a[5]
    far = torch.cat((a[3], torch.full((4000 // page,), -1, dtype=torch.int32, device=dev)))
    check([*a[:3], far, a[4], wide, a[6]])


def test_many_pages_of_one(dev):
    """More pages in a block's share than it holds at a time; one split, many row tiles."""
    B, H, Hkv, D = 1100, 32, 8, 64
    a = make(dev, 5000, [b % 3 for b in range(B)], H, Hkv, D, 1, seed=3)
    check(a, only=torch.tensor([0, 1, 2, 511, 512, 777, 1098, 1099]))
    a = make(dev, 9000, [b % 3 for b in range(17)], 128, 1, 128, 1, seed=4)
    check(a)


def test_very_many_sequences(dev):
    B = 40000
    a = make(dev, 100, [0] * 5, 2, 1, 8, 4, seed=1)
    g = gen(2)
    a[0] = torch.randn(B, 2, 8, generator=g).to(BF).to(dev)
    a[5] = a[3][torch.randint(0, 25, (B, 2), generator=g)].contiguous()
    a[6] = torch.randint(0, 9, (B,), generator=g, dtype=torch.int32).to(dev)
    check(a, only=torch.cat((torch.arange(40), torch.randint(0, B, (60,), generator=g), torch.arange(B - 40, B))))


@pytest.mark.parametrize("scale", [0.0, -0.5, 3.0, 1e-3])
def test_scales(dev, scale):
    check(make(dev, 90, [90, 17, 0], 4, 2, 64, 16, seed=3), scale)
    check(make(dev, 200, [3] * 50, 8, 2, 128, 16, seed=3), scale)


@pytest.mark.parametrize("kscale", [30.0, 1e4, 1e-4])
def test_peaked_and_flat(dev, kscale):
    check(make(dev, 1500, [40, 700, 0], 8, 2, 64, 16, seed=5, kscale=kscale))
    check(make(dev, 600, [40] * 40, 8, 2, 128, 16, seed=5, kscale=kscale))


@pytest.mark.parametrize("order", ["rising", "falling"])
def test_maximum_that_moves(dev, order):
    """Logits that grow by less and by more than the steps the kernel's maximum follows in."""
    for step in (0.01, 0.2, 3.0, 40.0):
        a = make(dev, 1000, [50, 3], 4, 1, 64, 16, seed=6)
        q, k, far = a[0], a[1], a[3]
        q.copy_(torch.eye(64)[0] * 8)
        j = torch.arange(1000)
        x = (j if order == "rising" else 999 - j).float() * step
        k[far.cpu()[j // 16].long(), 0, j % 16, 0] = x.to(BF).to(dev)
        check(a)


def test_odd_tables(dev):
    """Entries that name no page, lengths past the tables and below zero, an empty prefix table."""
    a = make(dev, 300, [40, 100, 0, 64], 8, 2, 64, 16, seed=7)
    for lengths, prefix in (([40, -5, 3, 10 ** 9], 300), ([0, 0, 0, 0], -3), ([5, 6, 7, 0], 2 ** 31 - 1)):
        b = [t.clone() for t in a]
        b[1].nan_to_num_(0.5)
        b[2].nan_to_num_(0.25)
        b[3][[2, 7]] = torch.tensor([-1, 10 ** 6], dtype=torch.int32, device=dev)
        b[5][1, 0] = b[1].shape[0]
        b[4].fill_(prefix)
        b[6].copy_(torch.tensor(lengths, dtype=torch.int32))
        check(b)
    b[3] = b[3][:0]
    check(b)
    b[3] = a[3] * 0 - 1  # a prefix of no page at all
    check(b)
    b[5] = b[5][:, :0]
    assert not check(b).any()
    c = [t[:0] if i in (1, 2) else t for i, t in enumerate(b)]
    assert not tbf16.paged_sdpa_prefix(*c).any()
    assert tbf16.paged_sdpa_prefix(a[0][:0], *a[1:5], a[5][:0], a[6][:0]).shape == (0, 8, 64)


def test_layouts(dev):
    a = make(dev, 333, [40, 100, 0, 64], 8, 2, 72, 16, seed=8)
    want = check(a)
    q, k, v, far, n, table, lengths = a
    cache = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]
    both = torch.stack((k, v), 2)  # (pages, Hkv, 2, page, D): K and V of a head side by side
    odd_q = torch.empty(4, 8, 73, dtype=BF, device=dev)[..., 1:].copy_(q)
    out_q = torch.empty(8, 4, 72, dtype=BF, device=dev).transpose(0, 1).copy_(q)
    far2 = torch.stack((far, far), 1)[:, 0]
    table2 = torch.stack((table, table), 2)[..., 0]
    for b in ((q, *cache, far, n, table, lengths), (q, both[:, :, 0], both[:, :, 1], far, n, table, lengths),
              (odd_q, k, v, far2, n[0], table2, lengths), (out_q, k, v, far, n, table, torch.stack((lengths, lengths), 1)[:, 0])):
        assert torch.equal(tbf16.paged_sdpa_prefix(*b), want)


def test_same_as_long_tables(dev):
    """A prefix of whole pages: paged_sdpa on tables that begin with it, each within its tolerance."""
    a = make(dev, 320, [40, 100, 0, 64], 8, 2, 128, 16, seed=9)
    check(a)
    q, k, v, far, n, table, lengths = a
    long = torch.cat((far[:20].expand(4, 20), table), 1)
    o = tbf16.paged_sdpa(q, k, v, long, lengths + 320)
    ref, bound = prefix_sdpa64(q, k, v, far, 320, table, lengths)
    assert ((o.cpu().double() - ref).abs() <= bound).all()


@pytest.mark.parametrize("B,H,D", [(3, 4, 64), (40, 8, 128), (200, 8, 64), (5, 4, 256)])
def test_infinite_and_nan_keys_and_values(dev, B, H, D):
    a = make(dev, 200, [20] * B, H, 2, D, 16, seed=10)
    q, k, v, far = a[0], a[1], a[2], a[3].cpu().long()
    v[far[3], 0, 5, 7] = float("inf")
    v[far[9], 1, 2, 3] = float("-inf")
    o = check(a)
    assert (o[:, :H // 2, 7] == float("inf")).all() and (o[:, H // 2:, 3] == float("-inf")).all()
    v[far[3], 0, 5, 7] = 3e38  # the largest values: sums have room
    v[far[9], 1, 2, 3] = -3e38
    check(a)
    k[far[4], 0, 1, 0] = float("nan")
    o = tbf16.paged_sdpa_prefix(*a)
    assert torch.isnan(o[:, :H // 2]).all() and torch.isfinite(o[:, H // 2:]).all()
    k[far[4], 0, 1, 0] = 0.5
    # logits of minus infinity alone: as a softmax, NaN; beside finite ones: left out
    q[0] = 0
    q[0, :, 0] = 1
    k[far[0], :, 0, 0] = float("-inf")
    check(a)
    one = [*a[:4], torch.ones_like(a[4]), a[5], a[6] * 0]
    assert torch.isnan(tbf16.paged_sdpa_prefix(*one)[0]).all()


def test_far_offsets(dev):
    """A cache of more than 2^31 elements."""
    pages, Hkv, page, D = 135000, 8, 16, 128
    cache = torch.empty(pages, Hkv, page, D, dtype=BF, device=dev)
    a = make(dev, 100, [30, 17], 16, Hkv, D, page, seed=11, spare=0)
    n = a[1].shape[0]
    move = torch.cat((torch.tensor([pages - 1, 0, 131073]), torch.randint(1, 131072, (n,), generator=gen(1))))[:n].to(dev)
    cache[move] = a[1]
    b = [a[0], cache, cache, move[a[3].long()].int(), a[4], move[a[5].long()].int(), a[6]]
    o = tbf16.paged_sdpa_prefix(*b)
    ref, bound = prefix_sdpa64(a[0], a[1], a[1], a[3], 100, a[5], a[6])
    assert ((o.cpu().double() - ref).abs() <= bound).all()


def test_streams_and_repeats(dev):
    """Two calls at once on two streams, each with its own workspace; the same bits every time."""
    a = make(dev, 3000, [b * 9 % 300 for b in range(40)], 32, 8, 128, 16, seed=12)
    b = make(dev, 1000, [b * 7 % 200 for b in range(30)], 16, 4, 128, 16, seed=13)
    wa, wb = check(a), check(b)
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(s):
            oa = tbf16.paged_sdpa_prefix(*a)
        with torch.cuda.stream(t):
            ob = tbf16.paged_sdpa_prefix(*b)
        torch.cuda.synchronize()
        assert torch.equal(oa, wa) and torch.equal(ob, wb)


@pytest.mark.parametrize("capacity", [80, 3000])
def test_graph(dev, capacity):
    """Captured once, replayed with other lengths and tables; short and long own tables."""
    a = make(dev, 500, [60] * 9, 8, 2, 64, 16, seed=14)
    a[5] = torch.cat((a[5], torch.zeros(9, (capacity - 64) // 16, dtype=torch.int32, device=dev)), 1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        tbf16.paged_sdpa_prefix(*a)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        o = tbf16.paged_sdpa_prefix(*a)
    for prefix, lengths in ((500, [60] * 9), (31, list(range(9))), (0, [0] * 9), (499, [0, 60] * 4 + [1])):
        a[4].fill_(prefix)
        a[6].copy_(torch.tensor(lengths, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        got = o.clone()
        assert torch.equal(got, check(a))


def test_two_graphs_of_one_pool(dev):
    """Graphs whose workspaces lie in the same memory, replayed in turns."""
    both = [make(dev, 900, [b * 5 % 100 for b in range(20)], 8, 2, 128, 16, seed=15),
            make(dev, 300, [b * 7 % 90 for b in range(33)], 16, 4, 64, 16, seed=16)]
    want = [check(a) for a in both]
    s = torch.cuda.Stream()
    graphs, outs = [], []
    torch.cuda.synchronize()
    for a in both:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s, pool=graphs[0].pool() if graphs else None):
            outs.append(tbf16.paged_sdpa_prefix(*a))
        graphs.append(g)
    for _ in range(4):
        for g, o, w, a in zip(graphs, outs, want, both):
            o.zero_()
            g.replay()
            assert torch.equal(o, w) and torch.equal(tbf16.paged_sdpa_prefix(*a), w)
