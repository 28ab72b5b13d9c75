"""The serving operators on the GPU against 64 bits: paged_write, paged_sdpa, the 8-bit
integer linear, and a decoding step made of them. Tolerances: tests/_serving64.py."""
import math

import pytest
import torch
import torch.nn as nn

import tbf16
from tbf16 import int8

from _serving64 import codes64, int8_linear64, paged_sdpa64

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make_cache(dev, lengths, Hkv, D, page, seed=0, spare=3, junk=float("nan"), kscale=1.0):
    """k_cache, v_cache, table, lengths with the pages in random order; every row that no
    position below its length uses holds `junk`, unused table entries point anywhere."""
    g = gen(seed)
    need = [-(-max(n, 0) // page) for n in lengths]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g)
    table = torch.randint(0, pages, (len(lengths), max(need + [1])), generator=g, dtype=torch.int32)
    k = (torch.randn(pages, Hkv, page, D, generator=g) * kscale).to(BF)
    v = (torch.randn(pages, Hkv, page, D, generator=g) * torch.exp2(torch.randint(-3, 4, (Hkv, 1, 1), generator=g))).to(BF)
    used = torch.zeros(pages, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(lengths):
        mine = order[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = mine.int()
        j = torch.arange(max(n, 0))
        used[mine[j // page], j % page] = True
    if junk is not None:
        for c in (k, v):
            c.masked_fill_(~used[:, None, :, None], junk)
    return k.to(dev), v.to(dev), table.to(dev), torch.tensor(lengths, dtype=torch.int32, device=dev)


def check_attend(q, k, v, table, lengths, scale=None):
    o = tbf16.paged_sdpa(q, k, v, table, lengths, scale)
    assert o.shape == q.shape and o.dtype == BF and o.is_contiguous()
    ref, bound = paged_sdpa64(q, k, v, table, lengths, scale)
    finite = torch.isfinite(ref)  # (not where an infinite value has a weight)
    assert torch.equal(torch.isfinite(o.cpu()), finite)
    err = (o.cpu().double() - ref).abs()[finite]
    assert (err <= bound[finite]).all(), (err - bound[finite]).max()
    return o


ATTEND = [  # H, Hkv, D, page, lengths
    (1, 1, 8, 1, [1]),
    (1, 1, 64, 16, [1, 0, 2]),
    (4, 4, 64, 16, [15, 16, 17, 31, 32, 33]),
    (8, 2, 128, 16, [1, 63, 64, 65, 100, 127, 128, 129, 0]),
    (16, 16, 128, 16, [700]),
    (20, 4, 80, 48, [3, 47, 48, 49, 500, 1499]),
    (6, 3, 72, 24, [25, 200, 0, 777]),
    (12, 12, 96, 7, [1, 6, 7, 8, 333]),
    (16, 1, 256, 16, [5, 300, 1025]),
    (8, 8, 256, 64, [64, 513]),
    (24, 1, 128, 32, [90, 700]),
    (32, 2, 64, 100, [99, 100, 101, 1000]),
    (64, 1, 128, 16, [1, 250]),
    (71, 1, 64, 16, [33, 400]),
    (130, 2, 64, 16, [40, 257]),
    (48, 2, 256, 8, [130, 9]),
    (5, 1, 40, 16, [18, 1]),
    (32, 8, 128, 16, [4096, 1, 2000, 3]),
    (4, 1, 128, 128, [20000]),
    (16, 8, 24, 3, [50] * 70),
    # rows of heads in several units, in both forms of the split
    (130, 2, 64, 16, [2000, 7]),
    (24, 1, 128, 32, [90, 300]),
    (80, 2, 128, 16, [1200, 31]),
    (40, 1, 256, 16, [900, 45]),
    (3, 1, 200, 16, [100, 7]),
    (16, 1, 128, 16, [500, 20]),
    (32, 2, 128, 16, [1500, 20]),
    (8, 4, 200, 16, [3000, 7, 0, 900]),
]


@pytest.mark.parametrize("H,Hkv,D,page,lengths", ATTEND)
def test_attend_shapes(dev, H, Hkv, D, page, lengths):
    k, v, table, ln = make_cache(dev, lengths, Hkv, D, page, seed=H + D + page)
    q = (torch.randn(len(lengths), H, D, generator=gen(1)) * 2).to(BF).to(dev)
    check_attend(q, k, v, table, ln)


@pytest.mark.parametrize("B,lengths_of", [(300, lambda b: b % 5), (257, lambda b: 1), (1000, lambda b: (b * 37) % 90)])
def test_attend_many_short(dev, B, lengths_of):
    lengths = [lengths_of(b) for b in range(B)]
    k, v, table, ln = make_cache(dev, lengths, 2, 64, 16, seed=B)
    q = torch.randn(B, 4, 64, generator=gen(2)).to(BF).to(dev)
    check_attend(q, k, v, table, ln)


@pytest.mark.parametrize("seed", range(30))
def test_attend_random_batches(dev, seed):
    """Where the runs of the waves and blocks begin and end in the batch."""
    r = __import__("random").Random(seed)
    B = r.choice((1, 2, 3, 9, 40, 150))
    Hkv, D, page = r.choice((1, 2, 5)), r.choice((8, 64, 72, 128)), r.choice((1, 5, 16, 33, 64))
    top = r.choice((33, 200, 1500)) if B > 9 else r.choice((40, 700, 6000))
    lengths = [r.choice((0, 1, r.randrange(top), r.randrange(top), 32 * r.randrange(1, top // 32 + 1))) for _ in range(B)]
    H = Hkv * r.choice((1, 3, 4, 8, 17))
    k, v, table, ln = make_cache(dev, lengths, Hkv, D, page, seed=seed)
    q = torch.randn(B, H, D, generator=gen(seed)).to(BF).to(dev)
    check_attend(q, k, v, table, ln)
    wide = torch.full((B, table.shape[1] + 5000 // page), -1, dtype=torch.int32, device=dev)  # room for long ones
    wide[:, :table.shape[1]] = table
    check_attend(q, k, v, wide, ln)


def test_attend_very_many_sequences(dev):
    B = 70000
    k = torch.randn(50, 1, 4, 8, generator=gen(1)).to(BF).to(dev)
    table = torch.randint(0, 50, (B, 2), generator=gen(2), dtype=torch.int32).to(dev)
    ln = torch.randint(0, 9, (B,), generator=gen(3), dtype=torch.int32).to(dev)
    q = torch.randn(B, 2, 8, generator=gen(4)).to(BF).to(dev)
    o = tbf16.paged_sdpa(q, k, k, table, ln)
    at = torch.cat((torch.arange(40), torch.randint(0, B, (100,), generator=gen(5)), torch.arange(B - 40, B)))
    ref, bound = paged_sdpa64(q[at], k, k, table[at], ln[at])
    assert ((o[at].cpu().double() - ref).abs() <= bound).all()


@pytest.mark.parametrize("scale", [0.0, -0.5, 3.0, 1e-3])
def test_attend_scales(dev, scale):
    k, v, table, ln = make_cache(dev, [90, 17], 2, 64, 16, seed=3)
    q = torch.randn(2, 4, 64, generator=gen(3)).to(BF).to(dev)
    check_attend(q, k, v, table, ln, scale)


def test_attend_large_values(dev):
    # logits in the thousands (one key takes all the weight); values near bf16's largest, one
    # of them rounded to infinity
    k, v, table, ln = make_cache(dev, [333, 40], 2, 128, 16, seed=4, kscale=40.0)
    q = (torch.randn(2, 4, 128, generator=gen(4)) * 40).to(BF).to(dev)
    check_attend(q, k, v, table, ln)
    big = torch.where(torch.isfinite(v), v * 1e37, v)
    check_attend(q, k, big, table, ln)


def test_attend_infinite_keys(dev):
    """A key of -infinity weighs nothing; one of +infinity, or a NaN, makes its sequence's heads NaN."""
    k, v, table, ln = make_cache(dev, [70, 70, 70, 5], 1, 64, 16, seed=5)
    q = torch.rand(4, 2, 64, generator=gen(5)).to(BF).to(dev) + 0.5
    at = lambda b, j: (int(table[b, j // 16]), 0, j % 16)  # noqa: E731
    k[at(0, 3)] = -math.inf
    k[at(0, 69)] = -math.inf
    k[at(1, 33)] = math.inf
    k[at(2, 69)] = math.nan
    for j in range(5):
        k[at(3, j)] = -math.inf
    o = tbf16.paged_sdpa(q, k, v, table, ln)
    ref, bound = paged_sdpa64(q, k, v, table, ln)
    assert not ref[0].isnan().any() and ref[1:].isnan().all()  # (only -infinities: NaN, as a softmax has it)
    assert o[1:].isnan().all()
    j = [j for j in range(70) if j not in (3, 69)]  # the bound without the infinite keys
    pages = torch.tensor([at(0, x)[0] for x in j])
    off = torch.tensor([x % 16 for x in j])
    k1, v1 = k[pages, :, off][None].transpose(1, 2), v[pages, :, off][None].transpose(1, 2)
    ref1, bound1 = paged_sdpa64(q[:1], k1, v1, torch.zeros(1, 1, dtype=torch.int32), torch.tensor([68]))
    assert torch.allclose(ref1[0], ref[0], rtol=1e-12, atol=0)
    assert ((o[0].cpu().double() - ref1[0]).abs() <= bound1[0]).all()


def test_attend_nan_value_and_query(dev):
    k, v, table, ln = make_cache(dev, [40, 40], 1, 64, 16, seed=6)
    q = torch.randn(2, 3, 64, generator=gen(6)).to(BF).to(dev)
    clean = tbf16.paged_sdpa(q, k, v, table, ln)
    q2 = q.clone()
    q2[0, 1, 5] = math.nan
    o = tbf16.paged_sdpa(q2, k, v, table, ln)
    assert o[0, 1].isnan().all()
    assert torch.equal(o[0, 0], clean[0, 0]) and torch.equal(o[0, 2], clean[0, 2]) and torch.equal(o[1], clean[1])
    v2 = v.clone()
    v2[int(table[1, 2]), 0, 39 % 16, 7] = math.nan
    o = tbf16.paged_sdpa(q, k, v2, table, ln)
    assert o[1, :, 7].isnan().all() and torch.isfinite(o[1, :, :7]).all() and torch.isfinite(o[1, :, 8:]).all()
    assert torch.equal(o[0], clean[0])


def test_attend_absent_pages_and_lengths(dev):
    """Entries outside the cache hold no keys; lengths past the table stop at its end,
    negative ones count as zero."""
    k, v, table, ln = make_cache(dev, [100, 100, 100, 100], 2, 64, 16, seed=7)
    q = torch.randn(4, 4, 64, generator=gen(7)).to(BF).to(dev)
    table[0, 2] = -1
    table[1, 0] = k.shape[0]
    table[1, 6] = 2 ** 31 - 1
    table[2] = -5
    check_attend(q, k, v, table, ln)
    assert (tbf16.paged_sdpa(q, k, v, table, ln)[2] == 0).all()
    full = make_cache(dev, [112], 2, 64, 16, seed=8)
    o = tbf16.paged_sdpa(q[:1], *full)
    for n in (113, 2 ** 31 - 1):
        assert torch.equal(o, tbf16.paged_sdpa(q[:1], *full[:3], torch.tensor([n], dtype=torch.int32, device=dev)))
    for n in (-1, -2 ** 31, 0):
        assert (tbf16.paged_sdpa(q[:1], *full[:3], torch.tensor([n], dtype=torch.int32, device=dev)) == 0).all()


def test_attend_shared_pages(dev):
    """Sequences with a common prefix hold the same pages; one sequence may hold a page twice."""
    k, v, table, ln = make_cache(dev, [200, 200, 200], 2, 64, 16, seed=9)
    table[1, :10] = table[0, :10]
    table[2, 3] = table[2, 4]
    q = torch.randn(3, 8, 64, generator=gen(9)).to(BF).to(dev)
    check_attend(q, k, v, table, ln)


def test_attend_layouts(dev):
    """Other orders of the cache's axes, q as a slice, tables and lengths as views, one tensor
    as keys and values: the same bits."""
    lengths = [130, 7, 64]
    k, v, table, ln = make_cache(dev, lengths, 4, 64, 16, seed=10)
    q = torch.randn(3, 8, 64, generator=gen(10)).to(BF).to(dev)
    o = check_attend(q, k, v, table, ln)
    rows = lambda c: c.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731  (pages, page, Hkv, D)
    assert torch.equal(o, tbf16.paged_sdpa(q, rows(k), rows(v), table, ln))
    both = torch.stack((k, v), 1)  # (pages, 2, Hkv, page, D)
    assert torch.equal(o, tbf16.paged_sdpa(q, both[:, 0], both[:, 1], table, ln))
    wide = torch.cat((k, v), -1)  # keys and values of a position side by side
    assert torch.equal(o, tbf16.paged_sdpa(q, wide[..., :64], wide[..., 64:], table, ln))
    qkv = torch.zeros(3, 16, 64, dtype=BF, device=dev)
    qkv[:, 3:11] = q
    assert torch.equal(o, tbf16.paged_sdpa(qkv[:, 3:11], k, v, table, ln))
    odd = torch.zeros(3 * 8 * 64 + 1, dtype=BF, device=dev)[1:].view(3, 8, 64)
    odd.copy_(q)
    assert torch.equal(o, tbf16.paged_sdpa(odd, k, v, table, ln))
    assert torch.equal(o, tbf16.paged_sdpa(q.transpose(1, 2).contiguous().transpose(1, 2), k, v, table, ln))
    t2 = torch.full((3, 40), -1, dtype=torch.int32, device=dev)
    t2[:, 5:5 + table.shape[1]] = table
    assert torch.equal(o, tbf16.paged_sdpa(q, k, v, t2[:, 5:5 + table.shape[1]], ln))
    assert torch.equal(o, tbf16.paged_sdpa(q, k, v, table.t().contiguous().t(), ln.repeat_interleave(2)[::2]))
    check_attend(q, k, k, table, ln)


def test_attend_far_pages(dev):
    """Offsets beyond 2^32 bytes and 2^32 elements."""
    pages, Hkv, page, D = 70000, 8, 64, 128  # 4.6e9 elements
    k = torch.empty(pages, Hkv, page, D, dtype=BF, device=dev)
    at = torch.tensor([0, 32767, 32768, 65535, 65536, 69999])
    small = torch.randn(2, 6, Hkv, page, D, generator=gen(11)).to(BF).to(dev)
    k[at] = small[0]
    ln = torch.tensor([6 * page - 5], dtype=torch.int32, device=dev)
    q = torch.randn(1, 16, D, generator=gen(12)).to(BF).to(dev)
    want = tbf16.paged_sdpa(q, small[0], small[0], torch.arange(6, dtype=torch.int32, device=dev)[None], ln)
    table = at.int().to(dev)[None]
    assert torch.equal(want, tbf16.paged_sdpa(q, k, k, table, ln))
    # and written there
    slots = (at * page + 9).int().to(dev)
    new = torch.randn(2, 6, Hkv, D, generator=gen(13)).to(BF).to(dev)
    v = torch.zeros_like(k)
    tbf16.paged_write(k, v, new[0], new[1], slots)
    assert torch.equal(k[at, :, 9], new[0]) and torch.equal(v[at, :, 9], new[1])
    assert int(v.view(torch.int16).count_nonzero()) == int(new[1].view(torch.int16).count_nonzero())


def test_attend_empty(dev):
    k = torch.zeros(3, 2, 16, 64, dtype=BF, device=dev)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
    assert tbf16.paged_sdpa(torch.zeros(0, 4, 64, dtype=BF, device=dev), k, k, i32(0, 3), i32(0)).shape == (0, 4, 64)
    q = torch.ones(2, 4, 64, dtype=BF, device=dev)
    assert (tbf16.paged_sdpa(q, k, k, i32(2, 0), i32(2) + 5) == 0).all()
    assert (tbf16.paged_sdpa(q, k[:0], k[:0], i32(2, 3), i32(2) + 5) == 0).all()
    many = torch.ones(300, 4, 64, dtype=BF, device=dev)
    for n, pages in ((0, 3), (3, 0), (900, 0), (3, 3)):
        assert (tbf16.paged_sdpa(many, k[:pages], k[:pages], i32(300, n), i32(300) + (5 if n * pages == 0 else 0)) == 0).all()


def test_attend_same_bits_again(dev):
    k, v, table, ln = make_cache(dev, [3000, 10, 1234, 500], 8, 128, 16, seed=14)
    q = torch.randn(4, 32, 128, generator=gen(14)).to(BF).to(dev)
    o = check_attend(q, k, v, table, ln)
    for _ in range(5):
        assert torch.equal(o, tbf16.paged_sdpa(q, k, v, table, ln))


# ---- write ---------------------------------------------------------------------------


@pytest.mark.parametrize("T,Hkv,D,page", [(1, 1, 8, 1), (7, 2, 64, 16), (64, 8, 128, 16), (130, 3, 80, 48), (1000, 4, 72, 5),
                                          (5000, 2, 256, 64)])
def test_write(dev, T, Hkv, D, page):
    """Tokens land in their slots, a third of them nowhere; every other row keeps its bits."""
    g = gen(T)
    pages = -(-T // page) + 4
    kv = torch.randn(2, pages, Hkv, page, D, generator=g).to(BF).to(dev)
    want = kv.clone()
    new = torch.randn(T, 2, Hkv, D, generator=g).to(BF).to(dev)
    slots = torch.randperm(pages * page, generator=g)[:T].int()
    lost = torch.rand(T, generator=g) < 0.3
    slots[lost] = torch.tensor([-1, pages * page, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32)[torch.arange(int(lost.sum())) % 4]
    tbf16.paged_write(kv[0], kv[1], new[:, 0], new[:, 1], slots.to(dev))
    s = slots[~lost].long().to(dev)
    for i in range(2):
        want[i][s // page, :, s % page] = new[~lost.to(dev), i]
    assert torch.equal(kv.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("T,distinct", [(2, 1), (64, 5), (1000, 400), (9000, 8000), (20000, 1), (70000, 66000), (140000, 70000)])
def test_write_repeated_slots(dev, T, distinct):
    """The last token of a slot stays, keys and values both."""
    g = gen(T)
    slots = torch.randint(0, distinct, (T,), generator=g)
    last = torch.zeros(distinct, dtype=torch.long) - 1
    last.scatter_reduce_(0, slots, torch.arange(T), "amax")
    new = torch.randn(T, 2, 1, 64, generator=g).to(BF).to(dev)
    cache = torch.zeros(2, -(-distinct // 16), 1, 16, 64, dtype=BF, device=dev)
    tbf16.paged_write(cache[0], cache[1], new[:, 0], new[:, 1], slots.int().to(dev))
    got = cache.transpose(2, 3).reshape(2, -1, 1, 64)
    named = (last >= 0).to(dev)
    last = last.to(dev)
    for i in range(2):
        assert torch.equal(got[i][:distinct][named], new[:, i][last[named]])
        assert (got[i][:distinct][~named] == 0).all() and (got[i][distinct:] == 0).all()


def test_write_layouts(dev):
    g = gen(20)
    k, v = (torch.randn(40, 2, 64, generator=g).to(BF).to(dev) for _ in range(2))
    slots = torch.randperm(64, generator=g)[:40].int().to(dev)
    want = torch.zeros(2, 4, 2, 16, 64, dtype=BF, device=dev)
    tbf16.paged_write(want[0], want[1], k, v, slots)

    def same(kc, vc, *kvs):
        before = kc._version
        tbf16.paged_write(kc, vc, *kvs)
        assert kc._version > before
        assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])

    z = lambda *s: torch.zeros(*s, dtype=BF, device=dev)  # noqa: E731
    same(z(4, 16, 2, 64).transpose(1, 2), z(4, 16, 2, 64).transpose(1, 2), k, v, slots)
    both = z(4, 2, 16, 128)
    same(both[..., :64], both[..., 64:], k, v, slots)
    fused = torch.cat((z(40, 24), k.reshape(40, -1), v.reshape(40, -1)), 1)  # one projection's output
    same(z(4, 2, 16, 64), z(4, 2, 16, 64), fused[:, 24:152].view(40, 2, 64), fused[:, 152:].view(40, 2, 64), slots)
    off = torch.cat((z(40, 3), k.reshape(40, -1), v.reshape(40, -1)), 1)  # rows that no 16 bytes divide
    same(z(4, 2, 16, 64), z(4, 2, 16, 64), off[:, 3:131].view(40, 2, 64), off[:, 131:].view(40, 2, 64), slots)
    same(z(4, 2, 16, 64), z(4, 2, 16, 64), k.transpose(0, 1).contiguous().transpose(0, 1), v, slots.repeat_interleave(2)[::2])
    c = z(4, 2, 16, 64), z(4, 2, 16, 64)
    tbf16.paged_write(*c, k[:0], v[:0], slots[:0])
    assert (c[0] == 0).all()


# ---- 8-bit integer linear --------------------------------------------------------------


@pytest.mark.parametrize("R,K", [(1, 1), (3, 7), (5, 16), (64, 100), (33, 1000), (9, 4096), (4, 20000), (2, 131072)])
def test_codes(dev, R, K):
    x = torch.randn(R, K, generator=gen(R + K))
    x[R // 2] *= 2.0 ** 90
    x = x.to(BF)
    q, s = int8.quantize_rows_i8(x.to(dev))
    cq, cs = codes64(x)
    assert q.dtype == torch.int8 and q.shape == (R, K) and s.shape == (R,)
    assert torch.equal(q.cpu().double(), cq)
    assert ((s.cpu().double() - cs[:, 0]).abs() <= 2.0 ** -24 * cs[:, 0]).all()


def test_codes_every_pair(dev):
    """Every 8-bit significand against every maximum's, at exponents where their quotients reach
    the borders between codes (ties among them: 127 x / a = n + 1/2)."""
    sig = torch.arange(128, 256).float()
    rows = []
    for e in range(9):
        rows.append(torch.cat((sig[None].expand(128, -1) * 2.0 ** -e, sig[:, None]), 1))
    x = torch.cat(rows)
    x = torch.where(x.abs() > x[:, -1:], x / 2, x)
    x[:, ::3] *= -1
    ties = 0
    for scale in (1.0, 2.0 ** 119, 2.0 ** -133, 2.0 ** -126, 2.0 ** -60, 2.0 ** 60):
        xs = (x.double() * scale).to(BF)
        q, s = int8.quantize_rows_i8(xs.to(dev))
        cq, cs = codes64(xs)
        assert torch.equal(q.cpu().double(), cq), scale
        frac = (127.0 * xs.double() / xs.double().abs().amax(1, keepdim=True)).abs() % 1
        ties += int((frac == 0.5).sum())
    assert ties > 100


def test_codes_special_rows(dev):
    x = torch.randn(6, 50, generator=gen(1)).to(BF)
    x[0] = 0
    x[1, 3] = math.inf
    x[2, 49] = -math.inf
    x[3, 0] = math.nan
    x[4] = -0.0
    q, s = int8.quantize_rows_i8(x.to(dev))
    assert (q[:5] == 0).all() and s[0] == 0 and s[4] == 0 and s[1:4].isnan().all() and torch.isfinite(s[5])


def check_linear(x, w, b=None, y=None):
    dev = x.device
    if y is None:
        y = tbf16.int8_linear(x, *tbf16.prepare_weight_i8(w), b)
    assert y.dtype == BF and y.shape == (*x.shape[:-1], w.shape[0])
    ref, bound = int8_linear64(x.reshape(-1, x.shape[-1]), w, b)
    err = (y.reshape(ref.shape).cpu().double() - ref).abs()
    assert (err <= bound).all(), (err - bound).max()
    return y


LINEAR = [(1, 1, 1), (1, 16, 8), (1, 4096, 512), (1, 1000, 1001), (2, 64, 64), (3, 100, 7), (5, 2560, 1024), (16, 2560, 1280),
          (17, 1040, 250), (31, 333, 96), (33, 96, 4096), (64, 4096, 640), (65, 512, 512), (100, 1000, 3001),
          (128, 1024, 128), (129, 640, 264), (200, 2048, 1024), (256, 4096, 256), (257, 130, 1030), (384, 384, 384),
          (513, 2049, 200), (1024, 512, 1024), (1500, 64, 2000), (2048, 200, 24), (4097, 136, 520), (8, 16, 40000),
          (700, 16, 16), (6, 4096, 100), (16, 4096, 33), (9, 8, 3000), (13, 4104, 70), (2, 32768, 24), (5, 24, 16),
          (1, 131072, 40), (40, 40000, 72), (300, 33000, 64)]


@pytest.mark.parametrize("M,K,N", LINEAR)
@pytest.mark.parametrize("bias", [False, True])
def test_linear_shapes(dev, M, K, N, bias):
    g = gen(M + K + N)
    x = torch.randn(M, K, generator=g) * torch.where(torch.rand(K, generator=g) < 0.02, 10.0, 1.0)
    w = (torch.randn(N, K, generator=g) * K ** -0.5).to(BF).to(dev)
    b = torch.randn(N, generator=g).to(BF).to(dev) if bias else None
    check_linear(x.to(BF).to(dev), w, b)


@pytest.mark.parametrize("M", [1, 2, 40, 300, 1100])
def test_linear_largest_sums(dev, M):
    """Every product 127 x 127 at the longest row: the int32 sums stay exact."""
    K = 131072
    x = torch.ones(M, K, dtype=BF, device=dev)
    w = torch.ones(24, K, dtype=BF, device=dev)
    w[1::2] = -1
    y = tbf16.int8_linear(x, *tbf16.prepare_weight_i8(w))
    want = torch.full((M, 24), float(K))
    want[:, 1::2] = -K
    # the sum 127 * 127 * 2^17 has 31 bits: a conversion, two scales of 2^-24 each and two factors
    assert ((y.cpu().double() - want).abs() <= (2.0 ** -8 + 6 * 2.0 ** -24) * K).all()
    assert torch.equal(y.cpu(), want.to(BF))


@pytest.mark.parametrize("M", [1, 3, 14, 30, 500])
def test_linear_special_rows(dev, M):
    x = torch.randn(M, 200, generator=gen(2)).to(BF).to(dev)
    w = torch.randn(90, 200, generator=gen(3)).to(BF).to(dev)
    b = torch.randn(90, generator=gen(4)).to(BF).to(dev)
    w[5] = 0
    w[7, 3] = math.inf
    w[89, 199] = math.nan
    w8 = tbf16.prepare_weight_i8(w)
    for bad in (math.inf, -math.inf, math.nan, 0.0):
        xb = x.clone()
        if bad == 0.0:
            xb[-1] = 0
        else:
            xb[-1, 77] = bad
        y = tbf16.int8_linear(xb, *w8, b)
        keep = [n for n in range(90) if n not in (7, 89)]
        assert y[:, 7].isnan().all() and y[:, 89].isnan().all()
        assert torch.equal(y[:-1, 5], b[5].expand(M - 1))
        if bad == 0.0:
            assert torch.equal(y[-1, keep], b[keep])
        else:
            assert y[-1].isnan().all()
        if M > 1:
            check_linear(xb[:-1], w[keep], b[keep], y=y[:-1][:, keep])


@pytest.mark.parametrize("scale", [1e30, 1e-25])
@pytest.mark.parametrize("M", [1, 4, 12, 20, 300])
def test_linear_extreme_scales(dev, scale, M):
    x = (torch.randn(M, 256, generator=gen(5)) * scale).to(BF).to(dev)
    w = (torch.randn(64, 256, generator=gen(6)) / 16).to(BF).to(dev)
    check_linear(x, w)


def test_linear_layouts(dev):
    g = gen(7)
    x = torch.randn(50, 200, generator=g).to(BF).to(dev)
    w = torch.randn(70, 200, generator=g).to(BF).to(dev)
    w8, ws = tbf16.prepare_weight_i8(w)
    y = check_linear(x, w)
    f = lambda *a: tbf16.int8_linear(*a)  # noqa: E731
    assert torch.equal(y, f(x.t().contiguous().t(), w8, ws))
    wide = torch.randn(50, 301, generator=g).to(BF).to(dev)
    wide[:, 5:205] = x
    assert torch.equal(y, f(wide[:, 5:205], w8, ws))
    assert torch.equal(y[::2], f(x[::2], w8, ws))
    assert torch.equal(y.view(5, 10, 70), f(x.view(5, 10, 200), w8, ws))
    assert torch.equal(y[:1].expand(9, 70), f(x[:1].expand(9, 200), w8, ws))
    assert torch.equal(y[0], f(x[0], w8, ws))
    assert torch.equal(y, f(x, w8.contiguous(), ws))          # rows of 200 bytes
    assert torch.equal(y, f(x, w8.t().contiguous().t(), ws.double()))
    junk = torch.full((70, 256), 77, dtype=torch.int8, device=dev)  # what lies behind a row does not matter
    junk[:, :200] = w8
    assert torch.equal(y, f(x, junk[:, :200], ws))
    flat = torch.zeros(70 * 208 + 1, dtype=torch.int8, device=dev)[1:].view(70, 208)
    flat[:, :200] = w8
    assert torch.equal(y, f(x, flat[:, :200], ws))
    assert f(x[:0], w8, ws).shape == (0, 70) and f(x, w8[:0], ws[:0]).shape == (50, 0)
    b = torch.randn(70, generator=g).to(BF).to(dev)
    assert torch.equal(f(x[:, :0], w8[:, :0], ws, b), b.expand(50, 70))
    pad = torch.zeros(71, dtype=BF, device=dev)[1:]
    pad.copy_(b)
    assert torch.equal(f(x, w8, ws, b), f(x, w8, ws, pad)) and torch.equal(f(x, w8, ws, b.float()), f(x, w8, ws, b))


def test_linear_rows_alone(dev):
    """A row's result does not depend on the rows beside it (int32 sums are exact)."""
    x = torch.randn(600, 520, generator=gen(8)).to(BF).to(dev)
    w8, ws = tbf16.prepare_weight_i8(torch.randn(136, 520, generator=gen(9)).to(BF).to(dev))
    y = tbf16.int8_linear(x, w8, ws)
    for n in (1, 2, 3, 4, 5, 8, 9, 16, 17, 64, 100, 128, 300):
        assert torch.equal(y[:n], tbf16.int8_linear(x[:n], w8, ws)), n


@pytest.mark.parametrize("M,K,N", [(4096, 640, 4096), (4300, 1041, 4099), (4096, 128, 4096), (2048, 4096, 2056), (1100, 2000, 8200),
                                   (9000, 136, 1500), (520, 4096, 16384), (2000, 260, 1000), (6000, 16, 3000), (3000, 4224, 700)])
def test_linear_large_tiles(dev, M, K, N):
    """Every tile's outputs are those of a few rows at a time, bit for bit."""
    x = torch.randn(M, K, generator=gen(M)).to(BF).to(dev)
    w8, ws = tbf16.prepare_weight_i8(torch.randn(N, K, generator=gen(N)).to(BF).to(dev))
    b = torch.randn(N, generator=gen(K)).to(BF).to(dev)
    y = tbf16.int8_linear(x, w8, ws, b)
    for m in range(0, M, 60):
        assert torch.equal(y[m:m + 60], tbf16.int8_linear(x[m:m + 60], w8, ws, b)), m


def test_linear_far_offsets(dev):
    """Outputs and weights past 2^31 elements and bytes."""
    g = gen(10)
    x = torch.randn(40000, 64, generator=g).to(BF).to(dev)
    w = torch.randn(65536, 64, generator=g).to(BF).to(dev)
    y = tbf16.int8_linear(x, *tbf16.prepare_weight_i8(w))
    m, n = torch.tensor([0, 1, 20000, 32767, 32768, 39999]), torch.tensor([0, 7, 255, 256, 40000, 65535])
    ref, bound = int8_linear64(x[m], w[n])
    assert ((y[m][:, n].cpu().double() - ref).abs() <= bound).all()
    del x, w, y
    K, N = 65536, 40000
    w8 = torch.randint(-127, 128, (N, K), dtype=torch.int8, device=dev)  # 2.6e9 bytes
    ws = torch.ones(N, device=dev)
    n = torch.tensor([0, 1, 32767, 32768, 39998, 39999])
    for M in (1, 3, 200):
        x = torch.randn(M, K, generator=g).to(BF)
        y = tbf16.int8_linear(x.to(dev), w8, ws)
        cx, sx = codes64(x)
        ref = (cx @ w8[n].cpu().double().t()) * sx
        assert ((y[:, n].cpu().double() - ref).abs() <= 2.0 ** -8 * ref.abs() * (1 + 2.0 ** -10) + 6 * 2.0 ** -24 * ref.abs()).all()


# ---- streams, graphs, modules -------------------------------------------------------------


def test_other_stream(dev):
    lengths = [500, 33, 0, 900]
    k, v, table, ln = make_cache(dev, lengths, 4, 128, 16, seed=30)
    q = torch.randn(4, 16, 128, generator=gen(30)).to(BF).to(dev)
    x = torch.randn(4, 2048, generator=gen(31)).to(BF).to(dev)
    w8, ws = tbf16.prepare_weight_i8(torch.randn(256, 2048, generator=gen(32)).to(BF).to(dev))
    want = tbf16.paged_sdpa(q, k, v, table, ln), tbf16.int8_linear(x, w8, ws)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(4):  # two streams at once
        for s in (s1, s2):
            with torch.cuda.stream(s):
                got.append((tbf16.paged_sdpa(q, k, v, table, ln), tbf16.int8_linear(x, w8, ws)))
    torch.cuda.synchronize()
    for o, y in got:
        assert torch.equal(o, want[0]) and torch.equal(y, want[1])


class Layer(nn.Module):
    """Attention of a decoder layer over a paged cache, between two linears."""

    def __init__(self, E, H, Hkv, D):
        super().__init__()
        self.H, self.Hkv, self.D = H, Hkv, D
        self.qkv = nn.Linear(E, (H + 2 * Hkv) * D)
        self.out = nn.Linear(H * D, E, bias=False)

    def forward(self, x, cache, slots, table, lengths):
        H, Hkv, D = self.H, self.Hkv, self.D
        q, k, v = self.qkv(x).view(x.shape[0], H + 2 * Hkv, D).split((H, Hkv, Hkv), 1)
        tbf16.paged_write(*cache, k, v, slots)
        return self.out(tbf16.paged_sdpa(q, *cache, table, lengths).flatten(1))


def layer64(m, x, cache, slots, table, lengths, linear):
    """The same step on the CPU in 64 bits (cache: float64 copies, written in place), with the
    linears by `linear` and what the operators hand on rounded to bf16 as they do."""
    H, Hkv, D = m.H, m.Hkv, m.D
    page = cache[0].shape[2]
    q, k, v = linear(m.qkv, x).view(-1, H + 2 * Hkv, D).split((H, Hkv, Hkv), 1)
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            cache[0][s // page, :, s % page] = k[t]
            cache[1][s // page, :, s % page] = v[t]
    o, _ = paged_sdpa64(q, *cache, table, lengths)
    return linear(m.out, o.to(BF).flatten(1))


@pytest.mark.parametrize("int8_layers", [False, True])
def test_decode_loop(dev, int8_layers):
    """A prompt, then tokens one at a time through a converted layer, in a padded batch: against
    the whole in 64 bits, eagerly and as a graph replayed with new slots and lengths."""
    E, H, Hkv, D, page, B = 256, 8, 2, 64, 16, 5
    torch.manual_seed(0)
    m = Layer(E, H, Hkv, D).to(BF).to(dev).requires_grad_(False)
    ws = {m.qkv: m.qkv.weight.cpu(), m.out: m.out.weight.cpu()}
    bs = {m.qkv: m.qkv.bias.cpu(), m.out: None}
    held = {"qkv": (ws[m.qkv], bs[m.qkv]), "out": (ws[m.out], None)}
    tbf16.convert(m, sdpa=False, int8=int8_layers)
    assert isinstance(m.qkv, tbf16.Int8Linear if int8_layers else tbf16.Linear)

    def linear(mod, x):
        w, b = held["qkv"] if mod is m.qkv else held["out"]
        if int8_layers:
            return int8_linear64(x, w, b)[0].to(BF)
        y = x.double() @ w.double().t()
        return (y if b is None else y + b.double()).to(BF)

    pages = 30
    cache = [torch.zeros(pages, Hkv, page, D, dtype=BF, device=dev) for _ in range(2)]
    cache64 = [torch.zeros(pages, Hkv, page, D, dtype=BF) for _ in range(2)]
    g = gen(40)
    table = torch.randperm(pages, generator=g)[:B * 5].view(B, 5).int()
    lengths = torch.tensor([37, 0, 15, 64, 1])  # sequence 1: nobody in its place
    slot = lambda b, j: int(table[b, j // page]) * page + j % page  # noqa: E731
    # the prompts, all rows at once
    slots = torch.tensor([slot(b, j) for b in range(B) for j in range(int(lengths[b]))] + [-1] * 3, dtype=torch.int32)
    x = torch.randn(len(slots), E, generator=g).to(BF)
    with torch.no_grad():
        kv = m.qkv(x.to(dev)).view(-1, H + 2 * Hkv, D)
        tbf16.paged_write(*cache, kv[:, H:H + Hkv], kv[:, H + Hkv:], slots.to(dev))
    for t, s in enumerate(slots.tolist()):  # the layer's own rows: a projection's rounding is not tested here
        if s >= 0:
            cache64[0][s // page, :, s % page] = kv[t, H:H + Hkv].cpu()
            cache64[1][s // page, :, s % page] = kv[t, H + Hkv:].cpu()

    xs, ss = torch.zeros(B, E, dtype=BF, device=dev), torch.zeros(B, dtype=torch.int32, device=dev)
    tb, ln = table.to(dev), torch.zeros(B, dtype=torch.int32, device=dev)

    def step(i):
        live = lengths > 0
        new = [slot(b, int(lengths[b])) if live[b] else -1 for b in range(B)]
        lengths[live] += 1
        xs.copy_(torch.randn(B, E, generator=gen(50 + i)).to(BF))
        ss.copy_(torch.tensor(new, dtype=torch.int32))
        ln.copy_(lengths.int())

    def check(y):
        want = layer64(m, xs.cpu(), cache64, ss.cpu(), tb.cpu(), ln.cpu(), linear)
        # a projection's or attention's output next to a border between two bf16 may round the
        # other way and change one input of the next by 2^-7 of itself: 4 of those in a row's
        # 512 products of random signs, and the last rounding
        err = (y.cpu().double() - want.double()).norm() / want.double().norm()
        assert err < 2.0 ** -7, err
        for c, c64 in zip(cache, cache64):
            assert (c.cpu().double() - c64.double()).abs().max() <= 2.0 ** -7 * c64.abs().max()
            c64.copy_(c.cpu())

    with torch.no_grad():
        for i in range(3):
            step(i)
            check(m(xs, cache, ss, tb, ln))
        ss.fill_(-1)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                m(xs, cache, ss, tb, ln)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = m(xs, cache, ss, tb, ln)
        for i in range(3, 12):
            step(i)
            graph.replay()
            check(y)
            torch.randn(1000, 1000, device=dev).sum().item()


def test_two_graphs_one_pool(dev):
    """Two captured calls that share their graph pool, replayed in turns."""
    cases = []
    for i, lengths in enumerate(([4000, 17], [100, 3000])):
        k, v, table, ln = make_cache(dev, lengths, 2, 128, 16, seed=60 + i)
        q = torch.randn(2, 16, 128, generator=gen(60 + i)).to(BF).to(dev)
        x = torch.randn(2, 4096, generator=gen(62 + i)).to(BF).to(dev)
        w = tbf16.prepare_weight_i8(torch.randn(512, 4096, generator=gen(64 + i)).to(BF).to(dev))
        cases.append((q, k, v, table, ln, x, w))
    run = lambda c: (tbf16.paged_sdpa(*c[:5]), tbf16.int8_linear(c[5], *c[6]))  # noqa: E731
    want = [run(c) for c in cases]
    pool, graphs, outs = None, [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(run(c))
        pool = pool or graph.pool()
        graphs.append(graph)
    for _ in range(4):
        for graph, out, w in zip(graphs, outs, want):
            for t in out:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1])


def test_int8_module(dev):
    torch.manual_seed(1)
    lin = nn.Linear(200, 104).to(BF).to(dev)
    w, b = lin.weight.detach().clone(), lin.bias.detach().clone()
    m = tbf16.convert(nn.Sequential(lin), sdpa=False, int8=True)
    assert isinstance(m[0], tbf16.Int8Linear) and set(m.state_dict()) == {"0.weight8", "0.weight_scale", "0.bias"}
    x = torch.randn(3, 20, 200).to(BF).to(dev)
    with torch.no_grad():
        y = m(x)
    check_linear(x, w, b, y=y)
    # reloaded, and moved (the rows' padding is lost): the same bits
    fresh = tbf16.convert(nn.Sequential(nn.Linear(200, 104).to(BF).to(dev)), sdpa=False, int8=True)
    fresh.load_state_dict(m.state_dict())
    moved = fresh.cpu().to(dev)
    with torch.no_grad():
        assert torch.equal(moved(x), y)
    # a gradient, and another dtype, go through the native op on the rebuilt weight
    x2 = x.detach().requires_grad_()
    m(x2).sum().backward()
    assert torch.allclose(x2.grad.float(), m[0].weight.float().sum(0).expand_as(x), rtol=0.02, atol=0.02)
    assert m(x.float()).dtype == torch.float32
    # weights are off by half a code
    assert ((m[0].weight.double() - w.double()).abs() <= (0.5 + 2.0 ** -8 * 128) * m[0].weight_scale[:, None]).all()
