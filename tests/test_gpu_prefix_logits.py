"""paged_sdpa_prefix on the GPU where the logits are known to the last bit: keys whose products with the queries
are whole numbers times a power of two, so that only what comes after them has to be allowed for."""
import numpy as np
import pytest
import torch

import tbf16

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
U23 = 2.0 ** -23


def gen(seed):
    return torch.Generator().manual_seed(seed)


def codes(z):
    """Whole numbers below 2^24 in size as three of at most 8 bits: z = z2 2^16 + z1 2^8 + z0."""
    return torch.stack((z >> 16, z >> 8 & 255, z & 255), -1)


def make(dev, far, own, H, D, page, power=0, seed=0, room=0):
    """Arguments of paged_sdpa_prefix where key j's product with every query of its head is z[j] 2^power: far
    (Hkv, n) and own, of each sequence (Hkv, n), hold the z. Sums of a query's three products are whole numbers below
    2^24, so exact in any order. Pages in random order, `room` more in the tables, rows that no position uses NaN."""
    g = gen(seed)
    Hkv, B = far.shape[0], len(own)
    need = [-(-z.shape[1] // page) for z in (far, *own)]
    pages = sum(need) + 1
    order = torch.randperm(pages, generator=g).int()
    k, v = (torch.full((pages, Hkv, page, D), float("nan"), dtype=BF) for _ in "kv")
    tables, at = [], 0
    for z, p in zip((far, *own), need):
        mine = order[at:at + p]
        at += p
        tables.append(mine)
        j = torch.arange(z.shape[1])
        rows = torch.zeros(z.shape[1], Hkv, D)
        rows[:, :, :3] = codes(z).transpose(0, 1).float()
        k[mine[j // page].long(), :, j % page] = rows.to(BF)
        v[mine[j // page].long(), :, j % page] = torch.randn(z.shape[1], Hkv, D, generator=g).to(BF)
    table = torch.full((B, max(need[1:]) + room), -1, dtype=torch.int32)
    for b, mine in enumerate(tables[1:]):
        table[b, :len(mine)] = mine
    q = torch.zeros(B, H, D)
    q[:, :, :3] = torch.tensor([2.0 ** (16 + power), 2.0 ** (8 + power), 2.0 ** power])
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    prefix = torch.cat((tables[0], torch.full((room,), -1, dtype=torch.int32)))
    return [t.to(dev) for t in (q.to(BF), k, v, prefix, i32([far.shape[1]]), table, i32([z.shape[1] for z in own]))]


def values_of(a, n, table):
    """The n values of a table's positions, (Hkv, n, D) in 64 bits."""
    j = torch.arange(n)
    v, page = a[2].cpu(), a[2].shape[2]
    return v[table.cpu().long()[j // page], :, j % page].transpose(0, 1).double()


def expected(a, far, own, power, scale, weight_bits=None):
    """(o, bound, weights' part of it) in 64 bits, with logits as the operators define them: fp32 products with scale
    log2(e). What may be off, of sum_j p_j |v_j| / sum_j p_j:
      2^-23 (d_j + 6)       a weight 2^-d_j: the rounding of d_j, of differences of maxima, exp2's of the weight and of
                            two joins
      2^-23 (n / 32 + 64)   n weighted values added 32 at a time, parts and joins
    and half a bf16 step of o."""
    c = np.float32(np.float32(scale) * np.float32(1.4426950408889634))
    H = a[0].shape[1]
    o, bound = [], []
    vf = values_of(a, far.shape[1], a[3])
    for b, z in enumerate(own):
        v = torch.cat((vf, values_of(a, z.shape[1], a[5][b])), 1)
        s = torch.cat((far, z), 1).numpy().astype(np.float32) * np.float32(2.0 ** power)  # exact
        x = torch.from_numpy((s * c).astype(np.float64))
        d = x.amax(1, keepdim=True) - x
        p = torch.exp2(-d)
        p = p / p.sum(1, keepdim=True)
        e = p * U23 * (d.clamp(max=1100) + 6 + v.shape[1] / 32 + 64)
        ref = (p[:, None] @ v)[:, 0]
        o.append(ref)
        bound.append(2.0 ** -8 * ref.abs() + (e[:, None] @ v.abs())[:, 0] + ref.abs() * e.sum(1, keepdim=True))
    rows = lambda t: torch.stack(t).repeat_interleave(H // far.shape[0], 1)  # noqa: E731
    return rows(o), rows(bound)


def close(o, ref, bound):
    """Within the bound, which leaves most outputs less than a fiftieth of themselves."""
    assert (bound <= ref.abs() / 50).double().mean() > 0.9
    assert torch.isfinite(o).all()
    err = (o.cpu().double() - ref).abs()
    assert (err <= bound).all(), (err - bound).max()


# B, H, Hkv, D: blocks of 64 and of 128 rows, head dims up to 64, 128 and 256, whole or padded
FORMS = [(2, 4, 2, 64), (33, 8, 2, 64), (3, 2, 1, 128), (33, 8, 2, 128), (5, 4, 2, 256), (3, 4, 1, 72), (40, 4, 1, 200), (2, 2, 2, 40)]


@pytest.mark.parametrize("B,H,Hkv,D", FORMS)
@pytest.mark.parametrize("n,first,second", [(2, 0, 1), (128, 5, 6), (128, 70, 3), (131, 1, 130), (640, 633, 20)])
def test_weights_keep_their_bits(dev, B, H, Hkv, D, n, first, second):
    """Two keys of almost one logit and values of 1 and -1: the output is the difference of their weights, about
    2^-14 of them. A weight may be off by 2^-23 (exp2), 2^-20 (the exponent, of up to 16 + 8), and 6 sums' 2^-23: less than 2^-19 in all,
    and half a bf16 step of the output is 2^-22. The other keys' weights are zero."""
    g = gen(n + D)
    z = torch.full((Hkv, n), -2 ** 23, dtype=torch.int64)
    z[:, first] = torch.randint(0, 2 ** 14, (Hkv,), generator=g)
    z[:, second] = z[:, first] + 1
    a = make(dev, z, [torch.zeros(Hkv, 0, dtype=torch.int64)] * B, H, D, 16, power=-13)
    q, k, v, table = a[0], a[1], a[2], a[3].long()
    # a query's own power of two: differences of 2^-13 to 2^-17, so that each row has weights of its own
    q.mul_(torch.exp2(-torch.randint(0, 5, (B, H, 1), generator=g).float()).to(dev))
    for at, sign in ((first, 1.0), (second, -1.0)):
        v[table[at // 16], :, at % 16] = sign
    o = tbf16.paged_sdpa_prefix(*a, scale=1.0).cpu().double()
    step = q.cpu().double()[:, :, 2]
    ref = torch.tanh(-step / 2)[..., None].expand(B, H, D)
    assert (ref.abs() < 2.0 ** -13).all()
    assert ((o - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -19).all(), (o - ref).abs().max() * 2.0 ** 19


def near_the_top(g, Hkv, n, sign):
    """Of n logits most differ from the largest, 2^23, by up to 7, some are zero."""
    z = sign * (2 ** 23 - 1 - torch.randint(0, 8, (Hkv, n), generator=g))
    return torch.where(torch.rand(Hkv, n, generator=g) < 0.1, 0 if sign > 0 else -2 ** 23, z)


@pytest.mark.parametrize("B,H,Hkv,D", FORMS)
@pytest.mark.parametrize("power,scale", [(-16, 1.0), (-13, 0.7), (-10, 1.0), (-4, 1.0), (-1, 1.0), (0, 1.0), (3, 1.0), (4, 0.09), (5, 1.0),
                                         (8, -1.0), (20, 1.0), (40, 0.125), (103, 1.0), (103, 1e-30), (0, 0.0)])
def test_large_logits(dev, B, H, Hkv, D, power, scale):
    """Logits up to 2^126 of which many are equal or neighbours, in the prefix and among the own keys: the same
    weights wherever a key lies, as paged_sdpa gives on tables that hold all of them."""
    g = gen(power + D)
    sign = -1 if power == 4 else 1
    far = near_the_top(g, Hkv, 208, sign)
    own = [near_the_top(g, Hkv, b % 40, sign) for b in range(B)]
    a = make(dev, far, own, H, D, 16, power, seed=D)
    ref, bound = expected(a, far, own, power, scale)
    close(tbf16.paged_sdpa_prefix(*a, scale=scale), ref, bound)
    q, k, v, table, _, tables, lengths = a
    close(tbf16.paged_sdpa(q, k, v, torch.cat((table.expand(B, -1), tables), 1), lengths + 208, scale=scale), ref, bound)


@pytest.mark.parametrize("B,H,Hkv,D", FORMS)
@pytest.mark.parametrize("step", [1, 16, 3 * 64, 40 * 64, 8000])
@pytest.mark.parametrize("falling", [False, True])
def test_maximum_that_moves(dev, B, H, Hkv, D, step, falling):
    """Logits that grow or fall by 1/64 to 125 from key to key."""
    j = torch.arange(1000).expand(Hkv, 1000)
    far = (999 - j if falling else j) * step
    own = [torch.randint(990 * step, 1001 * step, (Hkv, b % 7), generator=gen(b)) for b in range(B)]
    a = make(dev, far, own, H, D, 16, power=-6, seed=step)
    close(tbf16.paged_sdpa_prefix(*a, scale=1.0), *expected(a, far, own, -6, 1.0))


@pytest.mark.parametrize("B,H,Hkv,D", FORMS)
@pytest.mark.parametrize("power", [-16, 2, 6, 60])
def test_largest_values_at_large_logits(dev, B, H, Hkv, D, power):
    """Equal logits of any size with values near the type's largest: their sum has room."""
    far = torch.full((Hkv, 150), 2 ** 23 - 1)
    own = [torch.full((Hkv, b % 5), 2 ** 23 - 1) for b in range(B)]
    a = make(dev, far, own, H, D, 16, power)
    a[2].masked_fill_(~torch.isnan(a[2]), 3e38)
    close(tbf16.paged_sdpa_prefix(*a, scale=1.0), *expected(a, far, own, power, 1.0))


@pytest.mark.parametrize("B,H,Hkv,D", FORMS)
def test_large_tables_of_small_logits_and_one_large(dev, B, H, Hkv, D):
    """A key of 2^30 far behind 300 small ones, and before them."""
    for at in (299, 64, 0):
        far = torch.randint(0, 2 ** 10, (Hkv, 300), generator=gen(at))
        far[:, at] = 2 ** 23 - 1
        own = [torch.randint(0, 2 ** 10, (Hkv, b % 9), generator=gen(b)) for b in range(B)]
        a = make(dev, far, own, H, D, 16, power=7)
        close(tbf16.paged_sdpa_prefix(*a, scale=1.0), *expected(a, far, own, 7, 1.0))


def expected_of_rows(a, far, own, power, scale):
    """expected() with a power of its own for each query, (B, H)."""
    ref, bound = torch.empty(a[0].shape, dtype=torch.float64), torch.empty(a[0].shape, dtype=torch.float64)
    for t in power.unique().tolist():
        r, e = expected(a, far, own, t, scale)
        ref[power == t], bound[power == t] = r[power == t], e[power == t]
    return ref, bound


@pytest.mark.parametrize("B,H,Hkv,D", FORMS)
@pytest.mark.parametrize("most", [12, 30, 100])
def test_rows_of_every_size_side_by_side(dev, B, H, Hkv, D, most):
    """Queries of a power of two each, so that one wave has small logits, large ones, and some around where the maximum
    follows at once."""
    g = gen(most + D)
    far, own = near_the_top(g, Hkv, 208, 1), [near_the_top(g, Hkv, b % 40, 1) for b in range(B)]
    a = make(dev, far, own, H, D, 16, power=-16, seed=D)
    up = torch.randint(0, most, (B, H), generator=g)
    a[0].mul_(torch.exp2(up.float())[..., None].to(dev))
    for scale in (1.0, -1.0):
        close(tbf16.paged_sdpa_prefix(*a, scale=scale), *expected_of_rows(a, far, own, up - 16, scale))
