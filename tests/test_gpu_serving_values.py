"""paged_sdpa where single weights and values decide the output: weights whose difference is what
is left of them. Every form of the kernel: head dims of 64, 128 and 256 and below, one to four
blocks of 16 query heads, a block per unit and equal runs of the list of tiles."""
import pytest
import torch

import tbf16

from _serving64 import paged_sdpa64

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
# H, Hkv, D: (DP, RT) of (64, 1), (64, 2), (64, 4), (128, 1), (128, 2), (256, 1); rows of D padded and not
FORMS = [(8, 2, 64), (6, 1, 40), (24, 1, 64), (64, 1, 64), (50, 1, 56), (16, 4, 128), (8, 1, 80), (32, 1, 128), (40, 2, 96),
         (16, 1, 256), (4, 2, 160)]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def cache_of(dev, k, v, wide):
    """k, v (B, n, Hkv, D) as a cache of pages of 16 in order; a table of a page more than needed, or
    (wide) of so many that the list form runs."""
    B, n, Hkv, D = k.shape
    need = -(-n // 16)

    def pages(t):
        full = torch.full((B, need * 16, Hkv, D), float("nan"), dtype=BF)
        full[:, :n] = t
        return full.view(B * need, 16, Hkv, D).transpose(1, 2).contiguous().to(dev)

    table = torch.full((B, 200 if wide else need + 1), -1, dtype=torch.int32)
    table[:, :need] = torch.arange(B * need, dtype=torch.int32).view(B, need)
    return pages(k), pages(v), table.to(dev), torch.full((B,), n, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("H,Hkv,D", FORMS)
@pytest.mark.parametrize("wide", [False, True])
def test_attend_weights_that_cancel(dev, H, Hkv, D, wide):
    """Two keys of almost the same weight and opposite values: the output is the difference of the
    weights, 2^-10 to 2^-13 of either, so it shows what the weights lose on their way to it."""
    B = 6
    q = torch.randn(B, H, D, generator=gen(H)).to(BF)
    k = torch.zeros(B, 2, Hkv, D)
    k[:, 1] = torch.randn(B, Hkv, D, generator=gen(D)) * 2.0 ** -10
    r = torch.randn(B, Hkv, D, generator=gen(1)).to(BF)
    args = (q.to(dev), *cache_of(dev, k.to(BF), torch.stack((r, -r), 1), wide))
    o = tbf16.paged_sdpa(*args).cpu().double()
    ref, _ = paged_sdpa64(*args)
    # before the rounding to bf16 an output is off by at most 2^-20 of r: exp2 1 ulp (2^-23) of a weight of
    # at most 1, the logit behind it below 2^-24, and 8 fp32 roundings of sums of at most r
    bound = 2.0 ** -8 * ref.abs() + 2.0 ** -20 * r.abs().repeat_interleave(H // Hkv, 1).double()
    err = (o - ref).abs()
    assert (err <= bound).all(), ((err - bound).max(), err.max())
    assert ref.abs().median() < 2.0 ** -10  # (the difference is what is tested)


@pytest.mark.parametrize("D", [136, 152, 168, 184, 216, 232, 248])
@pytest.mark.parametrize("wide", [False, True])
def test_attend_rows_of_half_a_chunk(dev, D, wide):
    """Head dims past 128 whose last chunk of 16 is half there, up to the cache's last row."""
    B, n, Hkv = 3, 48, 2
    k, v = (torch.randn(B, n, Hkv, D, generator=gen(D + i)).to(BF) for i in range(2))
    q = torch.randn(B, 6, D, generator=gen(D + 2)).to(BF)
    args = (q.to(dev), *cache_of(dev, k, v, wide))
    o = tbf16.paged_sdpa(*args).cpu().double()
    ref, bound = paged_sdpa64(*args)
    err = (o - ref).abs()
    assert (err <= bound).all(), (err - bound).max()


@pytest.mark.parametrize("H,Hkv,D", FORMS)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("n", [1, 2, 40, 200])
def test_attend_infinite_values(dev, H, Hkv, D, wide, n):
    """An infinite value makes its element infinite whatever the weight's bits (a weight of 1 for the
    largest key, or for the only one), infinities of both signs and NaN make it NaN, and every other
    element keeps its bits."""
    B = 4
    q = torch.randn(B, H, D, generator=gen(H)).to(BF)
    k, v = (torch.randn(B, n, Hkv, D, generator=gen(D + i)).to(BF) for i in range(2))
    k[1] = 0  # every weight 1
    clean = tbf16.paged_sdpa(q.to(dev), *cache_of(dev, k, v, wide)).cpu()
    bad = v.clone()
    rows = [0, n // 2, n - 1]
    for i, j in enumerate(rows):
        bad[:, j, :, i] = float("inf")
        bad[:, j, :, 3 + i] = -float("inf")
        bad[:, j, :, D - 1 - i] = float("nan")
    bad[:, 0, :, 6], bad[:, n - 1, :, 6] = float("inf"), -float("inf")
    args = (q.to(dev), *cache_of(dev, k, bad, wide))
    o = tbf16.paged_sdpa(*args).cpu()
    ref, _ = paged_sdpa64(*args)
    for c in range(D):
        r = ref[..., c]
        if torch.isfinite(r).all():
            assert torch.equal(o[..., c], clean[..., c]), c
        else:
            assert not torch.isfinite(r).any()
            assert torch.equal(o[..., c].nan_to_num(7.0, 1.0, -1.0).double(), r.nan_to_num(7.0, 1.0, -1.0)), c
    assert (ref[..., :3] == float("inf")).all() and (ref[..., 3:6] == -float("inf")).all()


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("first", [False, True])
def test_attend_infinite_value_of_a_small_weight(dev, wide, first):
    """Weights down to 2^-90 of the largest, before and behind the largest key."""
    n, D = 300, 128
    q = torch.zeros(1, 4, D)
    q[..., 0] = 1
    k = torch.zeros(1, n, 1, D)
    far = torch.arange(1, 91.0)  # key i's weight is 2^-i of the largest
    at = torch.arange(200, 290) if first else torch.arange(5, 95)
    k[0, :, 0, 0] = -120 * D ** 0.5
    k[0, 2 if first else 298, 0, 0] = 0
    k[0, at, 0, 0] = -far * D ** 0.5
    v = torch.randn(1, n, 1, D, generator=gen(3)).to(BF)
    v[0, at, 0, torch.arange(90)] = float("inf")
    k = k.to(BF)
    args = (q.to(BF).to(dev), *cache_of(dev, k, v, wide))
    o = tbf16.paged_sdpa(*args, scale=D ** -0.5 * 0.6931).cpu()
    assert (o[..., :90] == float("inf")).all() and torch.isfinite(o[..., 90:]).all()


@pytest.mark.parametrize("H,Hkv,D", FORMS)
@pytest.mark.parametrize("wide", [False, True])
def test_attend_values_near_the_largest(dev, H, Hkv, D, wide):
    """Weights that grow along the keys, over values whose weighted mean bf16 holds."""
    n = 190
    q = torch.zeros(2, H, D)
    q[..., 0] = 1
    k = torch.zeros(2, n, Hkv, D)
    k[..., 0] = (torch.arange(n) / 4).view(n, 1)  # a weight 2^(1/4) of the one before it, 2^8 a tile
    v = (torch.rand(2, n, Hkv, D, generator=gen(D)) + 1) * 2.0 ** 125  # the weights' sum is at most 7 of the largest's
    args = (q.to(BF).to(dev), *cache_of(dev, k.to(BF), v.to(BF), wide))
    scale = 0.6931
    o = tbf16.paged_sdpa(*args, scale=scale).cpu().double()
    ref, bound = paged_sdpa64(*args, scale=scale)
    assert torch.isfinite(ref).all() and ((o - ref).abs() <= bound).all()
