"""paged_sdpa_prefix with tables of a server's capacity: the plan goes by what a table has room for, so short prefixes
behind long tables run in the blocks, splits and lists that long ones run in."""
import pytest
import torch

import tbf16

from test_gpu_prefix import SHAPES, check, make
from test_gpu_prefix_logits import FORMS, close, expected, near_the_top
from test_gpu_prefix_logits import make as make_exact

pytestmark = pytest.mark.gpu


def wide(a, far, own):
    """The tables as wide as `far` and `own` positions need, the entries past those in use -1."""
    page, dev = a[1].shape[2], a[0].device
    pad = lambda t, n: torch.cat((t, torch.full((*t.shape[:-1], max(0, n // page - t.shape[-1])), -1, dtype=torch.int32, device=dev)), -1)  # noqa: E731
    return [*a[:3], pad(a[3], far), a[4], pad(a[5], own), a[6]]


@pytest.mark.parametrize("far,own", [(1 << 15, 64), (1 << 19, 300), (1 << 19, 5000)])
@pytest.mark.parametrize("H,Hkv,D,page,prefix,lengths", SHAPES)
def test_shapes_behind_long_tables(dev, H, Hkv, D, page, prefix, lengths, far, own):
    check(wide(make(dev, prefix, lengths, H, Hkv, D, page, seed=H + D + page), far, own))


@pytest.mark.parametrize("power,scale", [(-16, 1.0), (0, 1.0), (5, 1.0), (40, 0.125)])
@pytest.mark.parametrize("B,H,Hkv,D", FORMS)
def test_large_logits_behind_long_tables(dev, B, H, Hkv, D, power, scale):
    g = torch.Generator().manual_seed(power + D)
    far, own = near_the_top(g, Hkv, 208, 1), [near_the_top(g, Hkv, b % 40, 1) for b in range(B)]
    a = wide(make_exact(dev, far, own, H, D, 16, power, seed=D), 1 << 19, 5000)
    close(tbf16.paged_sdpa_prefix(*a, scale=scale), *expected(a, far, own, power, scale))


@pytest.mark.parametrize("B,H,Hkv,D", FORMS)
def test_infinite_values_behind_long_tables(dev, B, H, Hkv, D):
    a = wide(make(dev, 200, [20] * B, H, Hkv, D, 16, seed=10), 1 << 19, 5000)
    v, far = a[2], a[3].cpu().long()
    v[far[3], 0, 5, 7] = float("inf")
    v[far[9], Hkv - 1, 2, 3] = float("-inf")
    check(a)
