"""paged_write on tensors of one allocation: refused where new tokens lie within the cache's rows,
taken where they lie apart. No GPU."""
import pytest
import torch

import tbf16
from tbf16 import paged

BF = torch.bfloat16


@pytest.fixture
def launches(monkeypatch):
    calls = []
    monkeypatch.setattr(paged, "_same_device", lambda *a: None)
    monkeypatch.setattr(paged, "launch", lambda name, *a: calls.append(name))
    return calls


def test_one_allocation(launches):
    pages, Hkv, page, D, T = 4, 2, 16, 64, 5
    n, t = pages * Hkv * page * D, T * Hkv * D
    slots = torch.zeros(T, dtype=torch.int32)
    arena = torch.zeros(2 * n + 3 * t, dtype=BF)
    cache = lambda at: arena[at:at + n].view(pages, Hkv, page, D)  # noqa: E731
    rows = lambda at: arena[at:at + t].view(T, Hkv, D)  # noqa: E731
    # keys, values, new keys, new values; and the new ones first, between and behind
    for kc, vc, k, v in [(0, n, 2 * n, 2 * n + t), (t, n + 2 * t, 0, n + t), (n, 0, 2 * n + 2 * t, 2 * n)]:
        tbf16.paged_write(cache(kc), cache(vc), rows(k), rows(v), slots)
    assert launches == ["tbf16_paged_write"] * 3
    own = torch.zeros(T, Hkv, D, dtype=BF)
    for k, v in [(rows(0), own), (own, rows(n)), (rows(n - 8), own), (own, rows(2 * n - t)), (rows(2 * n - 8), own)]:
        with pytest.raises(ValueError, match="storage"):
            tbf16.paged_write(cache(0), cache(n), k, v, slots)
    # both halves of one tensor, a row of new tokens at its end
    both = torch.zeros(pages + 1, 2, Hkv, page, D, dtype=BF)
    tbf16.paged_write(both[:pages, 0], both[:pages, 1], both[pages, 0, :, :T].transpose(0, 1), both[pages, 1, :, :T].transpose(0, 1),
                      slots)
    with pytest.raises(ValueError, match="storage"):
        tbf16.paged_write(both[:pages, 0], both[:pages, 1], both[1, 0, :, :T].transpose(0, 1), own, slots)
    assert len(launches) == 4
