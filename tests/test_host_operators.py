"""Refusals of the operators around the paged cache, on the host before any launch, and the C entry
points' own checks; no GPU."""
import pytest
import torch

import tbf16
from tbf16 import _ext, paged

from _operators64 import advance_by_hand

I32 = torch.int32


@pytest.fixture
def host(monkeypatch):
    """The operators' checks with the one for the device left out (tensors here are on the CPU)."""
    monkeypatch.setattr(paged, "_same_device", lambda *a: None)


def adv(B=3, n=4, pages=20):
    return {"page_table": torch.zeros(B, n, dtype=I32), "lengths": torch.zeros(B, dtype=I32), "counts": torch.zeros(B, dtype=I32),
            "free_pages": torch.zeros(pages, dtype=I32), "n_free": torch.zeros(1, dtype=I32), "page": 16, "tokens": 5}


packed = torch.zeros(100, dtype=I32)


@pytest.mark.parametrize("wrong,error,text", [
    (dict(page_table=torch.zeros(3, dtype=I32)), ValueError, "is not"),
    (dict(page_table=torch.zeros(3, 4)), TypeError, "page_table as int32"),
    (dict(page_table=torch.zeros(4, 3, dtype=I32).t()), ValueError, "rows must be"),
    (dict(page_table=torch.zeros(1, 4, dtype=I32).expand(3, 4)), ValueError, "rows must be"),
    (dict(lengths=torch.zeros(2, dtype=I32)), ValueError, "for 3 sequences"),
    (dict(lengths=torch.zeros(3, dtype=torch.int64)), TypeError, "lengths as int32"),
    (dict(lengths=torch.zeros(6, dtype=I32)[::2]), ValueError, "contiguous"),
    (dict(counts=torch.zeros(3, 1, dtype=I32)), ValueError, "for 3 sequences"),
    (dict(counts=torch.zeros(1, dtype=I32).expand(3)), ValueError, "contiguous"),
    (dict(free_pages=torch.zeros(4, 5, dtype=I32)), ValueError, "free_pages"),
    (dict(n_free=torch.zeros(2, dtype=I32)), ValueError, "one number"),
    (dict(prefix_length=torch.zeros(0, dtype=I32)), ValueError, "one number"),
    (dict(prefix_length=torch.zeros(1)), TypeError, "prefix_length as int32"),
    (dict(lengths=packed[:3], counts=packed[:3]), ValueError, "same memory"),
    (dict(free_pages=packed[:20], n_free=packed[19:20]), ValueError, "same memory"),
    (dict(page=0), ValueError, "positions"),
    (dict(page=2 ** 31), ValueError, "positions"),
    (dict(tokens=-1), ValueError, "room for"),
    (dict(tokens=2 ** 31), ValueError, "room for"),
])
def test_advance_refusals(host, wrong, error, text):
    with pytest.raises(error, match=text):
        tbf16.paged_advance(**{**adv(), **wrong})


def test_advance_packed_state_is_taken(host, monkeypatch):
    """One allocation for all of the state, its parts apart."""
    seen = []
    monkeypatch.setattr(paged, "launch", lambda *a: seen.append(a))
    a = adv()
    a.update(lengths=packed[:3], counts=packed[3:6], free_pages=packed[6:26], n_free=packed[26:27])
    slots, positions, starts = tbf16.paged_advance(**a)
    assert len(seen) == 1 and slots.shape == positions.shape == (5,) and starts.shape == (4,)


def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="ROCm"):
        tbf16.paged_advance(**adv())


def test_advance_abi_refusals():
    L = _ext.lib()
    err = lambda: L.tbf16_last_error().decode()  # noqa: E731

    def call(st=4, B=3, n=4, pages=20, nf=16, page=16, tokens=5, starts=16, ws=16, wsb=1000, table=16):
        return L.tbf16_paged_advance(table, st, B, n, 16, 16, 16, pages, nf, page, tokens, None, 16, 16, starts, ws, wsb, None)

    for bad, text in [(dict(B=-1), "table shape"), (dict(n=2 ** 31), "table shape"), (dict(n=2 ** 30), "table shape"),
                      (dict(st=3), "overlap"), (dict(page=0), "slots"), (dict(pages=2 ** 28), "slots"),
                      (dict(tokens=-1), "tokens"), (dict(tokens=2 ** 31), "tokens"), (dict(nf=None), "missing"),
                      (dict(starts=None), "missing"), (dict(ws=None), "missing"), (dict(table=18), "misaligned")]:
        assert call(**bad) == -1, bad
        assert text in err(), (bad, err())
    assert call(wsb=0) == -3 and "workspace" in err()
    assert L.tbf16_paged_advance_ws_bytes(100) >= 1200


def test_advance_by_hand():
    """The oracle's own cases: a page taken, given back, and who goes without."""
    table, lengths, stack = [[0, -1], [1, -1]], [3, 4], [9, 8, 5]
    got = advance_by_hand(table, lengths, [2, 1], stack, 3, 4, 5, 10)
    # page ids at or above the stack's size name no page: the cache has 3
    assert got == (1, [3, -1, -1, -1, -1], [13, 14, 14, -1, -1], [0, 2, 3])
    assert table == [[0, 5], [1, 8]] and lengths == [5, 5]
    table, lengths, stack = [[0, 2], [1, -1]], [5, 4], [3, 3, 3, 3]
    assert advance_by_hand(table, lengths, [-1, 1], stack, 0, 4, 2) == (0, [8, -1], [4, -1], [0, 0, 1])
    assert table == [[0, -1], [1, 2]] and lengths == [4, 5] and stack == [2, 3, 3, 3]
