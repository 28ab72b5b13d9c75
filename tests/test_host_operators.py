"""Refusals of the operators around the paged cache, on the host before any launch, and the C entry
points' own checks; no GPU."""
import pytest
import torch

import tbf16
from tbf16 import _ext, paged

from _operators64 import advance_by_hand, norm_rope64

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
    (dict(lengths=torch.zeros(3, dtype=torch.int64)), TypeError, "expected int32"),
    (dict(lengths=torch.zeros(6, dtype=I32)[::2]), ValueError, "contiguous"),
    (dict(counts=torch.zeros(3, 1, dtype=I32)), ValueError, "one dimension"),
    (dict(counts=torch.zeros(1, dtype=I32).expand(3)), ValueError, "contiguous"),
    (dict(free_pages=torch.zeros(4, 5, dtype=I32)), ValueError, "one dimension"),
    (dict(n_free=torch.zeros(2, dtype=I32)), ValueError, "one number"),
    (dict(prefix_length=torch.zeros(0, dtype=I32)), ValueError, "one number"),
    (dict(prefix_length=torch.zeros(1)), TypeError, "expected int32"),
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
                      (dict(starts=None), "missing"), (dict(table=18), "misaligned"), (dict(ws=18), "misaligned")]:
        assert call(**bad) == -1, bad
        assert text in err(), (bad, err())
    for bad in (dict(tokens=10 ** 5, wsb=0), dict(tokens=10 ** 5, ws=None), dict(B=5000, wsb=10 ** 4)):
        assert call(**bad) == -3 and "workspace" in err(), bad
    size = L.tbf16_paged_advance_ws_bytes
    assert size(100, 100) == 0 < size(100, 10 ** 5) < size(10 ** 4, 0) and size(0, 10 ** 5) > 0


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


BF = torch.bfloat16


def norm(S=5, H=4, Hkv=2, D=64, R=32, rows=10):
    return {"q": torch.zeros(S, H, D, dtype=BF), "k": torch.zeros(S, Hkv, D, dtype=BF), "q_weight": torch.ones(D, dtype=BF),
            "k_weight": torch.ones(D, dtype=BF), "cos": torch.ones(rows, R // 2), "sin": torch.zeros(rows, R // 2),
            "positions": torch.zeros(S, dtype=I32)}


@pytest.mark.parametrize("wrong,error,text", [
    (dict(q=torch.zeros(5, 64, dtype=BF)), ValueError, "are not"),
    (dict(q=torch.zeros(1, 1, 5, 4, 64, dtype=BF)), ValueError, "are not"),
    (dict(k=torch.zeros(6, 2, 64, dtype=BF)), ValueError, "are not"),
    (dict(k=torch.zeros(5, 2, 48, dtype=BF)), ValueError, "are not"),
    (dict(k=torch.zeros(5, 0, 64, dtype=BF)), ValueError, "are not"),
    (dict(q=torch.zeros(5, 4, 72, dtype=BF), k=torch.zeros(5, 2, 72, dtype=BF)), ValueError, "head dim 72"),
    (dict(q=torch.zeros(5, 4, 272, dtype=BF), k=torch.zeros(5, 2, 272, dtype=BF)), ValueError, "head dim 272"),
    (dict(q=torch.zeros(5, 4, 64)), TypeError, "bf16 q"),
    (dict(q_weight=torch.ones(32, dtype=BF)), ValueError, "weights"),
    (dict(q_weight=torch.ones(64)), TypeError, "weights both"),
    (dict(q_weight=torch.ones(64).half(), k_weight=torch.ones(64).half()), TypeError, "weights both"),
    (dict(cos=torch.ones(10, 8)), ValueError, "one shape"),
    (dict(cos=torch.ones(0, 16), sin=torch.ones(0, 16)), ValueError, "one shape"),
    (dict(cos=torch.ones(10, 16).double(), sin=torch.ones(10, 16).double()), TypeError, "fp32 cos"),
    (dict(cos=torch.ones(10, 12), sin=torch.ones(10, 12)), ValueError, "24 rotated"),
    (dict(cos=torch.ones(10, 40), sin=torch.ones(10, 40)), ValueError, "80 rotated"),
    (dict(cos=torch.ones(10, 0), sin=torch.ones(10, 0)), ValueError, "0 rotated"),
    (dict(positions=torch.zeros(5, dtype=torch.int64)), TypeError, "int32 positions"),
    (dict(positions=torch.zeros(4, dtype=I32)), ValueError, "positions"),
    (dict(eps=-1.0), ValueError, "eps"),
    (dict(eps=float("nan")), ValueError, "eps"),
    (dict(eps=float("inf")), ValueError, "eps"),
    (dict(), ValueError, "ROCm"),
])
@pytest.mark.parametrize("fn", [tbf16.qk_norm_rope, tbf16.autograd.qk_norm_rope])
def test_norm_rope_refusals(fn, wrong, error, text):
    with pytest.raises(error, match=text):
        fn(**{**norm(), **wrong})


def test_norm_rope_tables_have_no_gradient():
    a = norm()
    a["cos"] = a["cos"].requires_grad_()
    with pytest.raises(ValueError, match="no gradients of cos"):
        tbf16.autograd.qk_norm_rope(**a)


def test_norm_rope_abi_refusals():
    L = _ext.lib()
    err = lambda: L.tbf16_last_error().decode()  # noqa: E731
    st = 0, 64, 64

    def tail(rows=9, R=32, eps=1e-6, cos=16):
        return 16, 16, 0, cos, 16, rows, R, 16, 0, 1, eps, 0

    def fwd(B=1, S=2, H=4, Hkv=2, D=64, q=16, q_st=st, **kw):
        return L.tbf16_qk_norm_rope(q, 16, B, S, H, Hkv, D, *q_st, *st, *tail(**kw), 16, 16, None)

    def bwd(B=1, S=2, H=4, Hkv=2, D=64, q=16, q_st=st, ws=16, wsb=0, dwq=16, **kw):
        return L.tbf16_qk_norm_rope_bwd(q, 16, 16, 16, B, S, H, Hkv, D, *q_st, *st, *st, *st, *tail(**kw), None, None, dwq, None,
                                        ws, wsb, None)

    for bad, text in [(dict(B=-1), "tokens"), (dict(S=2 ** 31), "tokens"), (dict(H=0), "heads"), (dict(D=24), "head dim"),
                      (dict(D=272), "head dim"), (dict(R=8), "rotated"), (dict(R=0), "rotated"), (dict(R=80), "rotated"),
                      (dict(rows=0), "tables"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
                      (dict(q=24), "aligned"), (dict(q_st=(0, 64, 4)), "aligned"), (dict(cos=8), "misaligned")]:
        assert fwd(**bad) == -1 and text in err(), (bad, err())
        assert bwd(**bad) == -1 and text in err(), (bad, err())
    assert bwd() == -3 and "workspace" in err()
    assert bwd(ws=None, wsb=1 << 30) == -3
    assert fwd(B=0) == 0 and fwd(S=0) == 0 and bwd(S=0, dwq=None) == 0
    assert L.tbf16_qk_norm_rope_bwd_ws_bytes(2, 100, 4, 2, 64) > 0 == L.tbf16_qk_norm_rope_bwd_ws_bytes(0, 100, 4, 2, 64)


@pytest.mark.parametrize("near", [False, True])
def test_norm_rope64_against_differences(near):
    """The oracle's gradients by central differences, its rotation as a complex product."""
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(3, 2, 32, generator=g).double(), torch.randn(32, generator=g).double()
    ang = torch.rand(4, 8, generator=g).double() * 6
    pos = torch.tensor([2, -1, 0], dtype=I32)
    dy = torch.randn(3, 2, 32, generator=g).double()
    f = lambda x, w: norm_rope64(x, w, ang.cos(), ang.sin(), pos, 1e-3, near)[0]  # noqa: E731
    _, _, dx, _, dw, _ = norm_rope64(x, w, ang.cos(), ang.sin(), pos, 1e-3, near, dy)
    for t, grad in ((x, dx), (w, dw)):
        for _ in range(40):
            i = tuple(int(torch.randint(0, n, (), generator=g)) for n in t.shape)
            lo, hi = t.clone(), t.clone()
            lo[i] -= 1e-5
            hi[i] += 1e-5
            d = ((f(hi, w) - f(lo, w)) * dy).sum() / 2e-5 if t is x else ((f(x, hi) - f(x, lo)) * dy).sum() / 2e-5
            assert abs(d - grad[i]) <= 1e-7 * (1 + abs(grad[i]))
    y, z = f(x, w)[0, 0], x[0, 0] / torch.sqrt(x[0, 0].square().mean() + 1e-3) * w
    a, b = (z[0:16:2], z[1:16:2]) if near else (z[:8], z[8:16])
    turned = torch.complex(a, b) * torch.exp(1j * ang[2])
    got = torch.complex(y[0:16:2], y[1:16:2]) if near else torch.complex(y[:8], y[8:16])
    # (a quotient and a product with the reciprocal: a few roundings of 2^-53 of values below 8)
    assert (got - turned).abs().max() < 1e-14 and (y[16:] - z[16:]).abs().max() < 1e-14 and not f(x, w)[1].any()


def prefix(pages=4, Hkv=2, page=16, D=64, B=3, H=4, m=2, n=2):
    z = lambda *s, t=I32: torch.zeros(*s, dtype=t)  # noqa: E731
    return {"q": z(B, H, D, t=BF), "k_cache": z(pages, Hkv, page, D, t=BF), "v_cache": z(pages, Hkv, page, D, t=BF),
            "prefix_table": z(m), "prefix_length": z(1), "page_table": z(B, n), "lengths": z(B)}


@pytest.mark.parametrize("wrong,error,text", [
    (dict(k_cache=torch.zeros(4, 2, 16, 64)), TypeError, "bf16 cache"),
    (dict(v_cache=torch.zeros(4, 2, 16, 72, dtype=BF)), ValueError, "one shape"),
    (dict(k_cache=torch.zeros(4, 2, 16, 264, dtype=BF), v_cache=torch.zeros(4, 2, 16, 264, dtype=BF)), ValueError, "head dim"),
    (dict(q=torch.zeros(3, 4, 72, dtype=BF)), ValueError, "is not"),
    (dict(q=torch.zeros(3, 4, 64)), TypeError, "bf16 q"),
    (dict(q=torch.zeros(3, 5, 64, dtype=BF)), ValueError, "query heads"),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int64)), TypeError, "page_table as an int32"),
    (dict(page_table=torch.zeros(2, 2, dtype=I32)), ValueError, "sequences"),
    (dict(lengths=torch.zeros(4, dtype=I32)), ValueError, "sequences"),
    (dict(prefix_table=torch.zeros(1, 2, dtype=I32)), TypeError, "prefix_table as an int32"),
    (dict(prefix_table=torch.zeros(2)), TypeError, "prefix_table as an int32"),
    (dict(prefix_length=torch.zeros(3, dtype=I32)), TypeError, "one int32"),
    (dict(prefix_length=torch.zeros(1, dtype=torch.int64)), TypeError, "one int32"),
])
def test_prefix_refusals(host, wrong, error, text):
    with pytest.raises(error, match=text):
        tbf16.paged_sdpa_prefix(**{**prefix(), **wrong})


def test_prefix_host_tensors_are_refused():
    with pytest.raises(ValueError, match="ROCm"):
        tbf16.paged_sdpa_prefix(**prefix())


def test_prefix_abi_refusals():
    L = _ext.lib()
    err = lambda: L.tbf16_last_error().decode()  # noqa: E731
    s2, s3 = (128, 64), (2048, 1024, 64)

    def call(B=1, H=2, Hkv=2, D=64, qs=s2, kc=16, pages=4, page=16, ks=s3, vs=s3, pt=16, pn=100, n=400, ws=16, wsb=1 << 40, q=16):
        return L.tbf16_paged_attn_prefix(q, B, H, Hkv, D, *qs, kc, 16, pages, page, *ks, *vs, pt, pn, 16, 16, 400, n, 16, 1.0, 16,
                                         ws, wsb, None)

    for bad, text in [(dict(H=3), "multiple of key/value heads"), (dict(D=60), "multiple of 8"), (dict(D=264), "256"),
                      (dict(kc=18), "aligned"), (dict(ks=(2048, 1020, 64)), "strides"), (dict(vs=(2 ** 31, 1024, 64)), "stride"),
                      (dict(qs=(128, 60)), "q must"), (dict(q=24), "q must"), (dict(page=0), "bad cache"),
                      (dict(Hkv=0), "bad cache"), (dict(B=-1), "bad shape"), (dict(ws=24), "workspace"), (dict(ws=None), "workspace"),
                      (dict(pn=-1), "too wide"), (dict(n=2 ** 31), "too wide"), (dict(pt=6), "4-byte"), (dict(B=10 ** 9), "large")]:
        assert call(**bad) == -1, bad
        assert text in err(), (bad, err())
    assert call(B=64, wsb=0) == -3 and "workspace" in err()
    assert call(B=0) == 0
    small, large = (L.tbf16_paged_attn_prefix_ws_bytes(B, 32, 8, 128, 4096, 512) for B in (1, 64))
    assert 0 < small < large and L.tbf16_paged_attn_prefix_ws_bytes(0, 32, 8, 128, 4096, 512) == 0


def test_prefix_abi_more_outputs_than_a_launch_counts():
    """The join has 256 threads for 64 groups of four outputs, and a launch fewer than 2^32 threads."""
    L = _ext.lib()
    for B, H, D in ((2 ** 29 // 256, 256, 8), (2 ** 25 // 4, 4, 128), (2 ** 24 // 2, 2, 256)):
        assert L.tbf16_paged_attn_prefix_ws_bytes(B - 1, H, H, D, 64, 64) > 0
        assert L.tbf16_paged_attn_prefix_ws_bytes(B, H, H, D, 64, 64) == 0
        assert L.tbf16_paged_attn_prefix(16, B, H, H, D, H * D, D, 16, 16, 4, 16, 16 * H * D, 16 * D, D, 16 * H * D, 16 * D, D,
                                         16, 4, 16, 16, 4, 4, 16, 1.0, 16, 16, 1 << 60, None) == -1
        assert "large" in L.tbf16_last_error().decode()
