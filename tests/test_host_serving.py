"""Refusals of the serving operators, raised on the host before any launch, and the C entry
points' own checks; no GPU."""
import pytest
import torch
import torch.nn as nn

import tbf16
from tbf16 import _ext, int8, paged

BF = torch.bfloat16


def args(pages=4, Hkv=2, page=16, D=64, B=3, H=4, n=2):
    return {"q": torch.zeros(B, H, D, dtype=BF), "k_cache": torch.zeros(pages, Hkv, page, D, dtype=BF),
            "v_cache": torch.zeros(pages, Hkv, page, D, dtype=BF), "page_table": torch.zeros(B, n, dtype=torch.int32),
            "lengths": torch.zeros(B, dtype=torch.int32)}


def wargs(T=5, Hkv=2, D=64):
    a = args(Hkv=Hkv, D=D)
    return {"k_cache": a["k_cache"], "v_cache": a["v_cache"], "k": torch.zeros(T, Hkv, D, dtype=BF),
            "v": torch.zeros(T, Hkv, D, dtype=BF), "slots": torch.zeros(T, dtype=torch.int32)}


@pytest.fixture
def host(monkeypatch):
    """The operators' checks with the one for the device left out (tensors here are on the CPU)."""
    monkeypatch.setattr(paged, "_same_device", lambda *a: None)
    monkeypatch.setattr(int8, "_device", lambda *a: 0)


CACHE = [  # what is wrong, the error, part of its text
    (dict(k_cache=torch.zeros(4, 2, 16, 64)), TypeError, "bf16 cache"),
    (dict(v_cache=torch.zeros(4, 2, 16, 72, dtype=BF)), ValueError, "one shape"),
    (dict(v_cache=torch.zeros(5, 2, 16, 64, dtype=BF)), ValueError, "one shape"),
    (dict(k_cache=torch.zeros(8, 16, 64, dtype=BF), v_cache=torch.zeros(8, 16, 64, dtype=BF)), ValueError, "one shape"),
    (dict(k_cache=torch.zeros(4, 2, 16, 60, dtype=BF), v_cache=torch.zeros(4, 2, 16, 60, dtype=BF)), ValueError, "head dim"),
    (dict(k_cache=torch.zeros(4, 2, 16, 264, dtype=BF), v_cache=torch.zeros(4, 2, 16, 264, dtype=BF)), ValueError, "head dim"),
    (dict(k_cache=torch.zeros(4, 2, 0, 64, dtype=BF), v_cache=torch.zeros(4, 2, 0, 64, dtype=BF)), ValueError, "holds nothing"),
    (dict(k_cache=torch.zeros(4, 2, 64, 16, dtype=BF).transpose(2, 3)), ValueError, "contiguous"),
    (dict(k_cache=torch.zeros(4, 2, 16, 68, dtype=BF)[..., :64]), ValueError, "contiguous"),
    (dict(v_cache=torch.zeros(4 * 2 * 16 * 64 + 1, dtype=BF)[1:].view(4, 2, 16, 64)), ValueError, "aligned"),
]


@pytest.mark.parametrize("wrong,error,text", CACHE)
def test_cache_refusals(host, wrong, error, text):
    with pytest.raises(error, match=text):
        tbf16.paged_sdpa(**{**args(), **wrong})
    with pytest.raises(error, match=text):
        tbf16.paged_write(**{**wargs(), **wrong})


@pytest.mark.parametrize("wrong,error,text", [
    (dict(q=torch.zeros(3, 4, 1, 64, dtype=BF)), ValueError, "is not"),
    (dict(q=torch.zeros(3, 4, 72, dtype=BF)), ValueError, "is not"),
    (dict(q=torch.zeros(3, 4, 64)), TypeError, "bf16 q"),
    (dict(q=torch.zeros(3, 5, 64, dtype=BF)), ValueError, "query heads"),
    (dict(q=torch.zeros(3, 0, 64, dtype=BF)), ValueError, "query heads"),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int64)), TypeError, "int32"),
    (dict(page_table=torch.zeros(6, dtype=torch.int32)), TypeError, "int32"),
    (dict(page_table=torch.zeros(2, 2, dtype=torch.int32)), ValueError, "sequences"),
    (dict(lengths=torch.zeros(3)), TypeError, "int32"),
    (dict(lengths=torch.zeros(4, dtype=torch.int32)), ValueError, "sequences"),
])
def test_attend_refusals(host, wrong, error, text):
    with pytest.raises(error, match=text):
        tbf16.paged_sdpa(**{**args(), **wrong})


def test_write_refusals(host):
    a = wargs()
    one = a["k_cache"]
    both = torch.zeros(2, 5, 2, 64, dtype=BF)
    for wrong, error, text in [
            (dict(k=torch.zeros(5, 2, 72, dtype=BF)), ValueError, "are not"),
            (dict(v=torch.zeros(6, 2, 64, dtype=BF)), ValueError, "are not"),
            (dict(k=torch.zeros(5, 128, dtype=BF), v=torch.zeros(5, 128, dtype=BF)), ValueError, "are not"),
            (dict(k=both[0].float(), v=both[1].float()), TypeError, "bf16 k"),
            (dict(slots=torch.zeros(5, dtype=torch.int64)), TypeError, "int32"),
            (dict(slots=torch.zeros(4, dtype=torch.int32)), ValueError, "4 slots for 5"),
            (dict(v_cache=one), ValueError, "same memory"),
            (dict(k_cache=one[:1].expand(4, 2, 16, 64)), ValueError, "expanded"),
            (dict(k=one[0].transpose(0, 1)[:5]), ValueError, "storage"),
    ]:
        with pytest.raises(error, match=text):
            tbf16.paged_write(**{**a, **wrong})


def test_int8_refusals(host):
    x, w8, ws = torch.zeros(3, 32, dtype=BF), torch.zeros(8, 32, dtype=torch.int8), torch.ones(8)
    for call, error, text in [
            (lambda: tbf16.int8_linear(x.float(), w8, ws), TypeError, "bf16 x"),
            (lambda: tbf16.int8_linear(x, w8.float(), ws), TypeError, "int8 weight"),
            (lambda: tbf16.int8_linear(x, w8[0], ws), TypeError, "int8 weight"),
            (lambda: tbf16.int8_linear(x[:, :16], w8, ws), ValueError, "K=16"),
            (lambda: tbf16.int8_linear(x, w8, ws[:7]), ValueError, "7 scales"),
            (lambda: tbf16.int8_linear(x, w8, ws, torch.zeros(7)), ValueError, "bias"),
            (lambda: tbf16.int8_linear(torch.zeros(1, 131073, dtype=BF), torch.zeros(1, 131073, dtype=torch.int8), ws[:1]),
             ValueError, "131072"),
            (lambda: tbf16.quantize_rows_i8(torch.zeros(1, 131073, dtype=BF)), ValueError, "131072"),
            (lambda: tbf16.quantize_rows_i8(x.float()), TypeError, "bf16"),
            (lambda: tbf16.quantize_rows_i8(x[0]), ValueError, "(R, K)"),
    ]:
        with pytest.raises(error, match=text.replace("(", r"\(").replace(")", r"\)")):
            call()


def test_host_tensors_are_refused():
    for call in (lambda: tbf16.paged_sdpa(**args()), lambda: tbf16.paged_write(**wargs()),
                 lambda: tbf16.int8_linear(torch.zeros(1, 16, dtype=BF), torch.zeros(1, 16, dtype=torch.int8), torch.ones(1)),
                 lambda: tbf16.prepare_weight_i8(torch.zeros(1, 16, dtype=BF))):
        with pytest.raises(ValueError, match="ROCm"):
            call()


def test_convert_int8_is_for_inference():
    with pytest.raises(ValueError, match="inference"):
        tbf16.convert(nn.Linear(8, 8), train=True, int8=True, force=True)


def test_abi_refusals():
    L = _ext.lib()
    err = lambda: L.tbf16_last_error().decode()  # noqa: E731
    s2, s3, odd2, odd3, far3 = (128, 64), (2048, 1024, 64), (128, 60), (2048, 1020, 64), (2 ** 31, 1024, 64)

    def attn(B=1, H=2, Hkv=2, D=64, qs=s2, kc=16, vc=16, pages=4, page=16, ks=s3, vs=s3, ws=16, wsb=None, q=16):
        if wsb is None:
            wsb = 1 << 40
        return L.tbf16_paged_attn(q, B, H, Hkv, D, *qs, kc, vc, pages, page, *ks, *vs, 16, 400, 400, 16, 1.0, 16, ws, wsb, None)

    for bad, text in [(dict(H=3), "multiple of key/value heads"), (dict(D=60), "multiple of 8"), (dict(D=264), "256"),
                      (dict(kc=18), "aligned"), (dict(ks=odd3), "strides"), (dict(qs=odd2), "q must"), (dict(q=24), "q must"),
                      (dict(page=0), "bad cache"), (dict(Hkv=0), "bad cache"), (dict(vs=far3), "stride"), (dict(B=-1), "bad shape"),
                      (dict(ws=24), "workspace")]:
        assert attn(**bad) == -1, bad
        assert text in err(), (bad, err())
    assert attn(B=64, H=64, Hkv=2, D=128, wsb=0) == -3 and "workspace" in err()
    assert attn(B=0) == 0
    assert L.tbf16_paged_attn_ws_bytes(1, 64, 2, 128, 100) == 0 < L.tbf16_paged_attn_ws_bytes(1, 64, 2, 128, 6400)

    def write(T=2, ks=s2, kc=16, cs=s3, D=64, k=16, pages=4):
        return L.tbf16_paged_write(k, 16, T, 2, D, *ks, *s2, 16, kc, 16, pages, 16, *cs, *s3, None)

    for bad, text in [(dict(T=-1), "tokens"), (dict(ks=odd2), "strides"), (dict(kc=8), "aligned"), (dict(k=8), "aligned"),
                      (dict(D=4), "multiple of 8"), (dict(cs=odd3), "strides"), (dict(pages=-1), "bad cache")]:
        assert write(**bad) == -1, bad
        assert text in err(), (bad, err())
    assert write(T=0) == 0 and write(pages=0) == 0

    def linear(M=2, K=32, ldx=32, w=16, N=8, ldw=32, y=16, ldy=8, ws=16, wsb=1 << 40):
        return L.tbf16_linear_i8(16, M, K, ldx, w, N, ldw, 16, None, y, ldy, ws, wsb, None)

    for bad, text in [(dict(K=131073, ldx=131073), "131072"), (dict(ldx=31), "row stride"), (dict(w=8), "weight rows"),
                      (dict(ldw=40), "weight rows"), (dict(K=33, ldx=33), "weight rows"), (dict(ldy=4), "rows of y"),
                      (dict(N=9), "rows of y"), (dict(y=8), "rows of y"), (dict(ws=None, M=100), "workspace"), (dict(ws=24), "workspace"), (dict(M=-1), "bad shape")]:
        assert linear(**bad) == -1, bad
        assert text in err(), (bad, err())
    assert linear(wsb=0, M=100) == -3 and "workspace" in err()
    assert linear(M=0) == 0 and linear(N=0) == 0
    assert L.tbf16_linear_i8_ws_bytes(0, 32, 8) == 0 and L.tbf16_linear_i8_ws_bytes(5, 33, 8) >= 5 * 48 + 20
    assert L.tbf16_quantize_rows_i8(16, 2, 33, 33, 16, 32, 16, None) == -1 and "padded" in err()
    assert L.tbf16_quantize_rows_i8(16, 2, 32, 32, 8, 32, 16, None) == -1
    assert L.tbf16_quantize_rows_i8(None, 0, 32, 32, None, 32, None, None) == 0
