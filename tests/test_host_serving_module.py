"""Int8Linear through what programs do to modules: casts, moves, loading. No GPU (the weight is
quantised here by the 64-bit oracle)."""
import copy
import importlib
import io

import pytest
import torch
import torch.nn as nn

import tbf16
from tbf16 import int8

from _serving64 import codes64

BF = torch.bfloat16
convert = importlib.import_module("tbf16.convert")  # (the package's attribute of that name is the function)


@pytest.fixture(params=[(64, 24), (1000, 33), (7, 5)], ids=str)
def module(request, monkeypatch):
    K, N = request.param

    def prepare(w):
        codes, scale = codes64(w)
        rows = torch.zeros(w.shape[0], -(-w.shape[1] // 16) * 16, dtype=torch.int8)
        rows[:, :w.shape[1]] = codes.to(torch.int8)
        return rows[:, :w.shape[1]], scale[:, 0].float()

    monkeypatch.setattr(convert, "prepare_weight_i8", prepare)
    torch.manual_seed(K)
    m = tbf16.Int8Linear(nn.Linear(K, N).to(BF))
    return m, m.weight8.clone(), m.weight_scale.clone()


def unchanged(m, w8, ws):
    assert m.weight8.dtype == torch.int8 and torch.equal(m.weight8, w8)
    assert m.weight_scale.dtype == torch.float32 and torch.equal(m.weight_scale, ws)
    assert m.weight8.shape == (m.out_features, m.in_features)
    # and its rows are read in place, without a copy a call
    rows, ld = int8._weight_rows(m.weight8, m.in_features)
    assert rows is m.weight8 and ld % 16 == 0
    assert set(m.state_dict()) == {"weight8", "weight_scale", "bias"}


@pytest.mark.parametrize("cast", [lambda m: m.to(BF), lambda m: m.half(), lambda m: m.double(), lambda m: m.float(),
                                  lambda m: m.type(BF), lambda m: m.to(BF).half().float()])
def test_casts_keep_the_weight(module, cast):
    m, w8, ws = module
    seq = nn.Sequential(m, nn.Linear(3, 3).to(BF))
    cast(seq)
    unchanged(m, w8, ws)
    assert m.bias.dtype == seq[1].weight.dtype  # what is a parameter is cast


def test_moves_and_copies_keep_the_weight(module):
    m, w8, ws = module
    unchanged(copy.deepcopy(m), w8, ws)
    unchanged(copy.deepcopy(m).share_memory(), w8, ws)
    m.to("cpu", BF)
    unchanged(m, w8, ws)
    m._apply(lambda t: t.contiguous().clone())  # as a move to another device does
    unchanged(m, w8, ws)
    gone = copy.deepcopy(m).to("meta")
    assert gone.weight8.dtype == torch.int8 and gone.weight_scale.dtype == torch.float32
    back = gone.to_empty(device="cpu")
    back.load_state_dict(m.state_dict())
    unchanged(back, w8, ws)


@pytest.mark.parametrize("assign", [False, True])
@pytest.mark.parametrize("dense", [False, True])
def test_loading_keeps_the_rows(module, assign, dense):
    m, w8, ws = module
    f = io.BytesIO()
    torch.save({k: v.contiguous() if dense else v for k, v in m.state_dict().items()}, f)
    f.seek(0)
    other = copy.deepcopy(m)
    other.weight8.zero_()
    other.weight_scale.zero_()
    other.load_state_dict(torch.load(f, weights_only=True), assign=assign)
    unchanged(other, w8, ws)


def test_rounded_scales_are_refused(module, monkeypatch):
    monkeypatch.setattr(int8, "_device", lambda *a: 0)
    m, w8, ws = module
    x = torch.zeros(2, m.in_features, dtype=BF)
    for t in (BF, torch.float16, torch.int32):
        with pytest.raises(TypeError, match="fp32 scales"):
            tbf16.int8_linear(x, w8, ws.to(t))


def test_padded_rows():
    """Rows that the kernels read in place are left alone; others are copied, values unchanged."""
    w = torch.randint(-127, 128, (6, 200), dtype=torch.int8)
    for bad in (w, w[:, :199], w.t().contiguous().t(), torch.zeros(6 * 208 + 1, dtype=torch.int8)[1:].view(6, 208)):
        p = int8.padded_rows(bad)
        assert p is not bad and torch.equal(p, bad) and int8.padded_rows(p) is p
    for good in (w[:, :192].contiguous(), torch.zeros(5, 16, dtype=torch.int8), w[:, :0], torch.zeros(0, 16, dtype=torch.int8)):
        assert int8.padded_rows(good) is good
