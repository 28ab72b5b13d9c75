"""Int8Linear through what programs do to modules: casts, moves, loading. No GPU (the weight is
quantised here by the 64-bit oracle)."""
import copy
import importlib

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


def test_rounded_scales_are_refused(module, monkeypatch):
    monkeypatch.setattr(int8, "_device", lambda *a: 0)
    m, w8, ws = module
    x = torch.zeros(2, m.in_features, dtype=BF)
    for t in (BF, torch.float16, torch.int32):
        with pytest.raises(TypeError, match="fp32 scales"):
            tbf16.int8_linear(x, w8, ws.to(t))
