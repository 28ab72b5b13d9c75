"""Int8Linear on the GPU after what programs do to modules."""
import pytest
import torch
import torch.nn as nn

import tbf16
from tbf16 import int8

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.mark.parametrize("M", [1, 5, 40])
@pytest.mark.parametrize("K,N", [(1000, 136), (512, 64)])
def test_casts_and_moves_keep_the_bits(dev, M, K, N):
    torch.manual_seed(M)
    m = tbf16.convert(nn.Sequential(nn.Linear(K, N).to(BF).to(dev)), sdpa=False, int8=True)
    x = torch.randn(M, K).to(BF).to(dev)
    with torch.no_grad():
        y = m(x)
        for change in (lambda: m.to(BF), lambda: m.half(), lambda: m.cpu().to(dev), lambda: m.double().to("cpu", BF).to(dev)):
            change()
            m[0].bias.data = m[0].bias.data.to(BF)  # (bf16's values in every cast)
            assert torch.equal(m(x), y)
            assert int8._weight_rows(m[0].weight8, K)[0] is m[0].weight8  # read in place
