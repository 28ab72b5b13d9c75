"""The 8-bit linear in every form that the library chooses from (tests/_serving_shapes.py) against
64 bits."""
import pytest
import torch

import tbf16

from _serving_shapes import DECODE, TILES

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def codes(x):
    """tests/_serving64.py's codes64 for finite rows, on the device."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    return (127.0 * x / torch.where(top == 0, 1.0, top)).round(), top / 127.0


@pytest.mark.parametrize("M,K,N", DECODE + TILES)
def test_linear_forms(dev, M, K, N):
    g = torch.Generator(device=dev).manual_seed(M + 7 * K + 31 * N)
    x = (torch.randn(M, K, generator=g, device=dev) * torch.where(torch.rand(K, generator=g, device=dev) < 0.02, 10.0, 1.0)).to(BF)
    w = (torch.randn(N, K, generator=g, device=dev) * K ** -0.5).to(BF)
    b = torch.randn(N, generator=g, device=dev).to(BF)
    y = tbf16.int8_linear(x, *tbf16.prepare_weight_i8(w), b)
    assert y.shape == (M, N) and y.dtype == BF
    cx, sx = codes(x)
    for n in range(0, N, 8192):  # (the sums are whole numbers below 2^53: exact in any order)
        cw, sw = codes(w[n:n + 8192])
        p = torch.mm(cx, cw.t().contiguous()) * sx * sw.t()
        ref = p + b[n:n + 8192].double()
        # half a bf16 step, 2^-24 for each fp32 rounding of the product and for the bias's
        bound = 2.0 ** -8 * ref.abs() * (1 + 2.0 ** -10) + 6 * 2.0 ** -24 * p.abs()
        err = (y[:, n:n + 8192].double() - ref).abs()
        assert (err <= bound).all(), (err - bound).max()
