"""paged_sdpa_prefix while another stream writes the prefix's length: a call takes one length or another for each of
its blocks, stays within its tables, and the calls after it are right."""
import pytest
import torch

import tbf16

from test_gpu_prefix import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,H,Hkv,D,page", [(4, 16, 16, 128, 16), (40, 8, 2, 64, 3), (9, 8, 2, 256, 16), (64, 32, 8, 128, 1)])
def test_length_written_meanwhile(dev, B, H, Hkv, D, page):
    top = 3000
    a = make(dev, top, [b % 50 for b in range(B)], H, Hkv, D, page, seed=B)
    a[3] = a[3][:-(-top // page)].contiguous()  # every entry names a page
    a[1].nan_to_num_(0.5)
    a[2].nan_to_num_(0.5)
    lengths = [torch.tensor([n], dtype=torch.int32, device=dev) for n in (top, 0, 1, 64, 65, 700, 2047, -1, 2 ** 31 - 1)]
    calls, writes = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(30):
        with torch.cuda.stream(writes):
            for n in lengths * 3:
                a[4].copy_(n)
        with torch.cuda.stream(calls):
            for _ in range(6):
                tbf16.paged_sdpa_prefix(*a)
    torch.cuda.synchronize()
    for n in (top, 700, 0):
        a[4].fill_(n)
        check(a)
