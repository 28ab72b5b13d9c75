"""paged_advance while another stream writes its lengths, counts and stack: it stays within its arrays, and the calls
after it are right."""
import random

import pytest
import torch

import tbf16

from test_gpu_advance import check, state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,n,page,pages,tokens", [(20, 8, 16, 300, 300), (20, 8, 16, 300, 5000), (2100, 8, 16, 9000, 600), (2100, 4, 3, 500, 5000),
                                                   (4, 1 << 19, 4096, 1000, 5000), (4, 1 << 19, 4096, 1000, 900)])
def test_state_written_meanwhile(dev, B, n, page, pages, tokens):
    """The last two have tables whose positions count up to 2^31 - 1."""
    g = torch.Generator().manual_seed(n + tokens)
    i32 = lambda *s, v=0: torch.full(s, v, dtype=torch.int32, device=dev)  # noqa: E731
    top = min(n * page, 2 ** 31 - 1)
    table, lengths, counts, free, n_free = i32(B, n, v=-1), i32(B), i32(B), torch.arange(pages, dtype=torch.int32, device=dev), i32(1, v=pages)
    some = lambda lo, hi, s: torch.randint(lo, hi, s, generator=g).int().to(dev)  # noqa: E731
    many = [(some(0, top, (B,)) if i % 2 else top - 1 - some(0, 9, (B,)), some(-5, 7, (B,)) if i % 3 else some(0, tokens, (B,)), some(0, pages, (1,)))
            for i in range(12)]
    calls, writes = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(writes):
            for a, b, c in many:
                lengths.copy_(a)
                counts.copy_(b)
                n_free.copy_(c)
        with torch.cuda.stream(calls):
            for _ in range(6):
                slots, positions, starts = tbf16.paged_advance(table, lengths, counts, free, n_free, page, tokens)
    torch.cuda.synchronize()
    assert int(slots.min()) >= -1 and int(slots.max()) < pages * page and int(positions.min()) >= -1
    assert int(starts[0]) == 0 and int(starts.max()) <= tokens
    r = random.Random(5)
    small = state(r, 30, 6, 16, 40)
    check(dev, *small[:2], [r.choice((0, 1, 9, -4)) for _ in range(30)], *small[2:], 16, 200)
