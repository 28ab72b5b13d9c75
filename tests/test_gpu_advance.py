"""paged_advance on the GPU against tables kept by hand: whole numbers, equal."""
import random

import pytest
import torch

import tbf16

from _operators64 import advance_by_hand

pytestmark = pytest.mark.gpu


def state(r, B, n, page, spare, longest=None):
    """Consistent tables: (table, lengths, stack, n_free) as lists."""
    lengths = [r.randint(0, min(n * page, n * page if longest is None else longest)) for _ in range(B)]
    need = [-(-v // page) for v in lengths]
    pages = sum(need) + spare
    order = list(range(pages))
    r.shuffle(order)
    table, at = [], 0
    for k in need:
        table.append(order[at:at + k] + [r.choice((-1, 0, pages, 2 ** 30)) for _ in range(n - k)])
        at += k
    return table, lengths, order[at:] + [0] * at, pages - at


def put(dev, table, lengths, stack, n_free, n):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    return i32(table).reshape(len(table), n), i32(lengths), i32(stack), i32([n_free])


def check(dev, table, lengths, counts, stack, n_free, page, tokens, prefix=None, n=None, wide=0):
    """One call on the device and by hand; both states go on from it."""
    n = len(table[0]) if n is None else n
    t, ln, fr, nf = put(dev, table, lengths, stack, n_free, n)
    if wide:
        t = torch.cat((t, torch.full((len(table), wide), 77, dtype=torch.int32, device=dev)), 1)
    c = torch.tensor(counts, dtype=torch.int32, device=dev)
    p = None if prefix is None else torch.tensor([prefix], dtype=torch.int32, device=dev)
    slots, positions, starts = tbf16.paged_advance(t[:, :n] if wide else t, ln, c, fr, nf, page, tokens, p)
    for x, shape in ((slots, tokens), (positions, tokens), (starts, len(table) + 1)):
        assert x.dtype == torch.int32 and x.shape == (shape,) and x.is_contiguous()
    n_free, *want = advance_by_hand(table, lengths, counts, stack, n_free, page, tokens, max(prefix or 0, 0))
    assert nf.tolist() == [n_free] and ln.tolist() == lengths and fr.tolist() == stack
    assert t[:, :n].tolist() == table and (not wide or bool((t[:, n:] == 77).all()))
    assert [slots.tolist(), positions.tolist(), starts.tolist()] == want
    return n_free


@pytest.mark.parametrize("B,n,page,tokens", [(1, 1, 1, 3), (1, 5, 16, 40), (5, 4, 3, 30), (64, 10, 16, 70), (70, 3, 1, 100),
                                             (1030, 4, 16, 2500), (2048, 3, 48, 6000), (2049, 3, 48, 4096), (3000, 2, 16, 5000),
                                             (33, 300, 16, 9000), (2500, 2, 16, 1500)])
@pytest.mark.parametrize("spare", [0, 7, 10 ** 4])
def test_steps(dev, B, n, page, tokens, spare):
    """Several steps of mixed counts: growth, shrinking, ends, idle ones; too few pages and rows."""
    r = random.Random(B * 31 + spare)
    table, lengths, stack, n_free = state(r, B, n, page, spare)
    top = max(2, 2 * tokens // B)
    for step in range(4):
        counts = [r.choice((0, 1, 1, r.randint(0, top), -r.randint(0, top), -10 ** 9 if r.random() < 0.2 else 1)) for _ in range(B)]
        n_free = check(dev, table, lengths, counts, stack, n_free, page, tokens, step * 100 if step else None, n, wide=step % 2 * 3)


@pytest.mark.parametrize("B,most,tokens", [(1, 3000, 3000), (1, 2000, 2000), (1, 70000, 70000), (40, 200, 9000), (1500, 9, 9000), (2500, 3, 9000), (300, 13, 4096)])
def test_back_again(dev, B, most, tokens):
    r = random.Random(B)
    table, lengths, stack, n_free = state(r, B, -(-(2000 + most) // 16), 16, B * (most // 16 + 2), longest=2000)
    counts = [r.randint(0, most) for _ in range(B)]
    counts = [c if sum(counts[:b + 1]) <= tokens else 0 for b, c in enumerate(counts)]
    for row, v in zip(table, lengths):
        row[-(-v // 16):] = [-1] * (len(row) + (-v // 16))
    t, ln, fr, nf = put(dev, table, lengths, stack, n_free, len(table[0]))
    c = torch.tensor(counts, dtype=torch.int32, device=dev)
    slots, _, starts = tbf16.paged_advance(t, ln, c, fr, nf, 16, tokens)
    assert ln.tolist() == [v + c for v, c in zip(lengths, counts)] and starts[-1].item() == sum(counts)
    used = slots[slots >= 0].tolist()
    assert len(used) == len(set(used)) == sum(counts)
    tbf16.paged_advance(t, ln, -c, fr, nf, 16, 0)
    assert t.tolist() == table and ln.tolist() == lengths and nf.tolist() == [n_free]
    assert fr.tolist()[:n_free] == stack[:n_free]


def test_no_pages_left(dev):
    """The first that lacks pages, and who comes after it: only sequences that need none."""
    table, lengths = [[0, -1], [1, -1], [2, -1], [3, -1]], [2, 4, 4, 1]
    assert check(dev, table, lengths, [1, 4, 4, 2], [9, 5] + [0] * 8, 1, 4, 20) == 0
    assert lengths == [3, 8, 4, 3] and table[1] == [1, 9]
    # more pages asked for by those before: nobody behind gets the one that is left
    table, lengths = [[0, -1, -1], [1, -1, -1]], [4, 4]
    assert check(dev, table, lengths, [8, 1], [9] * 10, 1, 4, 20) == 1 and lengths == [4, 4]
    # who cannot fit its row asks for none
    table, lengths = [[0, -1], [1, -1]], [4, 4]
    assert check(dev, table, lengths, [5, 1], [9] * 10, 1, 4, 20) == 0 and lengths == [4, 5]


def test_odd_state(dev):
    """Lengths and counts out of range, entries that name no page, a stack that is full."""
    check(dev, [[0, 1], [2, 3]], [100, -5], [-1, 3], [4, 0, 0, 0, 0], 99, 4, 5)
    check(dev, [[7, -1], [2, 50]], [8, 8], [-8, -8], [4, 0, 0, 0, 0], -3, 4, 5)
    check(dev, [[0, 1], [2, 3]], [8, 8], [-8, -8], [0, 1, 2, 3, 4], 3, 4, 5)
    check(dev, [[99], [1]], [1, 1], [1, 2], [0, 1], 0, 4, 9, -7)  # tokens in a page that is none
    check(dev, [[0, 1], [2, 3]], [1, 2], [2 ** 31 - 1, 2 ** 31 - 1], [0, 1, 2, 3, 4], 5, 4, 9)
    check(dev, [[0, 1], [2, 3]], [5, 2], [-2 ** 31, -2 ** 31], [0, 1, 2, 3, 4], 0, 4, 9)
    check(dev, [[0, 1], [2, 3], [0, 0]], [1, 2, 1], [2 ** 31 - 1, 1, 2 ** 31 - 1], [0, 1, 2, 3, 4], 5, 4, 9, 2 ** 31 - 1)


def test_nothing(dev):
    check(dev, [], [], [], [0, 1], 2, 4, 3, n=2)
    check(dev, [], [], [], [0, 1], 2, 4, 5000, n=2)
    check(dev, [[], []], [0, 0], [1, 0], [0, 1], 2, 4, 3, n=0)
    check(dev, [[0]], [1], [1], [], 0, 4, 3)
    check(dev, [[0]], [1], [1], [0, 1], 2, 4, 0)
    check(dev, [[0]], [1], [-1], [0, 1], 0, 4, 0)


def test_large_batch(dev):
    B = 50000
    r = random.Random(1)
    table, lengths, stack, n_free = state(r, B, 2, 4, B)
    check(dev, table, lengths, [r.choice((-3, 0, 1, 2)) for _ in range(B)], stack, n_free, 4, B)


def test_graph_of_steps(dev):
    """Captured once, replayed with other counts; both forms (in one launch, in two)."""
    for B, tokens in ((20, 300), (20, 5000), (2100, 600)):
        r = random.Random(3)
        table, lengths, stack, n_free = state(r, B, 8, 16, 60 * B)
        t, ln, fr, nf = put(dev, table, lengths, stack, n_free, 8)
        c = torch.zeros(B, dtype=torch.int32, device=dev)
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            tbf16.paged_advance(t, ln, c, fr, nf, 16, tokens)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = tbf16.paged_advance(t, ln, c, fr, nf, 16, tokens)
        for _ in range(4):
            counts = [r.choice((0, 1, 13, -4, -200)) for _ in range(B)]
            c.copy_(torch.tensor(counts, dtype=torch.int32))
            g.replay()
            n_free, *want = advance_by_hand(table, lengths, counts, stack, n_free, 16, tokens)
            assert [x.tolist() for x in out] == want and nf.item() == n_free
            assert t.tolist() == table and ln.tolist() == lengths and fr.tolist() == stack


def test_page_named_twice(dev):
    """Two entries of one page, a page that is on the stack already: in bounds, each given back as it stands."""
    check(dev, [[3, 3], [3, -1]], [8, 4], [-8, -4], [4, 0, 0, 0, 0], 1, 4, 5)
    check(dev, [[1, 1, 1], [1, 1, 1]], [12, 12], [-12, -5], [0, 1, 2, 3], 2, 4, 5)
    check(dev, [[1, 1, 1], [1, 1, 1], [2, -1, -1]], [12, 12, 1], [-12, -5, 11], [0, 0, 0, 0, 0], 1, 4, 12)


def test_two_at_once(dev):
    """Batches of their own on two streams, with and without a workspace."""
    r = random.Random(8)
    runs = []
    for B, tokens in ((700, 1500), (2300, 9000)):
        table, lengths, stack, n_free = state(r, B, 6, 16, 3 * B)
        runs.append([put(dev, table, lengths, stack, n_free, 6), (table, lengths, stack), n_free, tokens, torch.cuda.Stream()])
    for _ in range(6):
        calls = []
        for t, (table, lengths, stack), n_free, tokens, s in runs:
            counts = [r.choice((0, 1, 5, -3, -200)) for _ in table]
            calls.append((counts, torch.tensor(counts, dtype=torch.int32, device=dev)))
        torch.cuda.synchronize()
        outs = []
        for (t, _, _, tokens, s), (_, c) in zip(runs, calls):
            with torch.cuda.stream(s):
                outs.append(tbf16.paged_advance(t[0], t[1], c, t[2], t[3], 16, tokens))
        torch.cuda.synchronize()
        for run, (counts, _), out in zip(runs, calls, outs):
            t, by_hand, n_free, tokens, _ = run
            run[2], *want = advance_by_hand(*by_hand[:2], counts, by_hand[2], n_free, 16, tokens)
            assert [x.tolist() for x in out] == want and t[3].item() == run[2]
            assert [x.tolist() for x in t[:3]] == list(by_hand)
