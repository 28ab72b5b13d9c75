"""paged_advance: tokens granted and taken back, where the state was as it should be and where it was not."""
import pytest
import torch

import tbf16

pytestmark = pytest.mark.gpu


def there_and_back(dev, table, lengths, counts, stack, n_free, page, tokens):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    t, ln, fr, nf, c = i32(table), i32(lengths), i32(stack), i32([n_free]), i32(counts)
    before = ln.clone()
    tbf16.paged_advance(t, ln, c, fr, nf, page, tokens)
    tbf16.paged_advance(t, ln, before - ln, fr, nf, page, 0)
    n = nf.item()
    return t.tolist(), ln.tolist(), fr.tolist()[:n]


def test_as_it_was(dev):
    """The second does not fit its row, the third's page is not there: neither has anything to take back."""
    state = [[0, -1, -1], [1, 2, 3], [4, -1, -1]], [3, 11, 4], [9, 8, 5] + [0] * 7
    assert there_and_back(dev, state[0], state[1], [8, 2, 5], state[2], 3, 4, 20) == (state[0], state[1], [9, 8, 5])


def test_entries_past_the_pages_become_none(dev):
    assert there_and_back(dev, [[0, 7]], [4], [1], [9, 8, 5] + [0] * 7, 3, 4, 5) == ([[0, -1]], [4], [9, 8, 5])


def test_ids_that_are_no_page_do_not_go_back(dev):
    """The stack has three entries, so the cache has three pages: 9 and 8 are none of them."""
    assert there_and_back(dev, [[0, -1]], [4], [1], [1, 2, 8], 3, 4, 5) == ([[0, -1]], [4], [1, 2])


def test_a_length_past_the_row_becomes_the_row(dev):
    assert there_and_back(dev, [[0, 1]], [100], [0], [2, 0, 0], 1, 4, 5)[0] == [[0, 1]]
