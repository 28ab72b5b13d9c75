"""Plain results of the operators around the paged cache: page tables kept by hand, norms and
rotations and attention in 64 bits, and how far the operators may be off them."""
import torch

U24 = 2.0 ** -24  # half a step of fp32


def advance_by_hand(table, lengths, counts, stack, n_free, page, tokens, prefix=0):
    """One sequence and one page after the other, on lists that are changed in place; returns
    (n_free, slots, positions, starts)."""
    pages, n = len(stack), len(table[0]) if table else 0
    n_free = min(max(n_free, 0), pages)
    up = lambda v: -(-v // page)  # noqa: E731
    cap = min(n * page, 2 ** 31 - 1)
    lengths[:] = [min(max(v, 0), cap) for v in lengths]
    for b in reversed(range(len(table))):
        if counts[b] < 0:
            less = max(0, lengths[b] + counts[b])
            for i in reversed(range(up(less), up(lengths[b]))):
                if 0 <= table[b][i] < pages and n_free < pages:
                    stack[n_free] = table[b][i]
                    n_free += 1
                table[b][i] = -1
            lengths[b] = less
    slots, positions, starts, asked, free = [], [], [0], 0, n_free
    for b, c in enumerate(counts):
        if c > 0:
            new, fits = lengths[b] + c, lengths[b] + c <= cap
            need = up(new) - up(lengths[b]) if fits else 0
            asked += need
            room = starts[-1] + c <= tokens
            starts.append(min(starts[-1] + c, tokens) if room else tokens)
            if fits and room and (need == 0 or asked <= free):
                for j in range(lengths[b], new):
                    if j % page == 0:
                        n_free -= 1
                        table[b][j // page] = stack[n_free]
                    at = table[b][j // page]
                    slots.append(at * page + j % page if 0 <= at < pages else -1)
                    positions.append(j + prefix)
                lengths[b] = new
            else:
                slots += [-1] * (starts[-1] - starts[-2])
                positions += [-1] * (starts[-1] - starts[-2])
        else:
            starts.append(starts[-1])
    pad = [-1] * (tokens - len(slots))
    return n_free, slots + pad, positions + pad, starts
