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


def rotate64(z, cos, sin, near, back=False):
    """The first 2 * cos.shape[-1] elements of z in pairs turned by the angles (or back)."""
    R = 2 * cos.shape[-1]
    a, b = (z[..., 0:R:2], z[..., 1:R:2]) if near else (z[..., :R // 2], z[..., R // 2:R])
    s = -sin if back else sin
    y = z.clone()
    ya, yb = a * cos - b * s, b * cos + a * s
    if near:
        y[..., 0:R:2], y[..., 1:R:2] = ya, yb
    else:
        y[..., :R // 2], y[..., R // 2:R] = ya, yb
    return y


def norm_rope64(x, w, cos, sin, pos, eps=1e-6, near=False, dy=None):
    """On the CPU in 64 bits, x (..., H, D), pos of its leading dimensions: (y, bound), and with dy
    (y, bound, dx, bound, dw, bound before the rounding of dw). u = half a step of fp32 for each rounding:
      r            the squares' sum (16 in turn, 4 steps across lanes, a product each) half of it, the mean, eps,
                   the root: under 16 u of r
      y            r, x r, w, and the rotation's two products and sum: 24 u of |z_i c| + |z_j s|
      dx           dy turned back (3 u of A = |dy_i c| + |dy_j s|), w, x r (18 u), the mean of D products (20 sums), their
                   difference, r, scale: under 80 u of r (A |w| + |x r| mean(A |w x r|))
      dw           products (22 u) and as many sums as a lane makes and the blocks' shares pass through
    and half a step of bf16 of what comes out as such."""
    D = x.shape[-1]
    x, w, pos = x.detach().cpu().double(), w.detach().cpu().double(), pos.cpu().long()
    at = pos.clamp(0, cos.shape[0] - 1)
    c, s = (t.cpu().double()[at].unsqueeze(-2) for t in (cos, sin))
    real = (pos >= 0)[..., None, None]
    r = 1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    u = x * r
    z = u * w
    y = torch.where(real, rotate64(z, c, s, near), 0.0)
    size = rotate64(z.abs(), c.abs(), -s.abs(), near)  # |z_i c| + |z_j s| in the first of a pair
    size = torch.maximum(size, rotate64(z.abs(), c.abs(), s.abs(), near))
    out = [y, torch.where(real, 2.0 ** -8 * y.abs() + 24 * U24 * size, 0.0)]
    if dy is None:
        return tuple(out)
    g = dy.detach().cpu().double()
    A = torch.maximum(rotate64(g.abs(), c.abs(), -s.abs(), near), rotate64(g.abs(), c.abs(), s.abs(), near))
    dz = torch.where(real, rotate64(g, c, s, near, back=True), 0.0)
    A = torch.where(real, A, 0.0)
    du = dz * w
    dx = r * (du - u * (du * u).mean(-1, keepdim=True))
    spread = r * (A * w.abs() + u.abs() * (A * (w * u).abs()).mean(-1, keepdim=True))
    tokens, H = pos.numel(), x.shape[-2]
    # (up to 8 times as many heads of the other kind: 256 waves at least take these, or one a token)
    sums = -(-H // (64 // (4 if D <= 64 else 8 if D <= 128 else 16))) * -(-tokens // 256) + 90
    flat = lambda t: t.flatten(0, -2)  # noqa: E731
    dw, dw_bound = flat(dz * u).sum(0), (22 + sums) * U24 * flat(A * u.abs()).sum(0)
    return (*out, dx, 2.0 ** -8 * dx.abs() + 80 * U24 * spread, dw, dw_bound)


def prefix_sdpa64(q, k_cache, v_cache, prefix_table, prefix_length, table, lengths, scale=None):
    """(o, bound) on the CPU: attention of each sequence over the prefix's positions and its own, from the
    definition in 64 bits. bound: half a bf16 step of o, and of the error before it at most e sum_j p_j
    |v_j| / sum_j p_j, where e sums
      2 (D + 4) 2^-23 max_j scale sum |q k_j|   a logit's products, D sums and factors, in a weight and in their sum
      2^-16 + 2^-17                             a weight as two bf16 (8 bits cut off, the rest, below 2^-7 of it, to 8
                                                bits: half of 2^-15); exp2 and the joins' factors
      (n / 32 + 64) 2^-23                       n weighted values added 32 at a time, the parts of the joins"""
    q, k_cache, v_cache, prefix_table, table = (t.cpu() for t in (q, k_cache, v_cache, prefix_table, table))
    B, H, D = q.shape
    pages, Hkv, page, _ = k_cache.shape
    G = H // Hkv
    sc = D ** -0.5 if scale is None else scale

    def places(ids, n):
        j = torch.arange(max(0, min(int(n), ids.shape[0] * page)))
        at = ids.long()[j // page] if len(j) else j
        ok = (at >= 0) & (at < pages)
        return at[ok], (j % page)[ok]
    far = places(prefix_table, prefix_length)
    shared = [(k_cache[far[0], h, far[1]].double(), v_cache[far[0], h, far[1]].double()) for h in range(Hkv)]
    o, bound = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, D, dtype=torch.float64)
    for b, n in enumerate(lengths.tolist()):
        at, off = places(table[b], n)
        if len(at) + len(far[0]) == 0:
            continue
        for h in range(Hkv):
            k = torch.cat((shared[h][0], k_cache[at, h, off].double()))
            v = torch.cat((shared[h][1], v_cache[at, h, off].double()))
            qg = q[b, h * G:(h + 1) * G].double()
            p = torch.softmax(qg @ k.t() * sc, -1)
            o[b, h * G:(h + 1) * G] = p @ v
            size = (qg.abs() @ k.abs().t() * abs(sc)).amax(-1, keepdim=True)
            e = 2 * (D + 4) * 2 * U24 * size + 1.5 * 2.0 ** -16 + (len(k) / 32 + 64) * 2 * U24
            bound[b, h * G:(h + 1) * G] = 2.0 ** -8 * o[b, h * G:(h + 1) * G].abs() + 1.01 * e * (p @ v.abs())
    return o, bound
