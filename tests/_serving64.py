"""64-bit results of the serving operators, and how far bf16 outputs may be off them."""
import torch

U24 = 2.0 ** -24  # half a step of fp32


def paged_sdpa64(q, k_cache, v_cache, table, lengths, scale=None):
    """(o, bound) on the CPU: o in 64 bits from the definition, and per element the largest
    error the operator's arithmetic allows:
      2^-8 |o|  the rounding to bf16 (half a step), on
      the error of o before it, at most e sum_j p_j |v_j| / sum_j p_j, where e sums
        2 (D + 4) 2^-23 max_j scale sum |q k_j|   a logit's products and their D sums and
                                                  factors, once in a weight and once in their sum
        2^-16                                     the weights as two bf16, exp2, the joins
        (n / 32 + 64) 2^-23                       n weighted values added 32 at a time
    """
    q, k_cache, v_cache, table = (t.cpu() for t in (q, k_cache, v_cache, table))
    B, H, D = q.shape
    pages, Hkv, page, _ = k_cache.shape
    G = H // Hkv
    sc = D ** -0.5 if scale is None else scale
    o, bound = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, D, dtype=torch.float64)
    for b, n in enumerate(lengths.tolist()):
        j = torch.arange(max(0, min(n, table.shape[1] * page)))
        at = table[b].long()[j // page] if len(j) else j
        ok = (at >= 0) & (at < pages)
        at, off = at[ok], (j % page)[ok]
        if len(at) == 0:
            continue
        for h in range(Hkv):
            k, v = k_cache[at, h, off].double(), v_cache[at, h, off].double()
            qg = q[b, h * G:(h + 1) * G].double()
            p = torch.softmax(qg @ k.t() * sc, -1)
            o[b, h * G:(h + 1) * G] = p @ v
            size = (qg.abs() @ k.abs().t() * abs(sc)).amax(-1, keepdim=True)
            e = 2 * (D + 4) * 2 * U24 * size + 2.0 ** -16 + (len(at) / 32 + 64) * 2 * U24
            bound[b, h * G:(h + 1) * G] = 2.0 ** -8 * o[b, h * G:(h + 1) * G].abs() + 1.01 * e * (p @ v.abs())
    return o, bound


def codes64(x):
    """(codes, scales) of bf16 rows in 64 bits: 127 x / max |x| has 15 by 8 bits, so its 53-bit
    quotient lies on the same side of every border as the exact one, and on the borders
    themselves it is exact."""
    x = x.cpu().double()
    top = x.abs().amax(-1, keepdim=True) if x.shape[-1] else torch.zeros(x.shape[0], 1, dtype=torch.float64)
    bad = ~torch.isfinite(top)
    code = torch.where(bad | (top == 0), 0.0, 127.0 * torch.where(bad, 0.0, x) / torch.where(top == 0, 1.0, top)).round()
    return code, torch.where(bad, torch.nan, top / 127.0)


def int8_linear64(x, w, bias=None):
    """(y, bound) on the CPU from bf16 x (M, K), w (N, K): both quantised as defined, summed in
    64 bits. bound: half a bf16 step of y, and 2^-24 for each of the product's fp32 roundings
    (two scales, the sum's conversion, two factors) and for the bias's."""
    (cx, sx), (cw, sw) = codes64(x), codes64(w)
    p = (cx @ cw.t()) * sx * sw.t()
    y = p if bias is None else p + bias.cpu().double()
    return y, 2.0 ** -8 * y.abs() * (1 + 2.0 ** -10) + 6 * U24 * p.abs()
