"""Plain forms, in 64 bits on the CPU, of the operators over paged keys and values, and pools to run them on."""

import math

import torch


def pool(lengths, page, kv_heads, dh, dtype, seed, spare=2, fill="normal"):
    """``(k_pages, v_pages, page_table)`` on the CPU for sequences of ``lengths`` tokens; table entries behind a sequence's pages
    name no page, and with ``fill="wild"`` every slot that no token has holds infinities and NaN."""
    g = torch.Generator().manual_seed(seed)
    needed = [-(-n // page) for n in lengths]
    pages = sum(needed) + spare
    k = torch.randn(pages, kv_heads, page, dh, generator=g).to(dtype)
    v = torch.randn(pages, kv_heads, page, dh, generator=g).to(dtype)
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lengths), max(needed + [1])), -7, dtype=torch.int32)
    held = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(needed):
        for c in range(n):
            table[b, c] = at = order.pop()
            held[at, : min(page, lengths[b] - c * page)] = True
    if fill == "wild":
        wild = torch.tensor([float("nan"), float("inf"), -float("inf")], dtype=dtype)
        for t in (k, v):
            t[(~held)[:, None, :].expand(-1, kv_heads, -1)] = wild[torch.arange(dh) % 3]
    return k, v, table


def sequence(pages, table, b, first, last, head):
    """Rows ``first .. last`` of a sequence under one head, in 64 bits."""
    page = pages.shape[2]
    return torch.stack([pages[table[b, t // page], head, t % page] for t in range(first, last + 1)]).double() \
        if last >= first else torch.zeros(0, pages.shape[3], dtype=torch.float64)


def attention(q, k_pages, v_pages, table, pos, window=None, k_pers=None, v_pers=None, scale=0.0):
    """``(output, bound on an fp32 evaluation's error)``, both ``[B, heads, dh]`` in 64 bits.

    The bound: with u = 2^-23 (tensor cores cut sums off instead of rounding them) a score of dh products is off by at most
    (dh + 4) u sum |q k| scale and its multiplication into a power of two by 2 u |s|; e^d - 1 is below 1.01 d for d < 0.02; a weight
    has 4 u of the exponential and of its two halves in 16 bits; n weights and products are summed with n u.  Numerator and
    denominator both carry that, so an output is off by at most twice it times the largest |v|."""
    B, heads, dh = q.shape
    kv_heads = k_pages.shape[1]
    group, scale = heads // kv_heads, scale or 1.0 / math.sqrt(dh)
    out, bound = torch.zeros(B, heads, dh, dtype=torch.float64), torch.zeros(B, heads, 1, dtype=torch.float64)
    u = 2.0 ** -23
    for b in range(B):
        p = int(pos[b])
        first = 0 if window is None else max(0, p - window)
        for h in range(kv_heads):
            k, v = sequence(k_pages, table, b, first, p, h), sequence(v_pages, table, b, first, p, h)
            if k_pers is not None:
                k, v = torch.cat((k_pers[h].double(), k)), torch.cat((v_pers[h].double(), v))
            n = k.shape[0]
            if n == 0:
                continue
            rows = slice(h * group, (h + 1) * group)
            x = q[b, rows].double()
            s = x @ k.T * scale
            out[b, rows] = torch.softmax(s, -1) @ v
            off = (dh + 4) * u * (x.abs() @ k.abs().T * scale).amax(-1) + 2 * u * s.abs().amax(-1)
            bound[b, rows, 0] = 2 * v.abs().amax() * (1.01 * off + (n + 8) * u)
    return out, bound


def rotated(x, positions, inv_freq, interleaved):
    """``x [heads, rows, dh]`` turned by ``positions [rows]``, in 64 bits."""
    y = x.double().clone()
    half = inv_freq.shape[0]
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    angle = positions.double()[:, None] * inv_freq.double()
    c, s = torch.cos(angle), torch.sin(angle)
    y[..., a], y[..., b] = x[..., a].double() * c - x[..., b].double() * s, x[..., b].double() * c + x[..., a].double() * s
    return y
