"""Plain forms, in 64 bits on the CPU, of pages in 8 bits and of attention for drafted trees, and pools to run them on."""

import math

import torch

import paged_reference as pr

LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
LEAST = 2.0 ** -100


def coded(x, form):
    """``(codes, scales)`` of rows ``x [.., dh]``: the codes nearest to ``x / scale`` in 64 bits, halves to the even one."""
    top = x.double().abs().amax(-1)
    scale = (top / LARGEST[form]).float().clamp(min=LEAST)
    scale[~torch.isfinite(top)] = math.nan
    t = torch.nan_to_num(x.double() / scale.double()[..., None], nan=0.0, posinf=0.0, neginf=0.0)
    t[torch.isnan(scale)] = 0.0
    if form is torch.int8:
        return t.round().to(torch.int8), scale
    step = 2.0 ** (torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3)
    return ((t / step).round() * step).float().to(form), scale


def meant(codes, scales):
    """What codes stand for, in 64 bits."""
    return codes.float().double() * scales.double()[..., None]


def pool8(lengths, page, kv_heads, dh, form, seed, spread=0.3):
    """``(k_pages, v_pages, table, scales)``; every slot that no token has holds a scale of NaN or infinity."""
    k, v, table = pr.pool(lengths, page, kv_heads, dh, torch.float32, seed, fill="wild")
    g = torch.Generator().manual_seed(seed + 17)
    pages, scales = [], []
    for t in (k, v):
        free = ~torch.isfinite(t).all(-1)
        codes, scale = coded(torch.where(free[..., None], torch.ones_like(t), t), form)
        scale = scale * torch.exp(spread * torch.randn(scale.shape, generator=g))
        scale[free] = torch.tensor([math.nan, math.inf])[torch.arange(int(free.sum())) % 2]
        pages.append(codes)
        scales.append(scale.contiguous())
    return pages[0], pages[1], table, tuple(scales)


def row(pages, scales, at, head, slot):
    """One key or value in 64 bits; ``scales`` None: of pages of the model's type."""
    x = pages[at, head, slot].float().double() if pages.dtype is not torch.float64 else pages[at, head, slot]
    return x if scales is None else x * scales[at, head, slot].double()


def sequence(pages, scales, table, b, first, last, head):
    page = pages.shape[2]
    rows = [row(pages, scales, int(table[b, t // page]), head, t % page) for t in range(first, last + 1)]
    return torch.stack(rows) if rows else torch.zeros(0, pages.shape[3], dtype=torch.float64)


def weighted(x, k, v, seen, scale):
    """``(output, bound)`` of one query ``x [dh]`` over the keys that it sees.  The bound is that of ``paged_reference.attention``
    with 12 more roundings to a score and to a weight: a key's scale into the score, queries as fp16 numbers times a power of two
    (2^-38 of the largest), a value's scale into the weight."""
    u = 2.0 ** -23
    k, v = k[seen], v[seen]
    n, dh = k.shape
    if n == 0:
        return torch.zeros(dh, dtype=torch.float64), 0.0
    s = k @ x * scale
    off = (dh + 16) * u * float((k.abs() @ x.abs()).max()) * scale + 2 * u * float(s.abs().max())
    off += dh * 2.0 ** -38 * float(x.abs().max()) * float(k.abs().max()) * scale
    return torch.softmax(s, 0) @ v, 2 * float(v.abs().max()) * (1.01 * off + (n + 20) * u)


def tree_attention(q, k_pages, v_pages, table, start, seen, counts=None, positions=None, window=None, k_pers=None, v_pers=None,
                   scale=0.0, scales=(None, None), pers_scales=(None, None), weight_off=0.0):
    """``(output [B, heads, nodes, dh], bound [B, heads, nodes, 1])`` in 64 bits, zero where nothing is written; ``weight_off``: by how
    much of itself a weight may be off besides."""
    B, heads, nodes, dh = q.shape
    kv_heads = k_pages.shape[1]
    group, scale = heads // kv_heads, scale or 1.0 / math.sqrt(dh)
    out, bound = torch.zeros(B, heads, nodes, dh, dtype=torch.float64), torch.zeros(B, heads, nodes, 1, dtype=torch.float64)
    for b in range(B):
        first, count = int(start[b]), nodes if counts is None else int(counts[b])
        if first < 0:
            continue
        for h in range(kv_heads):
            k = sequence(k_pages, scales[0], table, b, 0, first + count - 1, h)
            v = sequence(v_pages, scales[1], table, b, 0, first + count - 1, h)
            n_p = 0
            if k_pers is not None:
                n_p = k_pers.shape[1]
                kp, vp = (t[h].float().double() if s is None else meant(t[h], s[h]) for t, s in ((k_pers, pers_scales[0]), (v_pers, pers_scales[1])))
                k, v = torch.cat((kp, k)), torch.cat((vp, v))
            for i in range(count):
                visible = torch.ones(n_p + first + count, dtype=torch.bool)
                if window is not None:
                    visible[n_p: n_p + max(0, min(first, max(int(positions[b, i]), first) - window))] = False
                for j in range(count):
                    visible[n_p + first + j] = bool(int(seen[b, i]) >> j & 1)
                for g in range(group):
                    out[b, h * group + g, i], off = weighted(q[b, h * group + g, i].double(), k, v, visible, scale)
                    bound[b, h * group + g, i] = off + (2 * weight_off * float(v[visible].abs().max()) if visible.any() else 0.0)
    return out, bound


def one_token(q, k_pages, v_pages, table, pos, window=None, k_pers=None, v_pers=None, scale=0.0, scales=(None, None),
              pers_scales=(None, None)):
    """``paged_attention`` as the tree of one node that it is: ``(output [B, heads, dh], bound [B, heads, 1])``."""
    seen = torch.ones(len(pos), 1, dtype=torch.int64)
    none = (pos < 0)
    counts = (~none).long()
    out, bound = tree_attention(q[:, :, None], k_pages, v_pages, table, pos.clamp(min=0), seen, counts, pos.clamp(min=0)[:, None], window,
                                k_pers, v_pers, scale, scales, pers_scales)
    for b in none.nonzero()[:, 0].tolist():  # the persistent keys alone
        if k_pers is not None:
            o, off = _persistent(q[b], k_pers, v_pers, scale, pers_scales)
            out[b, :, 0], bound[b, :, 0] = o, off
    return out[:, :, 0], bound[:, :, 0]


def _persistent(q, k_pers, v_pers, scale, pers_scales):
    heads, dh = q.shape
    group, scale = heads // k_pers.shape[0], scale or 1.0 / math.sqrt(dh)
    out, bound = torch.zeros(heads, dh, dtype=torch.float64), torch.zeros(heads, 1, dtype=torch.float64)
    for h in range(heads):
        k, v = (t[h // group].float().double() if s is None else meant(t[h // group], s[h // group])
                for t, s in ((k_pers, pers_scales[0]), (v_pers, pers_scales[1])))
        out[h], bound[h] = weighted(q[h].double(), k, v, torch.ones(k.shape[0], dtype=torch.bool), scale)
    return out, bound


def ancestors(parents):
    """``(seen, depth)`` of one tree, by walking up from every node."""
    seen, depth = [], []
    for i in range(len(parents)):
        bits, n, j = 0, 0, i
        while j >= 0:
            bits |= 1 << j
            j = parents[j]
            n += 1
        seen.append(bits - (1 << 64) if bits >> 63 else bits)
        depth.append(n - 1)
    return torch.tensor(seen, dtype=torch.int64), torch.tensor(depth)
