"""A paged key-value cache in 8 bits, and drafted tokens over a paged cache, as cases that can be timed and compared.

``listed()`` holds the cases, ``draw(rng)`` gives more of the same ranges.  A case is a dict of plain values; its ``kind`` says
which operator it is:

    store      keys and values of new tokens into 8-bit pages, a scale for each token and head, keys and queries rotated by their
               positions on the way; what the pages then stand for is read back
    attend     attention of one new token per sequence over 8-bit pages (window, persistent keys, shared heads)
    tree       attention of the drafted tokens of a tree, each over the cached tokens, its ancestors and itself, over pages of
               the model's type or of 8 bits
    keep       the accepted path of a tree: its keys and values moved together in their pages

With ``own`` false ``run`` computes them from elementary operations in fp32; with ``own`` true it makes the package's calls.
"""

import math
import os
import sys

import torch

sys.path.insert(1, os.path.join(os.getcwd(), "titanmac-standalone_b200"))

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_EIGHTS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_LARGEST = {"int8": 127.0, "e4m3": 448.0}
_LEAST_SCALE = 2.0 ** -100
_MOST_BYTES = 5.5e8  # of keys and values that a drawn case reads
_MOST_PRODUCTS = 1e10  # of a drawn tree's queries and keys, number by number


def _store(dtype, pages, batch, rows, heads, kv_heads, head_dim, page, rotated, interleaved=False, first=0):
    """``rows`` new tokens for the longest sequence, fewer for the others; they start somewhere in ``0 .. first``."""
    return dict(kind="store", dtype=dtype, pages=pages, batch=batch, rows=rows, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                page=page, rotated=rotated, interleaved=interleaved, first=first)


def _attend(dtype, pages, batch, tokens, heads, kv_heads, head_dim, page, window=-1, persistent=0, skew=1.0):
    """The longest sequence has ``tokens`` keys, the others a share of that (``skew``: how fast it falls)."""
    return dict(kind="attend", dtype=dtype, pages=pages, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, page=page, window=window, persistent=persistent, skew=skew)


def _tree(dtype, pages, batch, tokens, nodes, branch, heads, kv_heads, head_dim, page, window=-1, persistent=0, skew=1.0):
    """Up to ``nodes`` drafted tokens behind up to ``tokens`` cached ones; node ``i`` is a child of node ``(i - 1) // branch``.
    ``pages``: "" for pages of the model's type."""
    return dict(kind="tree", dtype=dtype, pages=pages, batch=batch, tokens=tokens, nodes=nodes, branch=branch, heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, page=page, window=window, persistent=persistent, skew=skew)


def _keep(dtype, pages, batch, nodes, kept, kv_heads, head_dim, page, first=0):
    """Up to ``kept`` of ``nodes`` drafted tokens stay; the drafts start somewhere in ``0 .. first``."""
    return dict(kind="keep", dtype=dtype, pages=pages, batch=batch, nodes=nodes, kept=kept, kv_heads=kv_heads, head_dim=head_dim,
                page=page, first=first)


def listed():
    return [
        # a serving step of many sequences: one token each, heads that share keys
        dict(_store("bf16", "int8", 64, 1, 32, 8, 128, 16, 128, first=1000), name="store_step"),
        # prompts of several lengths go into the cache at once: the layer width of the long-context configuration
        dict(_store("bf16", "e4m3", 8, 4096, 16, 16, 128, 64, 128), name="store_prompts"),
        # a chunk of a prompt behind an earlier one, part of the head rotated in pairs of neighbours, pages of no power of two
        dict(_store("fp16", "int8", 3, 731, 10, 5, 64, 24, 32, interleaved=True, first=20000), name="store_chunk_odd"),
        # serving the default model: its window and persistent rows for 256 sequences
        dict(_attend("bf16", "int8", 256, 2048, 10, 10, 64, 64, window=512, persistent=16, skew=0.25), name="attend_window_batch"),
        # a mixed batch, a few long conversations among many short ones, heads that share keys, pages of no power of two
        dict(_attend("fp16", "e4m3", 48, 16384, 32, 8, 128, 24, skew=4.0), name="attend_ragged_grouped"),
        # long documents
        dict(_attend("bf16", "int8", 12, 65536, 32, 4, 128, 128, skew=0.5), name="attend_long"),
        # one answer being written, a few tokens drafted ahead: the default geometry
        dict(_tree("bf16", "", 1, 700, 8, 2, 10, 10, 64, 64, window=512, persistent=16), name="tree_one_sequence"),
        # the default model's window and persistent rows for many sequences
        dict(_tree("bf16", "", 64, 2048, 16, 3, 10, 10, 64, 64, window=512, persistent=16, skew=0.25), name="tree_window_batch"),
        # conversations of several lengths, an odd number of drafts, heads that share keys
        dict(_tree("fp16", "", 16, 16384, 33, 4, 32, 8, 128, 32), name="tree_ragged_grouped"),
        # long documents in 8 bits
        dict(_tree("bf16", "int8", 6, 65536, 12, 2, 32, 4, 128, 128, skew=0.5), name="tree_long_8bit"),
        # what follows a verified tree: 256 sequences of the default geometry
        dict(_keep("bf16", "", 256, 32, 6, 10, 64, 64, first=100), name="keep_batch"),
        # the same in 8 bits, pages of no power of two
        dict(_keep("bf16", "e4m3", 24, 61, 9, 8, 128, 17, first=500), name="keep_odd_8bit"),
    ]


def _log(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(("store", "attend", "attend", "tree", "tree", "keep"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    eight = rng.choice(("int8", "e4m3"))
    kv_heads = rng.choice((1, 2, 4, 5, 8, 10, 16))
    heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 7, 8))
    head_dim = rng.choice((64, 64, 128, 128, 32, 96, 256))
    page = rng.choice((16, 32, 64, 128, _log(rng, 1, 200)))
    size = _DTYPES[dtype].itemsize
    if kind == "store":
        row = (heads + 2 * kv_heads) * head_dim
        rows = _log(rng, 1, 4096)
        batch = _log(rng, 1, max(1, min(256, int(1e8 / (rows * row)))))
        # (in fp32 what is read back differs by a whole step where a rotation's last bit decides a rounding)
        rotated = 0 if dtype == "fp32" else rng.choice((0, head_dim // 2, head_dim))
        most = int(5e8 / (batch * kv_heads * head_dim * 2))  # earlier keys and values stand in the pages too
        return _store(dtype, eight, batch, rows, heads, kv_heads, head_dim, page, rotated, rng.random() < 0.4,
                      rng.choice((0, 0, _log(rng, 1, max(1, min(20000, most))))))
    if kind == "keep":
        nodes = _log(rng, 2, 64)
        return _keep(dtype, rng.choice(("", eight)), _log(rng, 1, 256), nodes, rng.randint(1, max(1, nodes // 2)), kv_heads, head_dim, page,
                     rng.choice((0, _log(rng, 1, 200))))
    if kind == "attend":
        tokens = _log(rng, 1, 65536)
        batch = _log(rng, 1, max(1, min(256, int(_MOST_BYTES / (tokens * kv_heads * head_dim * 2)))))
        window = rng.choice((-1, -1, _log(rng, 1, 4096)))
        return _attend(dtype, eight, batch, tokens, heads, kv_heads, head_dim, page, window, rng.choice((0, 0, 3, 16)),
                       rng.choice((0.25, 1.0, 4.0)))
    pages = rng.choice(("", eight))
    size = 1 if pages else size
    nodes = _log(rng, 1, 64)
    most = int(min(_MOST_BYTES / (2 * kv_heads * head_dim * size), _MOST_PRODUCTS / (heads * nodes * head_dim)))  # tokens in all
    tokens = _log(rng, 1, min(32768, most - nodes))
    batch = _log(rng, 1, max(1, min(64, most // (tokens + nodes))))
    window = rng.choice((-1, -1, _log(rng, 64, 4096)))
    return _tree(dtype, pages, batch, tokens, nodes, rng.choice((1, 2, 3, 4)), heads, kv_heads, head_dim, page, window,
                 rng.choice((0, 0, 3, 16)), rng.choice((0.25, 1.0, 4.0)))


# ---- what a user's program has in hand ---------------------------------------------------------------------------------


def _spread(case, most, skew=1.0):
    """Sizes of the sequences, the last of them ``most``: part of the case, their order is the seed's."""
    n = case["batch"]
    return [max(1, math.ceil(most * ((b + 1) / n) ** skew)) for b in range(n)]


def _starts(case):
    """Where the new tokens of the sequences begin, one place beside each size of ``_spread``."""
    n = case["batch"]
    return [case["first"] * ((5 * b + 1) % n + 1) // n for b in range(n)]


def _drafts(case):
    """Drafted tokens of the sequences, one number beside each size of ``_spread``: the first has all."""
    n = case["batch"]
    return [1 + (case["nodes"] - 1) * (n - (7 * b) % n) // n for b in range(n)]


def _shuffled(values, gen):
    order = torch.randperm(len(values), generator=gen)
    return torch.tensor(values)[order]


def _pool(lengths, page, gen):
    """``(page table, pages in the pool)``: every sequence's pages anywhere in a pool with some to spare, -1 behind them."""
    needed = (lengths + page - 1) // page
    columns = int(needed.max())
    pages = int(needed.sum()) + 3
    places = torch.randperm(pages, generator=gen)
    taken = torch.arange(columns)[None] < needed[:, None]
    table = torch.full((len(lengths), columns), -1, dtype=torch.int64)
    table[taken] = places[: int(needed.sum())]
    return table.to(torch.int32).cuda(), pages


def _ancestors(case):
    """``(seen, depth)`` of the tree's nodes: a 0/1 matrix of who sees whom, and how far from the root they are."""
    N = case["nodes"]
    seen, depth = torch.eye(N, dtype=torch.int64), [0] * N
    for i in range(1, N):
        parent = (i - 1) // case["branch"]
        seen[i] |= seen[parent]
        depth[i] = depth[parent] + 1
    return seen, torch.tensor(depth)


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    KV, D, page = case["kv_heads"], case["head_dim"], case["page"]

    def normal(*shape):
        return torch.randn(shape, generator=dev, device="cuda", dtype=dtype)

    def held(*shape):
        """``(keys or values as they are held, their scales)``, of normal numbers."""
        if not case["pages"]:
            return normal(*shape), None
        # codes of rows whose largest number is some three times their root mean square
        size = torch.randn(shape[:-1], generator=dev, device="cuda").mul_(0.3).exp_()
        if case["pages"] == "int8":
            codes = torch.randn(shape, generator=dev, device="cuda", dtype=torch.float16).mul_(40).round_().clamp_(-127, 127).to(torch.int8)
            return codes, size / 40
        codes = torch.randn(shape, generator=dev, device="cuda", dtype=torch.float16).mul_(140).clamp_(-448, 448).to(torch.float8_e4m3fn)
        return codes, size / 140

    def pool(pages):
        k_pages, k_scales = held(pages, KV, page, D)
        v_pages, v_scales = held(pages, KV, page, D)
        return dict(k_pages=k_pages, v_pages=v_pages, scales=None if k_scales is None else (k_scales, v_scales))

    if case["kind"] == "store":
        B, R, H = case["batch"], case["rows"], case["heads"]
        start, counts = _shuffled(list(zip(_starts(case), _spread(case, R))), gen).T
        table, pages = _pool(start + counts, page, gen)
        qkv = normal(B, R, H + 2 * KV, D).permute(0, 2, 1, 3)  # as one projection gives them
        half = case["rotated"] // 2
        inv_freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(1, half))
        return dict(case=case, q=qkv[:, :H], k=qkv[:, H:H + KV], v=qkv[:, H + KV:], table=table, **pool(pages),
                    start=start.to(torch.int32).cuda(), counts=counts.to(torch.int32).cuda(),
                    inv_freq=inv_freq.float().cuda() if half else None)
    if case["kind"] == "keep":
        B, N, most = case["batch"], case["nodes"], case["kept"]
        start, counts = _shuffled(list(zip(_starts(case), [1 + (3 * b) % most for b in range(B)])), gen).T
        table, pages = _pool(start + N, page, gen)
        kept = torch.full((B, most), -1, dtype=torch.int64)  # some of the first drafts, then others from further back
        for b, n in enumerate(counts.tolist()):
            here = min(int(torch.randint(1, n + 1, (), generator=gen)), n)
            here = max(here, 2 * n - N)
            kept[b, :here] = torch.arange(here)
            kept[b, here:n] = torch.sort(torch.randperm(N - n, generator=gen)[: n - here]).values + n
        return dict(case=case, table=table, **pool(pages), start=start.to(torch.int32).cuda(), counts=counts.to(torch.int32).cuda(),
                    kept=kept.to(torch.int32).cuda())
    B, H, Np = case["batch"], case["heads"], case["persistent"]
    state = dict(case=case, k_pers=None, v_pers=None, pers_scales=None)
    if case["kind"] == "attend":
        lengths = _shuffled(_spread(case, case["tokens"], case["skew"]), gen)
        state.update(q=normal(B, H, D), pos=(lengths - 1).to(torch.int32).cuda())
    else:
        start, counts = _shuffled(list(zip(_spread(case, case["tokens"], case["skew"]), _drafts(case))), gen).T
        lengths, N = start + counts, case["nodes"]
        seen, depth = _ancestors(case)
        bits = (seen << torch.arange(N)).sum(dim=1)  # (bit 63 is the sign)
        state.update(q=normal(B, N, H, D).permute(0, 2, 1, 3), start=start.to(torch.int32).cuda(), counts=counts.to(torch.int32).cuda(),
                     seen=bits.expand(B, N).contiguous().cuda(), positions=(start[:, None] + depth).to(torch.int32).cuda())
    table, pages = _pool(lengths, page, gen)
    state.update(table=table, **pool(pages))
    if Np:
        (state["k_pers"], a), (state["v_pers"], b) = held(KV, Np, D), held(KV, Np, D)
        state["pers_scales"] = None if a is None else (a, b)
    return state


# ---- the operators ------------------------------------------------------------------------------------------------------


def run(s):
    if own:
        return _run_own(s)
    return {"store": _plain_store, "attend": _plain_attend, "tree": _plain_tree, "keep": _plain_keep}[s["case"]["kind"]](s)


def _run_own(s):
    from titanmac_b200 import paged_append, paged_attention, paged_keep, paged_read, paged_tree_attention

    case = s["case"]
    if case["kind"] == "store":
        q = paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["start"], counts=s["counts"], q=s["q"],
                         q_out=_buffer(s, "q"), inv_freq=s["inv_freq"], interleaved=case["interleaved"], scales=s["scales"])
        k, v = paged_read(s["k_pages"], s["v_pages"], s["table"], s["start"], counts=s["counts"], scales=s["scales"],
                          k_out=_buffer(s, "k"), v_out=_buffer(s, "v"))
        return dict(k=k, v=v, q=q, k_scales=s["scales"][0], v_scales=s["scales"][1])
    if case["kind"] == "keep":
        paged_keep(s["k_pages"], s["v_pages"], s["table"], s["start"], s["kept"], s["counts"], scales=s["scales"])
        return _pages(s)
    window = None if case["window"] < 0 else case["window"]
    if case["kind"] == "attend":
        return paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["pos"], window=window, k_pers=s["k_pers"],
                               v_pers=s["v_pers"], scales=s["scales"], pers_scales=s["pers_scales"])
    return paged_tree_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["start"], s["seen"], counts=s["counts"],
                                positions=s["positions"], window=window, k_pers=s["k_pers"], v_pers=s["v_pers"], out=_buffer(s, "q"),
                                scales=s["scales"], pers_scales=s["pers_scales"])


def _buffer(s, name):
    """Where results of the shape of ``s[name] [B, heads, rows, head_dim]`` go, the heads of a row side by side; what is behind a
    sequence's last row stays as it is."""
    if name + "_out" not in s:
        B, H, R, D = s[name].shape
        s[name + "_out"] = torch.zeros((B, R, H, D), dtype=s[name].dtype, device=s[name].device).permute(0, 2, 1, 3)
    return s[name + "_out"]


def _pages(s):
    """All that ``paged_keep`` moves, whole: codes as they are, since they are moved and not computed."""
    found = dict(k_pages=s["k_pages"], v_pages=s["v_pages"])
    if s["scales"] is not None:
        found.update(k_scales=s["scales"][0], v_scales=s["scales"][1])
    return found


def _turn(x, cos, sin, interleaved):
    """``x [B, heads, rows, head_dim]`` in fp32, the first ``2 * cos.shape[-1]`` of a head rotated in pairs."""
    half = cos.shape[-1]
    part = x[..., : 2 * half]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half], part[..., half:])
    turned = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(turned, dim=-1).flatten(-2) if interleaved else torch.cat(turned, dim=-1)
    return torch.cat((turned, x[..., 2 * half:]), dim=-1)


def _code(x, form):
    """``(codes, scales)`` of rows of fp32 numbers."""
    largest = x.abs().amax(dim=-1)
    scale = (largest.double() / _LARGEST[form]).float().clamp(min=_LEAST_SCALE)  # (in fp32 torch multiplies by 1 / _LARGEST)
    scale = scale.masked_fill(~torch.isfinite(largest), math.nan)
    # the nearest code, in 64 bits: half a head's largest number, say, lies on a border, and the quotient's rounding would move it
    codes = x.double() / scale[..., None].double()
    codes = codes.masked_fill(torch.isnan(scale)[..., None], 0.0).clamp(-_LARGEST[form], _LARGEST[form])
    if form == "int8":
        return torch.round(codes).to(torch.int8), scale
    step = torch.ldexp(torch.ones_like(codes), torch.frexp(codes).exponent.clamp(min=-5) - 4)  # of numbers from 2^-6 on, three bits
    return (torch.round(codes / step) * step).float().to(torch.float8_e4m3fn), scale


def _new_slots(s, rows):
    """``(which rows are new tokens, their pages, their slots)`` for ``rows [B, R]`` counted from the start."""
    case, page = s["case"], s["case"]["page"]
    new = torch.arange(rows.shape[1], device=rows.device) < s["counts"][:, None]
    positions = s["start"].long()[:, None] + rows
    column = (positions // page).clamp(max=s["table"].shape[1] - 1)
    return new, s["table"].long().gather(1, column)[new], (positions % page)[new]


def _plain_store(s):
    case = s["case"]
    k, q, v = s["k"].float(), s["q"].float(), s["v"].float()
    rows = torch.arange(case["rows"], device=k.device).expand(case["batch"], -1)
    if case["rotated"]:
        positions = s["start"].long()[:, None] + rows
        angle = positions[:, None, :, None].double() * s["inv_freq"].double()
        cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
        k, q = _turn(k, cos, sin, case["interleaved"]), _turn(q, cos, sin, case["interleaved"])
    new, pages, slots = _new_slots(s, rows)
    found = {}
    for name, x, scales in (("k", k, s["scales"][0]), ("v", v, s["scales"][1])):
        codes, scale = _code(x, case["pages"])
        held = s[name + "_pages"].view(torch.uint8)  # (moving codes is moving bytes)
        held[pages, :, slots] = codes.view(torch.uint8).permute(0, 2, 1, 3)[new]
        scales[pages, :, slots] = scale.permute(0, 2, 1)[new]
        back = s[name + "_pages"].view(torch.uint8)[pages, :, slots].view(_EIGHTS[case["pages"]]).float() * scales[pages, :, slots][..., None]
        out = _buffer(s, name)
        out.permute(0, 2, 1, 3)[new] = back.to(out.dtype)
        found[name], found[name + "_scales"] = out, scales
    out = _buffer(s, "q")
    out.copy_(torch.where(new[:, None, :, None], q.to(out.dtype), out))
    return dict(found, q=out)


def _gathered(s, name, scale):
    """``[B, KV, persistent keys and then the sequence's, D]`` in fp32."""
    table = s["table"].long().clamp(min=0)
    B, KV, D = table.shape[0], s["case"]["kv_heads"], s["case"]["head_dim"]
    keys = s[name + "_pages"].view(torch.uint8)[table].view(s[name + "_pages"].dtype).float() if scale is not None \
        else s[name + "_pages"][table].float()
    if scale is not None:
        keys *= s["scales"][scale][table][..., None]
    keys = keys.permute(0, 2, 1, 3, 4).reshape(B, KV, -1, D)
    if s["k_pers"] is not None:
        pers = s[name + "_pers"].float()
        if scale is not None:
            pers = pers * s["pers_scales"][scale][..., None]
        keys = torch.cat((pers[None].expand(B, -1, -1, -1), keys), dim=2)
    return keys


def _weighted(q, keys, values, seen):
    """Attention of ``q [B, KV, rows, D]`` over ``keys`` where ``seen``."""
    scores = q @ keys.transpose(2, 3) / math.sqrt(q.shape[-1])
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    weights = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    total = weights.sum(dim=-1, keepdim=True)
    return (weights @ values) / total.masked_fill(total == 0, 1.0)


def _plain_attend(s):
    case = s["case"]
    B, H, D = s["q"].shape
    KV, eight = case["kv_heads"], s["scales"] is not None
    keys, values = _gathered(s, "k", 0 if eight else None), _gathered(s, "v", 1 if eight else None)
    at = torch.arange(keys.shape[2], device=keys.device) - case["persistent"]
    pos = s["pos"].long()[:, None]
    seen = (at <= pos) & (at >= 0)
    if case["window"] >= 0:
        seen &= at >= pos - case["window"]
    seen = (seen | (at < 0))[:, None, None]
    return _weighted(s["q"].float().view(B, KV, H // KV, D), keys, values, seen).reshape(B, H, D).to(s["q"].dtype)


def _plain_tree(s):
    case = s["case"]
    B, H, N, D = s["q"].shape
    KV, eight = case["kv_heads"], s["scales"] is not None
    keys, values = _gathered(s, "k", 0 if eight else None), _gathered(s, "v", 1 if eight else None)
    at = torch.arange(keys.shape[2], device=keys.device) - case["persistent"]
    start, counts = s["start"].long()[:, None, None], s["counts"].long()[:, None, None]
    node = at - start  # [B, 1, keys]
    seen = (at >= 0) & (node < 0)
    if case["window"] >= 0:
        seen = seen & (at >= s["positions"].long()[:, :, None] - case["window"])
    drafted = (node >= 0) & (node < counts)
    seen = seen | (drafted & ((s["seen"][:, :, None] >> node.clamp(0, 63)) & 1).bool()) | (at < 0)
    grouped = s["q"].float().reshape(B, KV, (H // KV) * N, D)
    seen = seen[:, None, None].expand(B, 1, H // KV, N, -1).reshape(B, 1, (H // KV) * N, -1)
    found = _weighted(grouped, keys, values, seen).reshape(B, H, N, D)
    out = _buffer(s, "q")
    out.copy_(torch.where((torch.arange(N, device=out.device) < counts[:, 0])[:, None, :, None], found.to(out.dtype), out))
    return out


def _plain_keep(s):
    kept = s["kept"].long().clamp(min=0)
    rows = torch.arange(kept.shape[1], device=kept.device).expand(kept.shape[0], -1)
    _, pages, slots = _new_slots(s, rows)
    _, from_pages, from_slots = _new_slots(s, kept)
    found = _pages(s)
    for x in found.values():
        x = x.view(torch.uint8) if x.element_size() == 1 else x  # (moving codes is moving bytes)
        x[pages, :, slots] = x[from_pages, :, from_slots]
    return found


def work(case):
    size = _DTYPES[case["dtype"]].itemsize
    KV, D = case["kv_heads"], case["head_dim"]
    token = 2 * KV * (D + 4 if case["pages"] else D * size)  # of keys and values, with their scales
    if case["kind"] == "store":
        rows, H = sum(_spread(case, case["rows"])), case["heads"]
        # the rows in; queries, pages and what these stand for out
        return dict(bytes=rows * ((2 * H + 4 * KV) * D * size + token) + case["batch"] * 8 + case["rotated"] * 2,
                    flops=rows * (3 * (H + KV) * case["rotated"] + 2 * KV * D * 3))
    if case["kind"] == "keep":
        rows = sum(1 + (3 * b) % case["kept"] for b in range(case["batch"]))
        return dict(bytes=2 * rows * token + 4 * rows, flops=0)
    H, Np, window = case["heads"], case["persistent"], case["window"]
    lengths = _spread(case, case["tokens"], case["skew"])
    if case["kind"] == "attend":
        keys = sum(min(n, window + 1) if window >= 0 else n for n in lengths)
        every = keys + case["batch"] * Np
        return dict(bytes=(keys + Np) * token + 2 * case["batch"] * H * D * size, flops=4 * every * H * D)
    depth, keys, pairs, nodes = _ancestors(case)[1].tolist(), 0, 0, 0
    for n, count in zip(lengths, _drafts(case)):
        context = [min(n, max(0, window - d)) if window >= 0 else n for d in depth[:count]]
        keys += max(context) + count
        pairs += sum(context) + sum(depth[:count]) + count * (1 + Np)
        nodes += count
    return dict(bytes=(keys + Np) * token + 2 * nodes * H * D * size, flops=4 * pairs * H * D)


# ---- the same from the definitions, in 64 bits --------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _exact_store, "attend": _exact_attend, "tree": _exact_tree, "keep": _exact_keep}[case["kind"]](s)


def _number(s, name, pages, head, slots):
    """Keys or values of one head at those places, in 64 bits."""
    x = s[name + "_pages"]
    if s["scales"] is None:
        return x[pages, head, slots].double()
    codes = x.view(torch.uint8)[pages, head, slots].view(x.dtype)
    return codes.double() * s["scales"][name == "v"][pages, head, slots].double()[..., None]


def _exact_store(s):
    case = s["case"]
    B, H, R, D = s["q"].shape
    KV, half, page = case["kv_heads"], case["rotated"] // 2, case["page"]
    i = torch.arange(half, device=s["q"].device)
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, half + i)
    found = {name: torch.zeros(s[name].shape, dtype=torch.float64, device=i.device) for name in "qkv"}
    scales = [x.double() for x in s["scales"]]
    for b, (start, count) in enumerate(zip(s["start"].tolist(), s["counts"].tolist())):
        at = torch.arange(start, start + count, device=i.device)
        new = {name: s[name][b, :, :count].double() for name in "qkv"}
        if half:  # a pair as a complex number, times exp(i angle)
            phase = torch.polar(torch.ones((count, half), dtype=torch.float64, device=i.device), at[:, None].double() * s["inv_freq"].double())
            for x in (new["k"], new["q"]):
                z = torch.complex(x[..., first], x[..., second]) * phase
                x[..., first], x[..., second] = z.real, z.imag
        found["q"][b, :, :count] = new["q"]
        pages = s["table"][b].long()[at // page]
        for x, held in ((new["k"], scales[0]), (new["v"], scales[1])):
            scale = (x.abs().amax(dim=2) / _LARGEST[case["pages"]]).float().double()  # (it is held in 32 bits)
            held[pages, :, at % page] = scale.T
            codes = x / scale[..., None]
            if case["pages"] == "int8":
                codes = codes.round()
            else:  # three bits behind the first one, which is worth 2^-6 at the least
                step = torch.exp2(torch.floor(torch.log2(codes.abs().clamp(min=2.0 ** -6))) - 3)
                codes = (codes / step).round() * step
            x.copy_(codes * scale[..., None])
        found["k"][b, :, :count], found["v"][b, :, :count] = new["k"], new["v"]
    return dict(found, k_scales=scales[0], v_scales=scales[1])


def _exact_attend(s):
    case = s["case"]
    KV, D, page = case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    group = case["heads"] // KV
    for b, pos in enumerate(s["pos"].tolist()):
        low = max(0, pos - case["window"]) if case["window"] >= 0 else 0
        at = torch.arange(low, pos + 1, device=out.device)
        pages = s["table"][b].long()[at // page]
        for h in range(KV):
            keys, values = _with_persistent(s, h, pages, at % page)
            rows = slice(h * group, (h + 1) * group)
            out[b, rows] = torch.softmax(s["q"][b, rows].double() @ keys.T * D ** -0.5, dim=-1) @ values
    return out


def _with_persistent(s, h, pages, slots):
    found = []
    for name in "kv":
        x = _number(s, name, pages, h, slots)
        if s["k_pers"] is not None:
            pers = s[name + "_pers"][h].double()
            if s["pers_scales"] is not None:
                pers = pers * s["pers_scales"][name == "v"][h].double()[:, None]
            x = torch.cat((x, pers))
        found.append(x)
    return found


def _exact_tree(s):
    case = s["case"]
    KV, D, page, Np, window = case["kv_heads"], case["head_dim"], case["page"], case["persistent"], case["window"]
    group = case["heads"] // KV
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    tree, depth = _ancestors(case)
    for b, (start, count) in enumerate(zip(s["start"].tolist(), s["counts"].tolist())):
        low = max(0, start - window) if window >= 0 else 0
        at = torch.arange(low, start + count, device=out.device)
        pages = s["table"][b].long()[at // page]
        hidden = torch.zeros((count, len(at) + Np), dtype=torch.bool, device=out.device)
        hidden[:, start - low: len(at)] = (tree[:count, :count] == 0).to(out.device)
        if window >= 0:
            hidden[:, : start - low] = at[: start - low] < start + depth[:count, None].to(out.device) - window
        for h in range(KV):
            keys, values = _with_persistent(s, h, pages, at % page)
            rows = slice(h * group, (h + 1) * group)
            scores = s["q"][b, rows, :count].double() @ keys.T * D ** -0.5
            out[b, rows, :count] = torch.softmax(scores.masked_fill(hidden, -math.inf), dim=-1) @ values
    return out


def _exact_keep(s):
    page = s["case"]["page"]
    found = {name: x.clone() for name, x in _pages(s).items()}
    before = _pages(s)
    for b, (start, count) in enumerate(zip(s["start"].tolist(), s["counts"].tolist())):
        for i, j in enumerate(s["kept"][b, :count].tolist()):
            to, source = (int(s["table"][b, t // page]) for t in (start + i, start + j))
            for name, x in before.items():
                found[name][to, :, (start + i) % page] = x[source, :, (start + j) % page]
    return found
