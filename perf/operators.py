"""Serving from a paged key-value cache, and what a model says of its tokens, as cases that can be timed and compared.

``listed()`` holds the cases, ``draw(rng)`` gives more of the same ranges.  A case is a dict of plain values; its ``kind`` says
which operator it is:

    append     keys and values of new tokens into a paged cache, keys and queries rotated by their positions on the way
    attend     attention of one new token per sequence over its paged keys (window, persistent keys, shared heads)
    logprobs   log-probabilities of given tokens, the entropy of every row and its most likely alternatives; with ``train``
               the gradient of the logits too

With ``own`` false ``run`` computes them from elementary operations in fp32; with ``own`` true it makes the package's calls.
"""

import math
import os
import sys

import torch

sys.path.insert(1, os.path.join(os.getcwd(), "titanmac-standalone_b200"))

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_MOST_BYTES = 2e9  # of keys and values that a drawn case reads


def _append(dtype, batch, rows, heads, kv_heads, head_dim, page, rotated, interleaved=False, first=0):
    """``rows`` new tokens for the longest sequence, fewer for the others; they start somewhere in ``0 .. first``."""
    return dict(kind="append", dtype=dtype, batch=batch, rows=rows, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                rotated=rotated, interleaved=interleaved, first=first)


def _attend(dtype, batch, tokens, heads, kv_heads, head_dim, page, window=-1, persistent=0, skew=1.0):
    """The longest sequence has ``tokens`` keys, the others a share of that (``skew``: how fast it falls)."""
    return dict(kind="attend", dtype=dtype, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                page=page, window=window, persistent=persistent, skew=skew)


def _logprobs(dtype, batch, tokens, vocab, top, train=False, masked=0):
    """``masked``: so many ids at the end of the vocabulary have a logit of -inf."""
    return dict(kind="logprobs", dtype=dtype, batch=batch, tokens=tokens, vocab=vocab, top=top, train=train, masked=masked)


def listed():
    return [
        # a serving step of many sequences: one token each, heads that share keys
        dict(_append("bf16", 64, 1, 32, 8, 128, 16, 128, first=1000), name="append_step"),
        # prompts of several lengths go into the cache at once: the layer width of the long-context configuration
        dict(_append("bf16", 8, 4096, 16, 16, 128, 64, 128), name="append_prompts"),
        # a chunk of a prompt behind an earlier one, part of the head rotated in pairs of neighbours, pages of no power of two
        dict(_append("fp16", 3, 731, 10, 5, 64, 24, 32, interleaved=True, first=100000), name="append_chunk_odd"),
        # one answer being written: the default geometry, all keys of a short conversation
        dict(_attend("bf16", 1, 700, 10, 10, 64, 64, persistent=16), name="attend_one_sequence"),
        # serving the default model: its window and persistent rows for 256 sequences
        dict(_attend("bf16", 256, 2048, 10, 10, 64, 64, window=512, persistent=16, skew=0.25), name="attend_window_batch"),
        # a mixed batch, a few long conversations among many short ones, heads that share keys
        dict(_attend("fp16", 48, 16384, 32, 8, 128, 32, skew=4.0), name="attend_ragged_grouped"),
        # long documents
        dict(_attend("bf16", 12, 65536, 32, 4, 128, 128, skew=0.5), name="attend_long"),
        # full precision, pages and a head size that fit no tile
        dict(_attend("fp32", 5, 3001, 8, 2, 96, 17, persistent=3), name="attend_fp32_odd"),
        # what a serving step reports of the tokens it chose: few rows, the default vocabulary, its padding masked
        dict(_logprobs("bf16", 8, 1, 128000, 20, masked=37), name="logprobs_step"),
        # scoring given texts with alternatives, a vocabulary whose rows start at any address
        dict(_logprobs("fp16", 2, 1500, 49999, 5), name="logprobs_score"),
        # a training step on log-probabilities and entropy at the default vocabulary
        dict(_logprobs("bf16", 4, 1024, 128000, 0, train=True), name="logprobs_train"),
        # the same of a small model in full precision, alternatives as well
        dict(_logprobs("fp32", 6, 47, 1001, 8, train=True), name="logprobs_train_small"),
    ]


def _log(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(("append", "attend", "logprobs"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if kind == "logprobs":
        vocab = _log(rng, 50, 128000)
        train = rng.random() < 0.5
        rows = _log(rng, 1, max(1, min(4096, int((5e8 if train else 2.5e8) / vocab))))
        batch = rng.choice([b for b in (1, 2, 3, 4, 7, 8) if b <= rows])
        return _logprobs(dtype, batch, max(1, rows // batch), vocab, min(vocab // 2, rng.choice((0, 1, 3, 5, 10, 20, 32))), train,
                         rng.choice((0, 0, 1, vocab // 10)))
    kv_heads = rng.choice((1, 2, 4, 5, 8, 10, 16))
    heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 7, 8))
    head_dim = rng.choice((64, 64, 128, 128, 32, 96, 256))
    page = rng.choice((16, 32, 64, 128, _log(rng, 1, 200)))
    size = _DTYPES[dtype].itemsize
    if kind == "append":
        row = (heads + 2 * kv_heads) * head_dim
        rows = _log(rng, 1, 4096)
        batch = _log(rng, 1, max(1, min(256, int(2e8 / (rows * row)))))
        interleaved = rng.random() < 0.4
        most = int(1e9 / (batch * kv_heads * head_dim * 2 * size))  # earlier keys and values stand in the pages too
        return _append(dtype, batch, rows, heads, kv_heads, head_dim, page, rng.choice((0, head_dim // 2, head_dim)), interleaved,
                       rng.choice((0, 0, _log(rng, 1, max(1, min(100000, most))))))
    tokens = _log(rng, 1, 65536)
    batch = _log(rng, 1, max(1, min(256, int(_MOST_BYTES / (tokens * kv_heads * head_dim * 2 * size)))))
    window = rng.choice((-1, -1, _log(rng, 1, 4096)))
    return _attend(dtype, batch, tokens, heads, kv_heads, head_dim, page, window, rng.choice((0, 0, 3, 16)), rng.choice((0.25, 1.0, 4.0)))


# ---- what a user's program has in hand ---------------------------------------------------------------------------------


def _spread(case, most, skew=1.0):
    """Sizes of the sequences, the last of them ``most``: part of the case, their order is the seed's."""
    n = case["batch"]
    return [max(1, math.ceil(most * ((b + 1) / n) ** skew)) for b in range(n)]


def _starts(case):
    """Where the new tokens of the sequences begin, one place beside each size of ``_spread``."""
    n = case["batch"]
    return [case["first"] * ((5 * b + 1) % n + 1) // n for b in range(n)]


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


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=dev, device="cuda", dtype=dtype)

    if case["kind"] == "append":
        B, R, H, KV, D = case["batch"], case["rows"], case["heads"], case["kv_heads"], case["head_dim"]
        start, counts = _shuffled(list(zip(_starts(case), _spread(case, R))), gen).T
        table, pages = _pool(start + counts, case["page"], gen)
        qkv = normal(B, R, H + 2 * KV, D).permute(0, 2, 1, 3)  # as one projection gives them
        half = case["rotated"] // 2
        inv_freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(1, half))
        return dict(case=case, q=qkv[:, :H], k=qkv[:, H:H + KV], v=qkv[:, H + KV:], table=table,
                    k_pages=normal(pages, KV, case["page"], D), v_pages=normal(pages, KV, case["page"], D),
                    start=start.to(torch.int32).cuda(), counts=counts.to(torch.int32).cuda(),
                    inv_freq=inv_freq.float().cuda() if half else None)
    if case["kind"] == "attend":
        H, KV, D = case["heads"], case["kv_heads"], case["head_dim"]
        lengths = _shuffled(_spread(case, case["tokens"], case["skew"]), gen)
        table, pages = _pool(lengths, case["page"], gen)
        state = dict(case=case, q=normal(case["batch"], H, D), k_pages=normal(pages, KV, case["page"], D),
                     v_pages=normal(pages, KV, case["page"], D), table=table, pos=(lengths - 1).to(torch.int32).cuda(),
                     k_pers=None, v_pers=None)
        if case["persistent"]:
            state.update(k_pers=normal(KV, case["persistent"], D), v_pers=normal(KV, case["persistent"], D))
        return state
    B, T, V = case["batch"], case["tokens"], case["vocab"]
    logits = torch.randn((B, T, V), generator=dev, device="cuda").mul_(2.5)
    targets = torch.randint(0, V - case["masked"], (B, T), generator=gen).cuda()
    likely = torch.rand((B, T, 1), generator=dev, device="cuda") * 12  # the model has an opinion of the text
    logits.scatter_add_(2, targets[..., None], likely)
    if case["masked"]:
        logits[..., V - case["masked"]:] = -math.inf
    if T > 1:  # the last token of a text has no next one
        targets[:, -1] = -100
    state = dict(case=case, logits=logits.to(dtype), targets=targets)
    if case["train"]:
        state.update(d_logprobs=torch.randn((B, T), generator=dev, device="cuda") / (B * T),
                     d_entropy=torch.full((B, T), 0.01 / (B * T), device="cuda"))
        if case["top"]:
            state.update(d_top=torch.randn((B, T, case["top"]), generator=dev, device="cuda") / (B * T))
    return state


# ---- the operators ------------------------------------------------------------------------------------------------------


def run(s):
    if own:
        return _run_own(s)
    return {"append": _plain_append, "attend": _plain_attend, "logprobs": _plain_logprobs}[s["case"]["kind"]](s)


def _run_own(s):
    from titanmac_b200 import paged_append, paged_attention, token_logprobs

    case = s["case"]
    if case["kind"] == "append":
        q = paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["start"], counts=s["counts"], q=s["q"],
                         q_out=_query_buffer(s), inv_freq=s["inv_freq"], interleaved=case["interleaved"])
        return dict(k_pages=s["k_pages"], v_pages=s["v_pages"], q=q)
    if case["kind"] == "attend":
        return paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["pos"],
                               window=None if case["window"] < 0 else case["window"], k_pers=s["k_pers"], v_pers=s["v_pers"])
    if not case["train"]:
        with torch.no_grad():
            out = token_logprobs(s["logits"], s["targets"], n_top=case["top"])
        found = dict(logprobs=out.logprobs, entropy=out.entropy)
    else:
        with torch.enable_grad():
            logits = s["logits"].detach().requires_grad_(True)
            out = token_logprobs(logits, s["targets"], n_top=case["top"])
            wanted, given = [out.logprobs, out.entropy], [s["d_logprobs"], s["d_entropy"]]
            if case["top"]:
                wanted.append(out.top_logprobs)
                given.append(s["d_top"])
            (d_logits,) = torch.autograd.grad(wanted, logits, given)
        found = dict(logprobs=out.logprobs.detach(), entropy=out.entropy.detach(), d_logits=d_logits)
    if case["top"]:
        found.update(top_ids=out.top_ids, top_logprobs=out.top_logprobs.detach())
    return found


def _query_buffer(s):
    """Where the rotated queries go, ``[B, heads, rows, head_dim]`` with the heads of a row side by side; what is behind a
    sequence's last new row stays as it is."""
    if "q_out" not in s:
        B, H, R, D = s["q"].shape
        s["q_out"] = torch.zeros((B, R, H, D), dtype=s["q"].dtype, device=s["q"].device).permute(0, 2, 1, 3)
    return s["q_out"]


def _turn(x, cos, sin, interleaved):
    """``x [B, heads, rows, head_dim]`` in fp32, the first ``2 * cos.shape[-1]`` of a head rotated in pairs."""
    half = cos.shape[-1]
    part = x[..., : 2 * half]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half], part[..., half:])
    turned = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(turned, dim=-1).flatten(-2) if interleaved else torch.cat(turned, dim=-1)
    return torch.cat((turned, x[..., 2 * half:]), dim=-1)


def _plain_append(s):
    case, page = s["case"], s["case"]["page"]
    k, q = s["k"].float(), s["q"].float()
    rows = torch.arange(case["rows"], device=k.device)
    positions = s["start"].long()[:, None] + rows  # [B, R]
    if case["rotated"]:
        angle = positions[:, None, :, None].double() * s["inv_freq"].double()
        cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
        k, q = _turn(k, cos, sin, case["interleaved"]), _turn(q, cos, sin, case["interleaved"])
    new = rows < s["counts"][:, None]
    column = (positions // page).clamp(max=s["table"].shape[1] - 1)
    pages, slots = s["table"].long().gather(1, column)[new], (positions % page)[new]
    s["k_pages"][pages, :, slots] = k.permute(0, 2, 1, 3)[new].to(s["k_pages"].dtype)
    s["v_pages"][pages, :, slots] = s["v"].permute(0, 2, 1, 3)[new]
    out = _query_buffer(s)
    out.copy_(torch.where(new[:, None, :, None], q.to(out.dtype), out))
    return dict(k_pages=s["k_pages"], v_pages=s["v_pages"], q=out)


def _plain_attend(s):
    case = s["case"]
    B, H, D = s["q"].shape
    KV = case["kv_heads"]
    table = s["table"].long().clamp(min=0)

    def gathered(pages, pers):  # [B, KV, persistent keys and then the sequence's, D]
        own_keys = pages[table].permute(0, 2, 1, 3, 4).reshape(B, KV, -1, D)
        if pers is not None:
            own_keys = torch.cat((pers[None].expand(B, -1, -1, -1), own_keys), dim=2)
        return own_keys.float()

    keys, values = gathered(s["k_pages"], s["k_pers"]), gathered(s["v_pages"], s["v_pers"])
    Np = case["persistent"]
    at = torch.arange(keys.shape[2], device=keys.device) - Np
    pos = s["pos"].long()[:, None]
    seen = (at <= pos) & (at >= 0)
    if case["window"] >= 0:
        seen &= at >= pos - case["window"]
    seen = (seen | (at < 0))[:, None, None]
    scores = s["q"].float().view(B, KV, H // KV, D) @ keys.transpose(2, 3) / math.sqrt(D)
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    weights = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    total = weights.sum(dim=-1, keepdim=True)
    out = (weights @ values) / total.masked_fill(total == 0, 1.0)
    return out.reshape(B, H, D).to(s["q"].dtype)


def _ranked(x):
    """Whole numbers in the order of ``x [.., V]``, the lower index first among equal values."""
    bits = (x.float() + 0.0).view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
    return (order << 32) - torch.arange(x.shape[-1], device=x.device)


def _plain_logprobs(s):
    case, targets = s["case"], s["targets"]
    x = s["logits"].float()
    top = x.amax(dim=-1, keepdim=True)
    logp = (x - top) - torch.log(torch.exp(x - top).sum(dim=-1, keepdim=True))
    p = torch.exp(logp)
    entropy = -(p * logp.masked_fill(p == 0, 0.0)).sum(dim=-1)
    counted = targets != -100
    at = targets.masked_fill(~counted, 0)[..., None]
    found = dict(logprobs=logp.gather(-1, at)[..., 0].masked_fill(~counted, 0.0), entropy=entropy)
    if case["top"]:
        keys = torch.topk(_ranked(s["logits"]), case["top"], dim=-1).values
        found["top_ids"] = (-keys) & 0xFFFFFFFF
        found["top_logprobs"] = logp.gather(-1, found["top_ids"])
    if case["train"]:
        d_logprobs, d_entropy = s["d_logprobs"].masked_fill(~counted, 0.0)[..., None], s["d_entropy"][..., None]
        pulled = d_logprobs
        if case["top"]:
            pulled = pulled + s["d_top"].sum(dim=-1, keepdim=True)
        d = -p * (pulled + d_entropy * (logp.masked_fill(p == 0, 0.0) + entropy[..., None]))
        d.scatter_add_(-1, at, d_logprobs)
        if case["top"]:
            d.scatter_add_(-1, found["top_ids"], s["d_top"])
        found["d_logits"] = d.to(s["logits"].dtype)
    return found


def work(case):
    size = _DTYPES[case["dtype"]].itemsize
    if case["kind"] == "append":
        rows = sum(_spread(case, case["rows"]))
        per_row = (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]
        turned = (case["heads"] + case["kv_heads"]) * case["rotated"]
        return dict(bytes=2 * rows * per_row * size + case["batch"] * 8 + case["rotated"] * 2, flops=3 * rows * turned)
    if case["kind"] == "attend":
        window = case["window"]
        keys = sum(min(n, window + 1) if window >= 0 else n for n in _spread(case, case["tokens"], case["skew"]))
        every = keys + case["batch"] * case["persistent"]
        D, H, KV = case["head_dim"], case["heads"], case["kv_heads"]
        return dict(bytes=2 * (keys + case["persistent"]) * KV * D * size + 2 * case["batch"] * H * D * size, flops=4 * every * H * D)
    rows, V = case["batch"] * case["tokens"], case["vocab"]
    passes = 2 if case["train"] else 1  # the logits, and their gradient
    # (a training step reads the logits once: nothing but the gradient itself has to come behind the last of a row)
    return dict(bytes=rows * (V * size * passes + 16 + 12 * case["top"] + 8 * (passes - 1)), flops=rows * V * (5 if passes == 1 else 12))


# ---- the same from the definitions, in 64 bits --------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "logprobs": _exact_logprobs}[case["kind"]](s)


def _exact_append(s):
    case = s["case"]
    B, H, R, D = s["q"].shape
    half, page = case["rotated"] // 2, case["page"]
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    q = torch.zeros((B, H, R, D), dtype=torch.float64, device=k_pages.device)
    i = torch.arange(half, device=q.device)
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, half + i)
    for b, (start, count) in enumerate(zip(s["start"].tolist(), s["counts"].tolist())):
        at = torch.arange(start, start + count, device=q.device)
        new_k, new_q = s["k"][b, :, :count].double(), s["q"][b, :, :count].double()
        if half:  # a pair as a complex number, times exp(i angle)
            phase = torch.polar(torch.ones((count, half), dtype=torch.float64, device=q.device), at[:, None].double() * s["inv_freq"].double())
            for x in (new_k, new_q):
                z = torch.complex(x[..., first], x[..., second]) * phase
                x[..., first], x[..., second] = z.real, z.imag
        pages = s["table"][b].long()[at // page]
        k_pages[pages, :, at % page] = new_k.transpose(0, 1)
        v_pages[pages, :, at % page] = s["v"][b, :, :count].double().transpose(0, 1)
        q[b, :, :count] = new_q
    return dict(k_pages=k_pages, v_pages=v_pages, q=q)


def _exact_attend(s):
    case = s["case"]
    KV, D, page = case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b, pos in enumerate(s["pos"].tolist()):
        low = max(0, pos - case["window"]) if case["window"] >= 0 else 0
        at = torch.arange(low, pos + 1, device=out.device)
        pages = s["table"][b].long()[at // page]
        for h in range(KV):
            keys, values = s["k_pages"][pages, h, at % page].double(), s["v_pages"][pages, h, at % page].double()
            if case["persistent"]:
                keys, values = torch.cat((keys, s["k_pers"][h].double())), torch.cat((values, s["v_pers"][h].double()))
            group = slice(h * (case["heads"] // KV), (h + 1) * (case["heads"] // KV))
            out[b, group] = torch.softmax(s["q"][b, group].double() @ keys.T * D ** -0.5, dim=-1) @ values
    return out


def _exact_logprobs(s):
    case = s["case"]
    B, T, V = s["logits"].shape
    logits, targets = s["logits"].view(-1, V), s["targets"].view(-1)
    found = dict(logprobs=[], entropy=[])
    if case["top"]:
        found.update(top_ids=[], top_logprobs=[])
    if case["train"]:
        found.update(d_logits=[])
    for a in range(0, B * T, 512):
        x, y = logits[a:a + 512].double(), targets[a:a + 512]
        logp = torch.log_softmax(x, dim=-1)
        p = logp.exp()
        one_hot = torch.zeros_like(p)
        given = (y >= 0).nonzero()[:, 0]
        one_hot[given, y[given]] = 1.0
        finite = torch.where(p > 0, logp, 0.0)
        entropy = -(p * finite).sum(dim=-1)
        found["logprobs"].append((one_hot * finite).sum(dim=-1))
        found["entropy"].append(entropy)
        if case["top"]:
            order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, : case["top"]]
            found["top_ids"].append(order)
            found["top_logprobs"].append(logp.gather(1, order))
        if case["train"]:
            g = s["d_logprobs"].view(-1)[a:a + 512].double()[:, None] * (y >= 0)[:, None]
            d = g * one_hot - g * p - s["d_entropy"].view(-1)[a:a + 512].double()[:, None] * p * (finite + entropy[:, None])
            if case["top"]:
                e = s["d_top"].view(-1, case["top"])[a:a + 512].double()
                d = (d - p * e.sum(dim=-1, keepdim=True)).scatter_add(1, order, e)
            found["d_logits"].append(d)
    shapes = dict(logprobs=(B, T), entropy=(B, T), top_ids=(B, T, -1), top_logprobs=(B, T, -1), d_logits=(B, T, V))
    return {name: torch.cat(parts).view(shapes[name]) for name, parts in found.items()}
