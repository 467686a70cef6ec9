"""Paged keys and values against plain forms in 64 bits: where tokens go, how they are rotated, what one token attends to."""

import pytest
import torch

import paged_reference as pr
from titanmac_b200 import PagedCache, TitanMAC, TitanMACConfig, _native, paged_append, paged_attention, token_logprobs

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _fresh_status():
    _native.poll_status(DEV)
    yield


def dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def numbers(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def reported():
    with pytest.raises(_native.TmwError):
        _native.poll_status(DEV)


def attend(lengths, heads, kv_heads, dh, page, dtype, window=None, n_p=0, seed=0, scale=0.0, fill="wild"):
    g = torch.Generator().manual_seed(seed + 1)
    k, v, table = pr.pool(lengths, page, kv_heads, dh, dtype, seed, fill=fill)
    q = torch.randn(len(lengths), heads, dh, generator=g).to(dtype)
    k_pers = v_pers = None
    if n_p:
        k_pers, v_pers = (torch.randn(kv_heads, n_p, dh, generator=g).to(dtype) for _ in range(2))
    pos = torch.tensor(lengths) - 1
    got = paged_attention(*dev(q, k, v, table), pos.to(torch.int32).to(DEV), window, *dev(k_pers, v_pers), scale=scale)
    _native.poll_status(DEV)
    want, bound = pr.attention(q, k, v, table, pos, window, k_pers, v_pers, scale)
    return got, want, bound


def check(got, want, bound):
    step = torch.finfo(got.dtype).eps / 2 if got.dtype != FF else 0.0  # one rounding of the output
    off = (got.double().cpu() - want).abs()
    allowed = bound + step * (want.abs() + bound) + torch.finfo(got.dtype).tiny
    assert (off <= allowed).all(), (off / allowed).max().item()


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("lengths,heads,kv_heads,dh,page,window,n_p", [
    ([1], 1, 1, 64, 16, None, 0),                        # one token
    ([1, 2, 15, 16, 17, 31, 33, 64], 4, 4, 64, 16, None, 0),  # tiles that end everywhere
    ([300], 10, 10, 64, 64, None, 16),                   # one sequence over many CTAs
    ([40, 1, 700, 0, 3], 8, 2, 128, 24, None, 3),        # ragged, a sequence without tokens, pages that end inside tiles
    ([513, 77, 0], 4, 2, 64, 7, 100, 5),                 # a window that begins inside a tile and a page
    ([50, 9], 2, 1, 64, 1, 0, 0),                        # the token itself alone, pages of one token
    ([129, 16], 16, 1, 128, 32, None, 0),                # sixteen heads on one
    ([65, 200], 14, 2, 96, 20, 150, 2),                  # seven heads on one
    ([90, 33], 40, 2, 32, 64, None, 1),                  # twenty heads on one
    ([150, 20], 6, 2, 256, 16, None, 17),                # wide heads
    ([70, 5], 3, 1, 16, 5, None, 0),
    ([70, 5], 3, 1, 8, 5, 30, 0),
    ([70, 5], 4, 2, 40, 16, None, 2),                    # a head size of no tile
    ([33, 12], 5, 5, 200, 48, None, 0),
    ([45, 100], 8, 2, 80, 16, None, 3),
    ([45, 100], 12, 1, 80, 9, 60, 0),
    ([45, 100], 3, 1, 192, 32, None, 0),
    ([70, 45], 20, 1, 192, 16, None, 1),
    ([70, 45], 2, 2, 144, 16, None, 1),                  # one head on one, wide, of no tile
    ([70, 45], 5, 1, 24, 16, None, 1),                   # five heads on one, on CUDA cores in every type
    ([70, 45], 18, 2, 16, 16, 20, 1),
])
def test_attention_against_64_bits(lengths, heads, kv_heads, dh, page, window, n_p, dtype):
    check(*attend(lengths, heads, kv_heads, dh, page, dtype, window, n_p, seed=len(lengths) * dh + page))


@pytest.mark.parametrize("dtype", [BF, FF])
def test_attention_of_many_short_sequences(dtype):
    """More sequences than threads of a CTA, several items to a CTA, sequences without tokens between them."""
    lengths = [(7 * b) % 40 for b in range(333)]
    check(*attend(lengths, 4, 2, 64, 16, dtype, seed=5))


def test_attention_of_a_large_batch():
    """Thousands of sequences: each lane of a warp counts the tiles of many, and most of the line lies in other CTAs."""
    g = torch.Generator().manual_seed(8)
    lengths = (torch.randint(0, 9, (5000,), generator=g) * (torch.rand(5000, generator=g) < 0.3)).tolist()
    lengths[777], lengths[4999] = 3000, 500
    check(*attend(lengths, 2, 1, 32, 16, BF, seed=6))


def test_calls_on_two_streams_at_once():
    """Different batches on two streams without a wait between them: nothing is shared but the pool."""
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    cases = []
    for i, lengths in enumerate(([700, 3, 90], [40] * 30)):
        k, v, table = pr.pool(lengths, 16, 2, 64, BF, i)
        q = torch.randn(len(lengths), 6, 64, generator=torch.Generator().manual_seed(i)).to(BF)
        pos = torch.tensor(lengths) - 1
        cases.append((dev(q, k, v, table) + [pos.to(torch.int32).to(DEV)], pr.attention(q, k, v, table, pos)))
    torch.cuda.synchronize(DEV)
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(paged_attention(*cases[i][0]))
    torch.cuda.synchronize(DEV)
    for results, (_, want) in zip(got, cases):
        check(results[0], *want)
        assert all(torch.equal(r, results[0]) for r in results)


@pytest.mark.parametrize("dtype,dh,heads", [(BF, 128, 8), (HF, 64, 3), (FF, 64, 2)])
def test_attention_of_one_long_sequence(dtype, dh, heads):
    """Every CTA has a part of the same item."""
    check(*attend([9000], heads, 1, dh, 64, dtype, seed=7, fill="normal"))


def test_attention_with_large_scores_and_a_scale():
    got, want, bound = attend([200, 31], 4, 2, 64, 16, FF, seed=9, scale=2.0)
    check(got, want, bound)


@pytest.mark.parametrize("dtype", [BF, HF, FF])
def test_weights_that_are_far_apart(dtype):
    """One key ahead of 4000 others by e^12: their weights are small and count together."""
    g = torch.Generator().manual_seed(3)
    n, dh = 4001, 64
    k, v, table = pr.pool([n], 64, 1, dh, dtype, 11)
    q = torch.zeros(1, 1, dh, dtype=dtype)
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    k[table[0, 3], 0, 5, 0] = 12.0  # score 12 at scale 1 / 8
    v[...] = (1.0 + 0.25 * torch.randn(v.shape, generator=g)).to(dtype)
    pos = torch.tensor([n - 1])
    got = paged_attention(*dev(q, k, v, table), pos.to(torch.int32).to(DEV))
    want, bound = pr.attention(q, k, v, table, pos)
    check(got, want, bound)


@pytest.mark.parametrize("dtype", [BF, FF])
def test_values_that_are_not_ordinary(dtype):
    """Seen infinities and NaN have the formula's consequences, for their own heads and sequences alone."""
    k, v, table = pr.pool([20, 20, 20, 20], 16, 2, 64, dtype, 2)
    q = torch.ones(4, 2, 64, dtype=dtype)
    k[table[0, 0], 0, 3] = float("nan")
    k[table[1, 0], 0] = -float("inf")  # all but the last four scores: weight 0
    k[table[1, 1], 1, :4] = float("inf")
    v[table[2, 1], 1, 2, 7] = float("inf")
    k[table[3, 0], 0] = -float("inf")
    k[table[3, 1], 0] = -float("inf")  # nothing but -inf
    pos = torch.full((4,), 19)
    got = paged_attention(*dev(q, k, v, table), pos.to(torch.int32).to(DEV)).double().cpu()
    want, bound = pr.attention(q, k, v, table, pos)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    fine = torch.isfinite(want)
    assert torch.isnan(got[0, 0]).all() and torch.isfinite(got[0, 1]).all() and torch.isfinite(got[1, 0]).all()
    assert ((got - want)[fine].abs() <= 2.0 ** -7 * want[fine].abs() + 1e-2).all()  # (the bound itself is not finite here)


def test_places_that_are_none():
    """A position or a page outside makes that sequence NaN, is reported, and leaves the others alone."""
    lengths = [40, 40, 40, 40]
    for change in ("page", "far_page", "position", "negative"):
        k, v, table = pr.pool(lengths, 16, 2, 64, BF, 4)
        q = torch.randn(4, 4, 64, generator=torch.Generator().manual_seed(1)).to(BF)
        pos = torch.full((4,), 39)
        want, bound = pr.attention(q, k, v, table, pos)
        if change == "page":
            table[2, 1] = k.shape[0]
        elif change == "far_page":
            table[2, 0] = -(1 << 31)
        else:
            pos[2] = 48 if change == "position" else -2
        got = paged_attention(*dev(q, k, v, table), pos.to(torch.int32).to(DEV))
        reported()
        assert torch.isnan(got[2]).all()
        rest = [0, 1, 3]
        check(got[rest], want[rest], bound[rest])
    # entries behind the tokens are not looked at, nor those in front of a window
    k, v, table = pr.pool(lengths, 16, 2, 64, BF, 4)
    want, bound = pr.attention(q, k, v, table, torch.full((4,), 39), window=5)
    table[:, :2] = 1 << 30
    check(paged_attention(*dev(q, k, v, table), numbers([39] * 4), window=5), want, bound)
    _native.poll_status(DEV)


def test_strides_outputs_and_the_same_bits_again():
    lengths, H, KV, dh = [300, 18, 1, 77], 8, 4, 64
    k, v, table = pr.pool(lengths, 16, KV, dh, BF, 8)
    wide = torch.randn(4, 3, H, dh + 3, generator=torch.Generator().manual_seed(2)).to(BF).to(DEV)
    q = wide[:, 1, :, 3:]  # rows at odd addresses
    table_wide = torch.full((4, table.shape[1] + 5), 99, dtype=torch.int32, device=DEV)
    table_wide[:, : table.shape[1]] = table.to(DEV)
    out = torch.full((4, H, dh + 1), 7.0, dtype=BF, device=DEV)
    k_d, v_d = dev(k, v)
    pos = numbers([n - 1 for n in lengths])
    got = paged_attention(q, k_d, v_d, table_wide[:, : table.shape[1]], pos, out=out[:, :, 1:])
    assert got.data_ptr() == out[:, :, 1:].data_ptr() and (out[:, :, 0] == 7).all()
    want, bound = pr.attention(q.cpu(), k, v, table, pos.cpu())
    check(got, want, bound)
    for _ in range(3):
        assert torch.equal(paged_attention(q, k_d, v_d, table_wide[:, : table.shape[1]], pos), got)


def test_offsets_past_31_bits():
    """A pool of 5 GB: pages whose offset no 32-bit number of elements or bytes holds."""
    pages, KV, page, dh = 20480, 1, 1024, 128  # 2.7e9 elements
    k = torch.empty((pages, KV, page, dh), dtype=BF, device=DEV)
    v = torch.empty_like(k)
    g = torch.Generator().manual_seed(1)
    new = [torch.randn(1, KV, 1500, dh, generator=g).to(BF) for _ in range(2)]
    table = torch.tensor([[pages - 1, 16500]], dtype=torch.int32, device=DEV)
    paged_append(*dev(*new), k, v, table, numbers([0]))
    assert torch.equal(k[pages - 1, 0].cpu(), new[0][0, 0, :1024]) and torch.equal(v[16500, 0, :476].cpu(), new[1][0, 0, 1024:])
    q = torch.randn(1, 4, dh, generator=g).to(BF)
    got = paged_attention(q.to(DEV), k, v, table, numbers([1499]))
    small = torch.zeros(2, KV, page, dh, dtype=BF), torch.zeros(2, KV, page, dh, dtype=BF)
    for t, x in zip(small, new):
        t[0, 0], t[1, 0, :476] = x[0, 0, :1024], x[0, 0, 1024:]
    check(got, *pr.attention(q, *small, torch.tensor([[0, 1]]), torch.tensor([1499])))


# ---- append -------------------------------------------------------------------------------------------------------------------


def expected_append(k, v, k_pages, v_pages, table, start, counts, q, q_out, inv_freq, interleaved):
    page = k_pages.shape[2]
    k_new, v_new = k_pages.double().clone(), v_pages.double().clone()
    q_new = None if q is None else q_out.double().clone()
    for b in range(k.shape[0]):
        if start[b] < 0:
            continue
        n = int(counts[b]) if counts is not None else k.shape[2]
        at = torch.arange(int(start[b]), int(start[b]) + n)
        turn = (lambda x: pr.rotated(x, at, inv_freq, interleaved)) if inv_freq is not None else (lambda x: x.double())
        k_turned = turn(k[b, :, :n])
        for r, t in enumerate(at.tolist()):
            k_new[table[b, t // page], :, t % page] = k_turned[:, r]
            v_new[table[b, t // page], :, t % page] = v[b, :, r].double()
        if q is not None:
            q_new[b, :, :n] = turn(q[b, :, :n])
    return k_new, v_new, q_new


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("B,rows,heads,kv_heads,dh,page,rotated,interleaved,starts", [
    (3, 1, 8, 2, 128, 16, 128, False, [0, 900, 16]),       # a decode step
    (2, 37, 4, 4, 64, 16, 64, True, [5, 0]),
    (2, 70, 10, 5, 64, 24, 32, False, [100000, 3]),        # half of the head, far away
    (2, 9, 3, 1, 64, 7, 20, False, [1, 2]),                # pairs that fit no vector
    (2, 9, 3, 1, 64, 7, 20, True, [1, 2]),
    (1, 5, 2, 1, 8, 3, 8, False, [4]),
    (1, 5, 2, 1, 8, 3, 2, True, [4]),
    (2, 6, 0, 3, 96, 10, 0, False, [0, 8]),                # no queries, no rotation
    (2, 6, 6, 3, 256, 10, 96, False, [0, 8]),
    (3, 1, 4, 2, 64, 1, 64, False, [2, -1, 0]),            # a row without a sequence
])
def test_append_against_64_bits(B, rows, heads, kv_heads, dh, page, rotated, interleaved, starts, dtype):
    g = torch.Generator().manual_seed(rows + dh)
    counts = [rows if rows == 1 else max(0, rows - 3 * b) for b in range(B)]
    lengths = [max(0, s) + rows for s in starts]
    k_pages, v_pages, table = pr.pool(lengths, page, kv_heads, dh, dtype, rows)
    k, v = (torch.randn(B, kv_heads, rows, dh, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(B, heads, rows, dh, generator=g).to(dtype) if heads else None
    q_out = torch.full_like(q, 3.0) if heads else None
    inv_freq = 100.0 ** (-torch.arange(rotated // 2) / max(1, rotated // 2)) if rotated else None
    with_counts = None if rows == 1 else torch.tensor(counts)
    want = expected_append(k, v, k_pages, v_pages, table, starts, with_counts, q, q_out, inv_freq, interleaved)
    d = dev(k, v, k_pages, v_pages, table)
    got_q = paged_append(*d, numbers(starts), None if rows == 1 else numbers(counts), *dev(q, q_out, inv_freq), interleaved)
    _native.poll_status(DEV)
    # one rounding of a rotation evaluated in fp32: cosine and sine off by 2^-23 each, two products and a sum by 2^-24, of normal
    # numbers below 8 (an absolute bound: the terms may cancel)
    most = 8.0
    step = torch.finfo(dtype).eps / 2
    for got, ref in ((d[2], want[0]), (got_q, want[2])):
        if ref is not None:
            off = (got.double().cpu() - ref).abs()
            assert (off <= step * ref.abs() + most * (2 * 2.0 ** -23 + 4 * 2.0 ** -24)).all(), off.max()
    assert torch.equal(d[3].double().cpu(), want[1])
    if not rotated:
        assert torch.equal(d[2].double().cpu(), want[0])


@pytest.mark.parametrize("dtype", [BF, FF])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_takes_any_strides_and_turns_in_place(interleaved, dtype):
    """Views of one projection's output, at odd addresses too: the same bits as from contiguous copies."""
    B, R, H, KV, dh, page = 2, 11, 4, 2, 64, 16
    g = torch.Generator().manual_seed(1)
    for shift in (0, 3):
        rows = torch.randn(B, R, (H + 2 * KV) * dh + 8, generator=g).to(dtype).to(DEV)[..., shift:shift + (H + 2 * KV) * dh]
        qkv = rows.unflatten(-1, (-1, dh)).permute(0, 2, 1, 3)
        q, k, v = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
        inv_freq = (10.0 ** -torch.linspace(0, 4, dh // 2)).to(DEV)
        k_pages, v_pages, table = dev(*pr.pool([40, 40], page, KV, dh, dtype, 3))
        k_same, v_same = k_pages.clone(), v_pages.clone()
        start = numbers([20, 7])
        want = paged_append(k.contiguous(), v.contiguous(), k_same, v_same, table, start, q=q.contiguous(), inv_freq=inv_freq,
                            interleaved=interleaved)
        got = paged_append(k, v, k_pages, v_pages, table, start, q=q, q_out=q, inv_freq=inv_freq, interleaved=interleaved)
        assert got.data_ptr() == q.data_ptr()
        assert torch.equal(got, want) and torch.equal(k_pages, k_same) and torch.equal(v_pages, v_same)


def test_append_far_positions():
    """The angle of a far token: in fp32 it would be off by more than a turn's hundredth."""
    dh, t = 64, 2_000_000_000
    inv_freq = torch.tensor([1.0, 0.3, 1e-3] + [0.0] * 29)
    k = torch.randn(1, 1, 1, dh, generator=torch.Generator().manual_seed(0))
    k_pages, v_pages = torch.zeros(1, 1, 64, dh, device=DEV), torch.zeros(1, 1, 64, dh, device=DEV)
    table = torch.full((1, t // 64 + 1), -1, dtype=torch.int32, device=DEV)
    table[0, t // 64] = 0
    q = paged_append(*dev(k, k), k_pages, v_pages, table, numbers([t]), q=k.to(DEV), inv_freq=inv_freq.to(DEV))
    want = pr.rotated(k[0], torch.tensor([t]), inv_freq, False)
    assert ((q[0].double().cpu() - want).abs() <= 4 * 8 * 2.0 ** -23).all()
    assert torch.equal(k_pages[0, 0, t % 64], q[0, 0, 0])


def test_append_places_that_are_none():
    """Tokens without a place are not stored, their queries are NaN, and it is reported; the others are stored."""
    B, R, KV, dh, page = 4, 10, 2, 64, 4
    g = torch.Generator().manual_seed(2)
    k, v, q = (torch.randn(B, KV, R, dh, generator=g).to(BF) for _ in range(3))
    k_pages, v_pages, table = pr.pool([12] * B, page, KV, dh, BF, 5)
    cases = [("page", [0] * 4, None), ("end", [0, 5, 0, 0], None), ("start", [0, -2, 0, 0], None), ("count", [0] * 4, [10, 11, 10, 10]),
             ("count", [0] * 4, [10, -1, 10, 10])]
    for kind, start, counts in cases:
        tab = table.clone()
        if kind == "page":
            tab[1, 1] = k_pages.shape[0]
        d = dev(k, v, k_pages, v_pages, tab)
        got_q = paged_append(*d, numbers(start), None if counts is None else numbers(counts), q.to(DEV))
        reported()
        lost = {"page": range(4, 8), "end": range(7, 10), "start": range(10), "count": range(10)}[kind]
        kept_start = [0 if s < 0 else s for s in start]
        want_k, want_v, _ = expected_append(k, v, k_pages, v_pages, table, kept_start, [10] * 4 if kind != "end" else [10, 7, 10, 10],
                                            None, None, None, False)
        for r in lost:
            t = kept_start[1] + r
            if t < 12:
                want_k[table[1, t // page], :, t % page] = k_pages[table[1, t // page], :, t % page].double()
                want_v[table[1, t // page], :, t % page] = v_pages[table[1, t // page], :, t % page].double()
        assert torch.equal(d[2].double().cpu(), want_k) and torch.equal(d[3].double().cpu(), want_v), kind
        nan = torch.zeros(B, R, dtype=torch.bool)
        nan[1, list(lost)] = True
        assert torch.equal(torch.isnan(got_q).all(-1).all(1).cpu(), nan), kind


# ---- both together, and what a caller may do ------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF, FF])
def test_cache_decodes_like_one_pass(dtype):
    """A ragged batch: prompts, then tokens one by one with rotation, against attention over everything that was appended."""
    H, KV, dh, page, w, n_p, steps = 6, 2, 64, 8, 20, 3, 6
    prompts = [0, 13, 30]
    B, g = 3, torch.Generator().manual_seed(6)
    table = torch.randperm(3 * 6, generator=g).view(3, 6).to(torch.int32)
    inv_freq = 100.0 ** (-torch.arange(dh // 2) / (dh // 2))
    cache = PagedCache(table.to(DEV), 18, page, KV, dh, w, n_p, dtype, inv_freq=inv_freq.to(DEV))
    pers = [torch.randn(KV, n_p, dh, generator=g).to(dtype) for _ in range(2)]
    cache.set_persistent(*dev(*pers))
    k, v = (torch.randn(B, KV, 36, dh, generator=g).to(dtype) for _ in range(2))
    cache.fill(k[:, :, :30].to(DEV), v[:, :, :30].to(DEV), counts=numbers(prompts))
    for step in range(steps):
        pos = torch.tensor([-1 if step < 2 else step - 2, 13 + step, 30 + step])
        q = torch.randn(B, H, dh, generator=g).to(dtype)
        new = [torch.stack([x[b, :, max(0, int(pos[b]))] for b in range(B)]) for x in (k, v)]
        at = pos.to(torch.int32).to(DEV)
        got = cache.decode(*dev(q, *new), at)
        # (queries and keys as the cache rounded them: test_append_against_64_bits holds those against the formula)
        turned = cache.append(*[x.to(DEV)[:, :, None] for x in new], at, q=q.to(DEV)[:, :, None],
                              q_out=torch.zeros(B, H, 1, dh, dtype=dtype, device=DEV))[:, :, 0]
        check(got, *pr.attention(turned.cpu(), cache.k_pages.cpu(), cache.v_pages.cpu(), table, pos, w, *pers))
    _native.poll_status(DEV)


def test_model_decodes_from_pages():
    """TitanMAC.prefill and decode_step with paged caches give what they give with rings, and sequences of their own lengths."""
    cfg = TitanMACConfig(vocab_size=64, d_model=128, n_heads=2, n_layers=2, d_ff=256, max_seq_len=128, window_size=24, n_persistent=4,
                         use_block_sparse=False)
    torch.manual_seed(0)
    model = TitanMAC(cfg).to(DEV).eval()  # fp32
    ids = torch.randint(0, 64, (2, 40), device=DEV)
    table = torch.randperm(2 * 8).view(2, 8).to(torch.int32).to(DEV)
    with torch.no_grad():
        want, rings = model.prefill(ids)
        paged = model.new_paged_caches(table, pages=16, page_size=16, dtype=FF)
        got, _ = model.prefill(ids, paged)
        assert torch.equal(got, want)
        token = want.argmax(-1)
        for i in range(30):
            pos = torch.full((2,), 40 + i, dtype=torch.int32, device=DEV)
            want, got = model.decode_step(token, pos, rings), model.decode_step(token, pos, paged)
            assert (got - want).abs().max() <= 2e-5 * (1 + want.abs().max())
            token = want.argmax(-1)
        # a row without a sequence does not disturb the other
        alone = model.decode_step(token, torch.tensor([70, -1], dtype=torch.int32, device=DEV), paged)
        both = model.decode_step(token, torch.tensor([70, 70], dtype=torch.int32, device=DEV), paged)
        assert torch.equal(alone[0], both[0])
    _native.poll_status(DEV)


@pytest.mark.parametrize("dtype", [FF, BF])
def test_serving_loop_says_what_the_whole_sequence_says(dtype):
    """Prompt into pages, then token by token: append, attend, logits, log-probabilities with alternatives - against
    TitanMAC.token_logprobs of the finished sequences."""
    cfg = TitanMACConfig(vocab_size=96, d_model=128, n_heads=2, n_layers=2, d_ff=256, max_seq_len=64, window_size=16, n_persistent=3,
                         use_block_sparse=False)
    torch.manual_seed(2)
    model = TitanMAC(cfg).to(device=DEV, dtype=dtype).eval()
    B, T, new = 3, 21, 12
    ids = torch.randint(0, 96, (B, T), device=DEV)
    table = torch.randperm(B * 5, device=DEV).view(B, 5).to(torch.int32)
    with torch.no_grad():
        logits, caches = model.prefill(ids, model.new_paged_caches(table, B * 5, 7, dtype))
        said, entropies = [], []
        for i in range(new):
            token = logits.argmax(-1)
            out = token_logprobs(logits, token, n_top=4)
            assert torch.equal(out.top_ids[:, 0], token) and torch.equal(out.top_logprobs[:, 0], out.logprobs)
            said.append(out.logprobs), entropies.append(out.entropy)
            ids = torch.cat((ids, token[:, None]), 1)
            logits = model.decode_step(token, torch.full((B,), T + i, dtype=torch.int32, device=DEV), caches)
        whole = model.token_logprobs(ids)
    _native.poll_status(DEV)
    # fp32: sums of some hundred terms in another order, twice over.  bf16: some 24 roundings of half a step on a token's way
    # through two layers, of logits below 2, and as many again on the other side
    most = 2e-5 if dtype == FF else 2 * 24 * 2.0 ** -8 * 2.0
    for got, want in ((said, whole.logprobs), (entropies, whole.entropy)):
        assert (torch.stack(got, 1) - want[:, T - 1:T - 1 + new]).abs().max() <= most


def test_filling_in_pieces():
    """A prompt in two pieces at any place is the prompt at once."""
    k, v = (torch.randn(2, 2, 50, 64, device=DEV).to(BF) for _ in range(2))
    table = torch.randperm(8, device=DEV).view(2, 4).to(torch.int32)
    caches = [PagedCache(table, 8, 13, 2, 64, None, 0, BF, inv_freq=(10.0 ** -torch.linspace(0, 4, 32)).to(DEV)) for _ in range(2)]
    caches[0].fill(k, v)
    caches[1].fill(k[:, :, 29:], v[:, :, 29:], t0=29)
    caches[1].fill(k[:, :, :29], v[:, :, :29])
    assert torch.equal(caches[0].k_pages, caches[1].k_pages) and torch.equal(caches[0].v_pages, caches[1].v_pages)
    with pytest.raises(ValueError):
        caches[0].fill(k, v, t0=-1)


def test_two_captured_steps_replay_together():
    """Two graphs over one pool, replayed on two streams at once with new positions, tables and tokens."""
    H, KV, dh, page = 8, 2, 128, 16
    g = torch.Generator().manual_seed(4)
    table = torch.arange(64, dtype=torch.int32).view(2, 32).flip(1).contiguous().to(DEV)
    cache = PagedCache(table, 64, page, KV, dh, None, 0, BF)
    k, v = (torch.randn(2, KV, 512, dh, generator=g).to(BF).to(DEV) for _ in range(2))
    cache.fill(k[:, :, :500], v[:, :, :500])
    q = torch.randn(2, H, dh, generator=g).to(BF).to(DEV)
    caches, inputs, graphs, streams = [], [], [], [torch.cuda.Stream(DEV) for _ in range(2)]
    for b in range(2):
        one = PagedCache(table[b:b + 1], 0, page, KV, dh, None, 0, BF)
        one.k_pages, one.v_pages = cache.k_pages, cache.v_pages
        held = [q[b:b + 1].clone(), k[b:b + 1, :, 500].clone(), v[b:b + 1, :, 500].clone(), numbers([500])]
        one.decode(*held)
        torch.cuda.synchronize(DEV)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = one.decode(*held)
        caches.append(one), inputs.append((held, out)), graphs.append(graph)
    for t in (500, 501, 502, 510):
        torch.cuda.synchronize(DEV)
        for b in range(2):
            held, _ = inputs[b]
            held[1].copy_(k[b:b + 1, :, t]), held[2].copy_(v[b:b + 1, :, t]), held[3].fill_(t)
        torch.cuda.synchronize(DEV)
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize(DEV)
        for b in range(2):
            want, bound = pr.attention(q[b:b + 1].cpu(), cache.k_pages.cpu(), cache.v_pages.cpu(), table[b:b + 1].cpu(), torch.tensor([t]))
            check(inputs[b][1], want, bound)


def test_refusals():
    k_pages, v_pages, table = dev(*pr.pool([20, 20], 16, 2, 64, BF, 0))
    q, pos = torch.zeros(2, 4, 64, dtype=BF, device=DEV), numbers([0, 0])
    ok = (q, k_pages, v_pages, table, pos)

    def refused(error, i, value, **kw):
        args = list(ok)
        args[i] = value
        with pytest.raises(error):
            paged_attention(*args, **kw)

    refused(RuntimeError, 0, q.cpu())
    refused(TypeError, 0, q.half())
    refused(ValueError, 0, q[:, :3])
    refused(ValueError, 0, q[..., :32])
    refused(ValueError, 0, q[0])
    refused(ValueError, 0, q.transpose(1, 2).contiguous().transpose(1, 2))
    refused(TypeError, 2, v_pages.float())
    refused(ValueError, 2, v_pages[:1])
    refused(ValueError, 1, k_pages.transpose(1, 2))
    refused(TypeError, 3, table.long())
    refused(ValueError, 3, table[:1])
    refused(TypeError, 4, pos.long())
    refused(ValueError, 4, pos[:1])
    refused(ValueError, 0, q, window=-1)
    refused(ValueError, 0, q, k_pers=k_pages[0])
    refused(ValueError, 0, q, k_pers=k_pages[0, :1], v_pers=k_pages[0, :1])
    refused(_native.TmwError, 0, q, scale=-1.0)
    refused(ValueError, 0, q, out=q)
    with pytest.raises(_native.TmwError):  # head_dim 12
        paged_attention(q[..., :12].contiguous(), k_pages[..., :12].contiguous(), v_pages[..., :12].contiguous(), table, pos)
    k = torch.zeros(2, 2, 3, 64, dtype=BF, device=DEV)
    good = dict(k=k, v=k, k_pages=k_pages, v_pages=v_pages, page_table=table, start=pos)
    for error, change in [(ValueError, dict(k=k[0])), (ValueError, dict(v=k[:, :, :2])), (TypeError, dict(k=k.float())),
                          (TypeError, dict(start=pos.long())), (TypeError, dict(counts=pos.long())), (ValueError, dict(q_out=k)),
                          (ValueError, dict(q=k, q_out=k[:, :1])), (TypeError, dict(inv_freq=torch.zeros(2, dtype=BF, device=DEV))),
                          (ValueError, dict(inv_freq=torch.zeros(33, device=DEV))), (RuntimeError, dict(counts=pos.cpu()))]:
        with pytest.raises(error):
            paged_append(**{**good, **change})
    with pytest.raises(ValueError):
        PagedCache(table, 4, 0, 2, 64, None, 0, BF)
    with pytest.raises(TypeError):
        PagedCache(table, 4, 16, 2, 64, None, 0, torch.float64)
    # nothing to do is fine
    assert paged_append(k[:0], k[:0], k_pages, v_pages, table[:0], pos[:0]) is None
    assert paged_append(k[:, :, :0], k[:, :, :0], k_pages, v_pages, table, pos) is None
    assert paged_attention(q[:0], k_pages, v_pages, table[:0], pos[:0]).shape == (0, 4, 64)
    none = paged_attention(q, k_pages[:0], v_pages[:0], table[:, :0], numbers([-1, -1]))
    assert (none == 0).all()
    _native.poll_status(DEV)
