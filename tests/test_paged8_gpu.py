"""Pages in 8 bits against plain forms in 64 bits: what is written, what is read back, what one token attends to."""

import math

import pytest
import torch

import paged_drafts_reference as dr
import paged_reference as pr
from titanmac_b200 import PagedCache, _native, paged_append, paged_attention, paged_read

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32
I8, E4 = torch.int8, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _fresh_status():
    _native.poll_status(DEV)
    yield


def dev(*ts):
    return [None if t is None else tuple(x.to(DEV) for x in t) if isinstance(t, tuple) else t.to(DEV) for t in ts]


def numbers(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def reported():
    with pytest.raises(_native.TmwError):
        _native.poll_status(DEV)


def check(got, want, bound):
    step = torch.finfo(got.dtype).eps / 2 if got.dtype != FF else 0.0  # one rounding of the output
    off = (got.double().cpu() - want).abs()
    allowed = bound + step * (want.abs() + bound) + torch.finfo(got.dtype).tiny
    # what lies half a step beyond the type's largest number, or may within the bound, rounds to infinity: 65520 = 65504 + 16 in fp16
    largest = torch.finfo(got.dtype).max
    beyond = (want.abs() + bound >= largest * (1 + torch.finfo(got.dtype).eps / 4)) & (got.double().cpu() == want.sign() * math.inf)
    assert ((off <= allowed) | beyond).all(), (off / allowed).max().item()


# ---- attention of one token -------------------------------------------------------------------------------------------


def attend(lengths, heads, kv_heads, dh, page, dtype, form, window=None, n_p=0, seed=0, scale=0.0, spread=0.3):
    g = torch.Generator().manual_seed(seed + 1)
    k, v, table, scales = dr.pool8(lengths, page, kv_heads, dh, form, seed, spread)
    q = torch.randn(len(lengths), heads, dh, generator=g).to(dtype)
    pers, pers_scales = (None, None), None
    if n_p:
        (kp, ks), (vp, vs) = (dr.coded(torch.randn(kv_heads, n_p, dh, generator=g), form) for _ in range(2))
        pers, pers_scales = (kp, vp), (ks, vs)
    pos = torch.tensor(lengths) - 1
    got = paged_attention(*dev(q, k, v, table), pos.to(torch.int32).to(DEV), window, *dev(*pers), scale=scale, scales=dev(scales)[0],
                          pers_scales=dev(pers_scales)[0])
    _native.poll_status(DEV)
    return got, *dr.one_token(q, k, v, table, pos, window, *pers, scale, scales, pers_scales or (None, None))


@pytest.mark.parametrize("form", [I8, E4])
@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("lengths,heads,kv_heads,dh,page,window,n_p", [
    ([1], 1, 1, 64, 16, None, 0),
    ([1, 2, 15, 16, 17, 31, 33, 64], 4, 4, 64, 16, None, 0),  # tiles that end everywhere
    ([300], 10, 10, 64, 64, None, 16),                   # one sequence over many CTAs
    ([40, 1, 700, 0, 3], 8, 2, 128, 24, None, 3),        # ragged, a sequence without tokens, pages that end inside tiles
    ([513, 77, 0], 4, 2, 64, 7, 100, 5),                 # a window that begins inside a tile and a page
    ([50, 9], 2, 1, 64, 1, 0, 0),                        # the token itself alone, pages of one token
    ([129, 16], 16, 1, 128, 32, None, 0),                # sixteen heads on one
    ([65, 200], 14, 2, 96, 20, 150, 2),                  # seven heads on one
    ([90, 33], 40, 2, 32, 64, None, 1),                  # twenty heads on one
    ([150, 20], 6, 2, 256, 16, None, 17),                # wide heads
    ([70, 41], 18, 1, 256, 16, None, 0),
    ([70, 5], 3, 1, 16, 5, None, 0),
    ([45, 100], 8, 2, 80, 16, None, 3),                  # head sizes of no tile
    ([45, 100], 3, 1, 192, 32, None, 0),
    ([70, 45], 2, 2, 144, 16, None, 1),
])
def test_attention_against_64_bits(lengths, heads, kv_heads, dh, page, window, n_p, dtype, form):
    check(*attend(lengths, heads, kv_heads, dh, page, dtype, form, window, n_p, seed=len(lengths) * dh + page))


@pytest.mark.parametrize("form", [I8, E4])
@pytest.mark.parametrize("dtype", [BF, FF])
def test_attention_of_many_short_sequences(dtype, form):
    check(*attend([(7 * b) % 40 for b in range(333)], 4, 2, 64, 16, dtype, form, seed=5))


@pytest.mark.parametrize("dtype", [BF, HF, FF])
def test_scales_of_every_size(dtype):
    """Scales of the tokens that differ by factors of 10^9: small ones of likely tokens count as much as large ones."""
    check(*attend([90, 33], 8, 4, 64, 16, dtype, I8, seed=3, spread=5.0, scale=2.0 ** -12))


@pytest.mark.parametrize("form", [I8, E4])
@pytest.mark.parametrize("dtype", [BF, FF])
def test_value_scales_of_every_size(dtype, form):
    """Values' scales that differ by factors of 10^12 and more, keys' that do not: a token's weight does not depend on its value's."""
    k, v, table, scales = dr.pool8([90, 33], 16, 4, 64, form, 3)
    g = torch.Generator().manual_seed(4)
    scales = (scales[0], scales[1] * 2.0 ** torch.randint(-40, 41, scales[1].shape, generator=g))
    q = torch.randn(2, 8, 64, generator=g).to(dtype)
    got = paged_attention(*dev(q, k, v, table), numbers([89, 32]), scales=dev(scales)[0])
    check(got, *dr.one_token(q, k, v, table, torch.tensor([89, 32]), scales=scales))
    # small values alone: every token of head 0 has a scale of 2^-60, of head 1 of 2^60
    scales[1][:, 0] = 2.0 ** -60
    scales[1][:, 1] = 2.0 ** 60
    got = paged_attention(*dev(q, k, v, table), numbers([89, 32]), scales=dev(scales)[0])
    check(got, *dr.one_token(q, k, v, table, torch.tensor([89, 32]), scales=scales))


@pytest.mark.parametrize("dtype", [BF, FF])
def test_queries_of_every_size(dtype):
    """Numbers of one query that differ by 2^60; other heads' are large or small as a whole."""
    k, v, table, scales = dr.pool8([77], 16, 2, 64, I8, 4)
    q = torch.randn(1, 4, 64, generator=torch.Generator().manual_seed(1))
    q[0, 0, ::3] *= 2.0 ** -40
    q[0, 1] *= 2.0 ** 14
    q[0, 2] *= 2.0 ** -30
    q[0, 3] = 0.0
    q = q.to(dtype)
    got = paged_attention(*dev(q, k, v, table), numbers([76]), scale=2.0 ** -14, scales=dev(scales)[0])
    check(got, *dr.one_token(q, k, v, table, torch.tensor([76]), scale=2.0 ** -14, scales=scales))


@pytest.mark.parametrize("dtype,dh", [(BF, 128), (HF, 64), (FF, 64), (BF, 80)])
def test_a_row_of_nan_reaches_its_own_head_alone(dtype, dh):
    k, v, table, scales = dr.pool8([60, 60], 16, 3, dh, E4, 9)
    q = torch.randn(2, 6, dh, generator=torch.Generator().manual_seed(2)).to(dtype)
    at = int(table[0, 1])
    scales[0][at, 1, 3] = math.nan  # a key of head 1
    scales[1][at, 2, 3] = math.nan  # a value of head 2
    got = paged_attention(*dev(q, k, v, table), numbers([59, 59]), scales=dev(scales)[0])
    assert torch.isnan(got[0, 2:]).all() and torch.isfinite(got[0, :2]).all() and torch.isfinite(got[1]).all()


@pytest.mark.parametrize("dtype,dh", [(BF, 64), (FF, 96)])
def test_what_has_no_page(dtype, dh):
    k, v, table, scales = dr.pool8([60, 40, 10], 16, 2, dh, I8, 9)
    q = torch.randn(3, 4, dh, generator=torch.Generator().manual_seed(2)).to(dtype)
    want, bound = dr.one_token(q, k, v, table, torch.tensor([59, 39, 9]), scales=scales)
    table[0, 1] = 1000
    got = paged_attention(*dev(q, k, v, table), numbers([59, 39, 4000]), scales=dev(scales)[0])
    reported()
    assert torch.isnan(got[0]).all() and torch.isnan(got[2]).all()
    check(got[1:2], want[1:2], bound[1:2])


def test_outputs_and_queries_with_strides():
    k, v, table, scales = dr.pool8([60, 40], 16, 2, 64, I8, 1)
    wide = torch.randn(2, 4, 131, generator=torch.Generator().manual_seed(2)).to(BF)
    q = wide[:, :, 3:67]
    out = torch.zeros(2, 4, 99, dtype=BF, device=DEV)
    back = paged_attention(wide.to(DEV)[:, :, 3:67], *dev(k, v, table), numbers([59, 39]), scales=dev(scales)[0], out=out[:, :, 1:65])
    check(back, *dr.one_token(q, k, v, table, torch.tensor([59, 39]), scales=scales))
    assert (out[:, :, 0] == 0).all() and (out[:, :, 65:] == 0).all()


# ---- writing and reading back ---------------------------------------------------------------------------------------------


def empty_pool(start, counts, page, kv_heads, dh, form, seed):
    k, v, table = pr.pool([s + c for s, c in zip(start, counts)], page, kv_heads, dh, torch.float32, seed)
    (k, ks), (v, vs) = dr.coded(k, form), dr.coded(v, form)
    return k, v, table, (ks, vs)


@pytest.mark.parametrize("form", [I8, E4])
@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("kv_heads,dh,page,rows,start,counts,heads", [
    (2, 64, 16, 1, [0, 5, 99], [1, 1, 1], 4), (3, 128, 24, 19, [0, 17], [19, 3], 3), (1, 96, 7, 40, [3], [33], 0), (2, 16, 16, 5, [0, 1], [0, 5], 2),
    (1, 256, 64, 9, [60], [9], 1), (5, 48, 3, 6, [1, 2, 3], [6, 2, 1], 5)])
def test_append_writes_the_nearest_codes(kv_heads, dh, page, rows, start, counts, heads, dtype, form):
    """Without a rotation nothing is rounded before the codes: they and the scales are the definition's, bit for bit."""
    g = torch.Generator().manual_seed(dh + rows)
    k_pages, v_pages, table, scales = empty_pool(start, counts, page, kv_heads, dh, form, dh)
    k, v = (torch.randn(len(start), kv_heads, rows, dh, generator=g).to(dtype) for _ in range(2))
    k[0, 0, 0, 1] = -0.5 * k[0, 0, 0].abs().max()  # on a border of int8
    q = torch.randn(len(start), max(heads, 1), rows, dh, generator=g).to(dtype)
    d = dev(k_pages, v_pages, scales)
    out = paged_append(*dev(k, v), *d[:2], table.to(DEV), numbers(start), numbers(counts), q=q.to(DEV) if heads else None, scales=d[2])
    _native.poll_status(DEV)
    want = [t.clone() for t in (k_pages.float(), v_pages.float(), *scales)]
    for b, (s, c) in enumerate(zip(start, counts)):
        for i, (x, pages, scale) in enumerate(((k, want[0], want[2]), (v, want[1], want[3]))):
            codes, sizes = dr.coded(x[b], form)
            for r in range(c):
                at, slot = int(table[b, (s + r) // page]), (s + r) % page
                pages[at, :, slot], scale[at, :, slot] = codes[:, r].float(), sizes[:, r]
    for got, x in zip((d[0].float(), d[1].float(), *d[2]), want):
        assert torch.equal(got.cpu(), x)
    if heads:
        for b, c in enumerate(counts):
            assert torch.equal(out[b, :, :c].cpu(), q[b, :, :c])


@pytest.mark.parametrize("form", [I8, E4])
@pytest.mark.parametrize("dtype", [BF, FF])
@pytest.mark.parametrize("dh,rotated,interleaved,shift,by_row", [
    (64, 64, False, 0, False), (64, 32, True, 0, True), (128, 128, False, 0, True), (96, 20, False, 0, False), (96, 22, True, 0, False),
    (64, 64, False, 1, False), (64, 64, True, 3, True), (256, 128, False, 0, False)])
def test_append_rotates_before_it_rounds(dh, rotated, interleaved, shift, by_row, dtype, form):
    """A rotated number in fp32 is off by 8 units of 2^-24 of its pair (two products, a sum, and the sine and cosine's), the scale
    by as much of itself; a code by half a step of its own besides."""
    B, kv_heads, heads, rows, page = 2, 2, 3, 13, 5
    g = torch.Generator().manual_seed(dh)
    start, counts = [7, 100000], [13, 9]
    k_pages, v_pages = (torch.zeros(64, kv_heads, page, dh).to(form) for _ in range(2))
    table = torch.full((B, 20100), -1, dtype=torch.int32)
    for b, (s, c) in enumerate(zip(start, counts)):
        for n, col in enumerate(range(s // page, (s + c - 1) // page + 1)):
            table[b, col] = b * 32 + n
    scales = tuple(torch.zeros(64, kv_heads, page) for _ in range(2))
    wide = torch.randn(B, kv_heads * 2 + heads, rows, dh + shift, generator=g).to(dtype)
    inv_freq = (10000.0 ** (-torch.arange(rotated // 2) / (rotated // 2))).float()
    positions = torch.randint(0, 200000, (B, rows), generator=g, dtype=torch.int32) if by_row else None
    d = dev(k_pages, v_pages, scales, wide)
    x = d[3][..., shift:]
    q = paged_append(x[:, :kv_heads], x[:, kv_heads:2 * kv_heads], *d[:2], table.to(DEV), numbers(start), numbers(counts), q=x[:, 2 * kv_heads:],
                     inv_freq=inv_freq.to(DEV), interleaved=interleaved, scales=d[2], positions=None if positions is None else positions.to(DEV))
    _native.poll_status(DEV)
    x = wide[..., shift:]
    u = 2.0 ** -24
    for b, (s, c) in enumerate(zip(start, counts)):
        at = positions[b, :c] if by_row else torch.arange(s, s + c)
        k = pr.rotated(x[b, :kv_heads, :c], at, inv_freq, interleaved)
        size = x[b, :kv_heads, :c].double().abs().amax(-1, keepdim=True) * math.sqrt(2)
        off = 8 * u * size
        for r in range(c):
            page_at, slot = int(table[b, (s + r) // page]), (s + r) % page
            scale = d[2][0][page_at, :, slot].cpu().double()[:, None]
            assert ((scale * dr.LARGEST[form] - k[:, r].abs().amax(-1, keepdim=True)).abs() <= off[:, r] + 4 * u * scale * dr.LARGEST[form]).all()
            got = d[0][page_at, :, slot].float().cpu().double() * scale
            t = (k[:, r] / scale).abs()
            half = 0.5 if form is I8 else 2.0 ** (torch.floor(torch.log2(t.clamp(min=2.0 ** -6))) - 4)
            assert ((got - k[:, r]).abs() <= half * scale * (1 + 2.0 ** -20) + 2 * off[:, r]).all()
        want = pr.rotated(x[b, 2 * kv_heads:, :c], at, inv_freq, interleaved)
        size = x[b, 2 * kv_heads:, :c].double().abs().amax(-1, keepdim=True) * math.sqrt(2)
        step = torch.finfo(dtype).eps / 2 if dtype != FF else 0.0
        assert ((q[b, :, :c].double().cpu() - want).abs() <= 8 * u * size + step * (want.abs() + 8 * u * size)).all()


@pytest.mark.parametrize("form", [I8, E4])
def test_append_of_rows_that_are_special(form):
    """Zeros, subnormal numbers, the largest ones, infinities and NaN."""
    k = torch.randn(1, 1, 6, 32, generator=torch.Generator().manual_seed(0))
    k[0, 0, 0] = 0.0
    k[0, 0, 1] *= 1e-40
    k[0, 0, 2] *= 3e38 / k[0, 0, 2].abs().max()
    k[0, 0, 3, 5] = math.inf
    k[0, 0, 4, 31] = math.nan
    pages = [torch.ones(1, 1, 16, 32).to(form).to(DEV) for _ in range(2)]
    scales = tuple(torch.ones(1, 1, 16, device=DEV) for _ in range(2))
    paged_append(k.to(DEV), k.to(DEV), *pages, numbers([[0]]), numbers([0]), scales=scales)
    codes, sizes = dr.coded(k[0, 0], form)
    for p, s in zip(pages, scales):
        assert torch.equal(p[0, 0, :6].float().cpu(), codes.float())
        assert torch.equal(torch.nan_to_num(s[0, 0, :6], nan=-1.0).cpu(), torch.nan_to_num(sizes, nan=-1.0))
    back, _ = paged_read(*pages, numbers([[0]]), numbers([0]), 6, dtype=FF, scales=scales)
    assert torch.isnan(back[0, 0, 3:5]).all() and (back[0, 0, 0] == 0).all() and torch.isfinite(back[0, 0, 2]).all()


@pytest.mark.parametrize("dtype,form", [(BF, I8), (HF, E4), (FF, I8), (FF, E4), (BF, None), (FF, None)])
@pytest.mark.parametrize("dh,page,rows,start,counts", [(64, 16, 7, [0, 40, -1], [7, 2, 7]), (16, 5, 33, [3, 0], [33, 0]), (256, 64, 20, [50], [20]),
                                                       (8, 3, 4, [2], [4])])
def test_read_gives_what_is_meant(dh, page, rows, start, counts, dtype, form):
    if form is not None and dh % 16:
        pytest.skip("no such pages")
    lengths = [max(s, 0) + c for s, c in zip(start, counts)]
    if form is None:
        k, v, table = pr.pool(lengths, page, 3, dh, dtype, 2)
        scales = None
    else:
        k, v, table, scales = dr.pool8(lengths, page, 3, dh, form, 2)
    for shift in (0, 1):  # outputs at any address too
        out = [torch.full((len(start), rows, 3, dh + shift), 7.0, dtype=dtype, device=DEV).permute(0, 2, 1, 3)[..., shift:] for _ in range(2)]
        got = paged_read(*dev(k, v, table), numbers(start), counts=numbers(counts), scales=dev(scales)[0], k_out=out[0], v_out=out[1])
        _native.poll_status(DEV)
        for t, pages, scale in zip(got, (k, v), scales or (None, None)):
            for b, (s, c) in enumerate(zip(start, counts)):
                c = 0 if s < 0 else c
                assert (t[b, :, c:] == 7).all()
                for h in range(3):
                    for r in range(c):
                        at, slot = int(table[b, (s + r) // page]), (s + r) % page
                        want = pages[at, h, slot] if scale is None else (pages[at, h, slot].float() * scale[at, h, slot]).to(dtype)
                        assert torch.equal(t[b, h, r].cpu(), want)


def test_read_of_what_has_no_place():
    k, v, table, scales = dr.pool8([20, 20], 16, 1, 32, I8, 2)
    table[0, 1] = 99
    got, _ = paged_read(*dev(k, v, table), numbers([10, 10]), 10, dtype=BF, scales=dev(scales)[0])
    reported()
    assert torch.isnan(got[0, 0, 6:]).all() and torch.isfinite(got[0, 0, :6]).all() and torch.isfinite(got[1]).all()
    got, _ = paged_read(*dev(k, v, table), numbers([-2, 30]), 10, dtype=BF, scales=dev(scales)[0])
    reported()
    assert torch.isnan(got[0]).all() and torch.isnan(got[1, 0, 2:]).all()


@pytest.mark.parametrize("form", [I8, E4])
def test_append_of_what_has_no_place(form):
    """A wrong page, a wrong start and a wrong count: nothing is stored, the queries are NaN, the other sequence is as it would be."""
    start, counts, page = [14, 3, -2, 0, -1], [4, 2, 2, 9, 4], 16
    k_pages, v_pages, table, scales = empty_pool([32] * 5, [0] * 5, page, 1, 32, form, 1)
    table[0, 1] = -5
    x = torch.randn(5, 1, 4, 32, generator=torch.Generator().manual_seed(1)).to(BF)
    d = dev(k_pages, v_pages, scales)
    q_out = torch.full((5, 1, 4, 32), 7.0, dtype=BF, device=DEV)
    paged_append(*dev(x, x), *d[:2], table.to(DEV), numbers(start), numbers(counts), q=x.to(DEV), q_out=q_out, scales=d[2])
    reported()
    assert torch.isnan(q_out[0, 0, 2:]).all() and torch.equal(q_out[0, 0, :2].cpu(), x[0, 0, :2])
    assert torch.isnan(q_out[2, 0, :2]).all() and (q_out[2, 0, 2:] == 7).all() and torch.isnan(q_out[3]).all() and (q_out[4] == 7).all()
    want_k, want_s = k_pages.float().clone(), scales[0].clone()
    for b, r in ((0, 0), (0, 1), (1, 0), (1, 1)):
        codes, size = dr.coded(x[b, :, r], form)
        at, slot = int(table[b, (start[b] + r) // page]), (start[b] + r) % page
        want_k[at, :, slot], want_s[at, :, slot] = codes.float(), size
    assert torch.equal(d[0].float().cpu(), want_k) and torch.equal(d[2][0].cpu(), want_s)


@pytest.mark.parametrize("form", [I8, E4])
@pytest.mark.parametrize("inv", [False, True])
def test_a_cache_in_8_bits_decodes(form, inv):
    """A cache filled with prompts, then token by token, against what its pages stand for."""
    B, H, KV, dh, n_p = 3, 4, 2, 64, 5
    g = torch.Generator().manual_seed(3)
    table = torch.randperm(3 * 8, generator=g, dtype=torch.int64).view(3, 8).to(torch.int32)
    inv_freq = (100.0 ** (-torch.arange(32) / 32)).float().to(DEV) if inv else None
    cache = PagedCache(table.to(DEV), 24, 16, KV, dh, 40, n_p, BF, inv_freq=inv_freq, page_dtype=form)
    kp, vp = (torch.randn(KV, n_p, dh, generator=g).to(BF) for _ in range(2))
    cache.set_persistent(*dev(kp, vp))
    for t, x in zip((*[c.float().cpu() for c in (cache.k_pers, cache.v_pers)], *[c.cpu() for c in cache.pers_scales]),
                    (*(dr.coded(x, form)[0].float() for x in (kp, vp)), *(dr.coded(x, form)[1] for x in (kp, vp)))):
        assert torch.equal(t, x)
    k, v = (torch.randn(B, KV, 60, dh, generator=g).to(BF) for _ in range(2))
    cache.fill(*dev(k, v), counts=numbers([60, 31, 1]))
    pos = [60, 31, 1]
    for step in range(3):
        q, k1, v1 = (torch.randn(B, n, dh, generator=g).to(BF) for n in (H, KV, KV))
        at = [p + step for p in pos[:2]] + [-1 if step == 1 else pos[2] + (step + 1) // 2]
        got = cache.decode(*dev(q, k1, v1), numbers(at))
        turned = torch.zeros_like(q)
        if inv:  # (the queries as the append leaves them are another test's)
            scratch = [torch.zeros(3, KV, 16, dh, dtype=BF, device=DEV) for _ in range(2)]
            turned = paged_append(*dev(k1[:, :, None], v1[:, :, None]), *scratch, numbers([[0] * 10, [1] * 10, [2] * 10]), numbers(at), q=q[:, :, None].to(DEV),
                                  q_out=turned[:, :, None].to(DEV), inv_freq=inv_freq)[:, :, 0].cpu()
        held = [c.cpu() for c in (cache.k_pages, cache.v_pages, cache.k_pers, cache.v_pers)]
        want, bound = dr.one_token(turned if inv else q, held[0], held[1], table, torch.tensor(at), 40, held[2], held[3],
                                   scales=tuple(s.cpu() for s in cache.scales), pers_scales=tuple(s.cpu() for s in cache.pers_scales))
        check(got, want, bound)
    _native.poll_status(DEV)


def test_captured_calls_share_nothing():
    """Two graphs of the same cache's calls, replayed at once on two streams, and an eager call beside them."""
    k, v, table, scales = dr.pool8([700, 90], 16, 2, 64, I8, 5)
    q = torch.randn(2, 6, 64, generator=torch.Generator().manual_seed(5)).to(BF)
    args, sc, pos = dev(q, k, v, table), dev(scales)[0], numbers([699, 89])
    want = paged_attention(*args, pos, scales=sc)
    graphs, outs, streams = [], [], [torch.cuda.Stream(DEV) for _ in range(2)]
    torch.cuda.synchronize(DEV)
    for s in streams:
        with torch.cuda.stream(s):
            paged_attention(*args, pos, scales=sc)
        torch.cuda.synchronize(DEV)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(paged_attention(*args, pos, scales=sc))
        graphs.append(graph)
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        assert torch.equal(paged_attention(*args, pos, scales=sc), want)
    torch.cuda.synchronize(DEV)
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
