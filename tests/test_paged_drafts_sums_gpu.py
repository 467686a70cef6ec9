"""Drafted trees where their sums are delicate: what single numbers of a value do to the rows that see them and to those that do not,
sums over very many keys, values that cancel."""

import math

import pytest
import torch

import paged_drafts_reference as dr
from test_paged_drafts_gpu import BF, DEV, E4, FF, HF, I8, Case, check, dev, numbers
from titanmac_b200 import _native, paged_attention, paged_tree_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _fresh_status():
    _native.poll_status(DEV)
    yield


# ---- codes that are no number ------------------------------------------------------------------------------------------------


def spoil(codes, table, token, at, code):
    """Number ``at`` of a token's row, under every head, becomes a code that is no number."""
    page = codes.shape[2]
    codes.view(torch.uint8)[int(table[0, token // page]), :, token % page, at] = code


# mma.sync with pages by TMA and by copies, tcgen05, CUDA cores; a tree in one tile, across two, with nothing in front of it
@pytest.mark.parametrize("dtype,dh,nodes,heads,page,start", [
    (BF, 64, 40, 2, 16, 70), (HF, 128, 40, 1, 16, 20), (BF, 32, 40, 2, 12, 70), (HF, 96, 40, 4, 16, 3), (BF, 256, 40, 1, 24, 0),
    (BF, 64, 40, 4, 16, 70), (HF, 128, 40, 2, 16, 200), (HF, 64, 40, 6, 32, 0), (BF, 128, 40, 1, 64, 37),
    (BF, 144, 40, 2, 16, 70), (FF, 64, 40, 2, 16, 70)])
def test_codes_that_are_no_number_reach_those_that_see_them(dtype, dh, nodes, heads, page, start):
    """A key of nodes that few see has such a code; single numbers of others' values have; one token in front of the deeper nodes' window
    has: exactly the outputs that the formula makes no number are none, the others are what they would be."""
    window = 30
    case = Case([start], [nodes], nodes, heads, 1, dh, page, dtype, E4, window=window, n_p=3, seed=1)
    parents = [-1] + [0 if i == 20 else i - 1 for i in range(1, nodes)]  # 1 .. 19 and 20 .. 39 are two branches
    seen, depth = dr.ancestors(parents)
    case.seen, case.positions = seen[None], (start + depth)[None].to(torch.int32)
    bound = case.want()[1]
    for node, at, code in ((10, 5, 0x7F), (15, dh - 1, 0xFF), (30, slice(0, None, 2), 0x7F), (39, slice(None), 0xFF)):
        spoil(case.v, case.table, start + node, at, code)
    spoil(case.k, case.table, start + 35, 3, 0x7F)
    if start > window:
        spoil(case.v, case.table, start - window, 1, 0xFF)  # seen by the root alone
    want = case.want()[0]
    nan = torch.isnan(want)
    assert not nan[:, :, 20:30].any() and not nan[:, :, 1:10].any() and nan[:, :, 10:20, 5].all() and nan[:, :, 35:].all()
    assert not nan[:, :, 10:20, 6].any() and nan[:, :, 0].any() == (start > window)
    got = case.run().cpu()
    _native.poll_status(DEV)
    assert torch.equal(torch.isnan(got), nan)
    check(got.masked_fill(nan, 0), want.masked_fill(nan, 0), bound)


# ---- very many keys ----------------------------------------------------------------------------------------------------------


def pages_of(form, dh, values, g):
    """One page of 64 tokens, keys of normal numbers; ``(k, v, scales)`` and what they stand for."""
    k = torch.randn(1, 1, 64, dh, generator=g)
    if form is None:
        k, v = k.to(HF), values.to(HF)
        return (k, v, None), (k.double(), v.double())
    (k, ks), (v, vs) = dr.coded(k, form), dr.coded(values, form)
    if (values == 1).all():
        v, vs = torch.full(v.shape, 64.0).to(form), torch.full_like(vs, 2.0 ** -6)
    return (k, v, (ks, vs)), (dr.meant(k, ks), dr.meant(v, vs))


def long_chains(B, tokens, nodes, dh, held, g):
    """Chains of ``nodes`` behind ``tokens`` that all lie in one page, which the tables name over and over."""
    k, v, scales = held
    table = torch.zeros(B, (tokens + nodes + 63) // 64, dtype=torch.int32, device=DEV)
    q = torch.randn(B, 1, nodes, dh, generator=g).to(HF).to(DEV)
    seen = torch.tensor([[-1 if i == 63 else (2 << i) - 1 for i in range(nodes)]] * B, device=DEV)
    out = paged_tree_attention(q, k.to(DEV), v.to(DEV), table, numbers([tokens] * B), seen, scales=dev(scales)[0])
    _native.poll_status(DEV)
    return q, out


# With as many sequences as SMs one CTA has all the keys of each; with one sequence every CTA has an equal part of it.  (64 tokens to a tile:
# 8202 and 40 are a tile more than 128, 16484 two more than 256.)
MUCH = [("all", 5000), ("all", 8202), ("all", 16484), ("all", 400_000), (1, 2_500_000)]


def batch(B):
    return torch.cuda.get_device_properties(DEV).multi_processor_count if B == "all" else B


@pytest.mark.parametrize("form", [None, I8, E4])
@pytest.mark.parametrize("dh,nodes", [(128, 6), (128, 40), (64, 60)])
@pytest.mark.parametrize("B,tokens", MUCH)
def test_sums_over_very_many_keys_lose_nothing(B, tokens, dh, nodes, form):
    """Values that are all one: an output is one, whatever the weights.  512 products in a row may each cut off 2^-23 of the sum; a row's
    sum of weights is rounded by 2^-24 some 100 times on the way through as many keys, parts are added up at most 200 times; a weight is held
    in 22 bits: 6.1e-5 + 1.8e-5 + 2.4e-7 at the most, less than the half step 2^-12 of fp16 below one."""
    g = torch.Generator().manual_seed(2)
    held, _ = pages_of(form, dh, torch.ones(1, 1, 64, dh), g)
    _, out = long_chains(batch(B), tokens, nodes, dh, held, g)
    assert (out == 1).all(), (out.float() - 1).abs().max().item()


@pytest.mark.parametrize("form", [None, I8, E4])
@pytest.mark.parametrize("dh,nodes", [(128, 40), (64, 60)])
@pytest.mark.parametrize("B,tokens", MUCH[1:3] + MUCH[4:])
def test_outputs_over_very_many_keys(B, tokens, dh, nodes, form):
    """The same with values of normal numbers, against the formula in 64 bits, a page's token counted as often as it is seen.  A sum is off by what
    its weights are, by what the scores are, and by what the test above allows, all of the largest value; then one rounding."""
    g = torch.Generator().manual_seed(3)
    held, (k, v) = pages_of(form, dh, torch.randn(1, 1, 64, dh, generator=g), g)
    B = batch(B)
    q, out = long_chains(B, tokens, nodes, dh, held, g)
    k, v = k[0, 0].to(DEV), v[0, 0].to(DEV)
    s = q[:, 0].double() @ k.T / math.sqrt(dh)  # [B, nodes, 64]
    slot = torch.arange(64, device=DEV)
    times = (tokens // 64 + (slot < tokens % 64)).double()
    node = torch.arange(nodes, device=DEV)
    times = times + ((node[None, :, None] <= node[:, None, None]) & ((tokens + node)[None, :, None] % 64 == slot)).sum(1)  # [nodes, 64]
    w = torch.exp(s - s.amax(-1, keepdim=True)) * times
    want = w @ v / w.sum(-1, keepdim=True)
    u = 2.0 ** -23
    off = (dh + 16) * u * (q[:, 0].double().abs() @ k.abs().T).amax() / math.sqrt(dh) + 2 * u * s.abs().amax()
    bound = 2 * v.abs().amax() * (1.01 * off + 2.0 ** -22 + 6.1e-5 + 1.8e-5)
    step = torch.finfo(HF).eps / 2
    error = (out[:, 0].double() - want).abs() - step * (want.abs() + bound)
    assert (error <= bound).all(), (error / bound).max().item()


# ---- values that cancel ------------------------------------------------------------------------------------------------------


# How much of itself a weight may be off by, besides what the values' product makes of it: its score, a number of a key here, exact but
# for three roundings of at most 2^3 / 2 (the exponent of two), ex2.approx to 2^-22, sums of at most 16 products that may each cut off
# 2^-23 and of 12 roundings; the weight itself as it meets the values, 24 bits in the attention of one token, 16 in a tree over bf16
# pages, 22 over fp16 pages and codes.
SUMS = 3 * 2.0 ** -22 + 2.0 ** -22 + 16 * 2.0 ** -23 + 12 * 2.0 ** -24
TREE = {BF: 2.0 ** -16, HF: 2.0 ** -22, FF: 2.0 ** -23}


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("nodes", [6, 40])
def test_values_that_cancel(nodes, dtype):
    """Four tokens' values leave next to nothing of one another, so an output is what its weights have lost; a chain's last node and the
    attention of one token at its place."""
    g = torch.Generator().manual_seed(nodes)
    start, page, dh, heads = 70, 16, 64, 2
    tokens = start + nodes
    columns = (tokens + page - 1) // page
    k, v = torch.zeros(columns, heads, page, dh), torch.zeros(columns, heads, page, dh)
    k[..., 0] = (torch.randn(columns, heads, page, generator=g) * 0.8).clamp(-2, 2).to(dtype).float()
    table = torch.randperm(columns, generator=g)[None].to(torch.int32)
    q = torch.zeros(1, heads, nodes, dh)
    q[..., 0] = 8.0  # times 1 / sqrt(64)
    size = torch.zeros(heads, dh, dtype=torch.float64)
    want = torch.zeros(heads, dh, dtype=torch.float64)
    for h in range(heads):
        at = [(int(table[0, t // page]), t % page) for t in range(tokens)]
        w = torch.softmax(torch.stack([k[a, h, b, 0].double() for a, b in at]), 0)
        left = torch.zeros(dh, dtype=torch.float64)
        for n, t in enumerate(torch.tensor([5, 20, 41, 66]) + torch.tensor(nodes // 3)):
            x = 50 + 50 * torch.rand(dh, generator=g) if n == 0 else (-left / w[t]).float()
            x = x.to(dtype).float()
            v[at[t][0], h, at[t][1]] = x
            left += w[t] * x.double()
            size[h] += w[t] * x.double().abs()
        want[h] = left
    case = [t.to(dtype) for t in (k, v)] + [table]
    seen = torch.tensor([[(2 << i) - 1 for i in range(nodes)]], device=DEV)
    tree = paged_tree_attention(*dev(q.to(dtype), *case), numbers([start]), seen)[0, :, -1]
    one = paged_attention(*dev(q[:, :, -1].to(dtype), *case), numbers([tokens - 1]))[0]
    _native.poll_status(DEV)
    for got, more in ((tree, TREE[dtype]), (one, 2.0 ** -23)):
        off = (got.double().cpu() - want).abs()
        bound = size * (SUMS + more)
        step = torch.finfo(dtype).eps / 2 * (want.abs() + bound) + torch.finfo(dtype).tiny
        assert (off <= bound + step).all(), (off / (bound + step)).max().item()


# ---- values whose scales lie far apart ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("form", [I8, E4])
@pytest.mark.parametrize("dh,nodes,heads,page", [(64, 6, 2, 16), (64, 6, 2, 12), (128, 40, 2, 16), (64, 60, 1, 16), (144, 6, 2, 16)])
def test_scales_as_far_apart_as_is_allowed(dh, nodes, heads, page, form):
    """Values of zeros, whose scale is the least one, between some of 2^12: the zeros count in a row's sum of weights."""
    case = Case([70], [nodes], nodes, heads, 1, dh, page, BF, form, seed=nodes, branch=1)
    for t in range(70 + nodes):
        at = int(case.table[0, t // page]), slice(None), t % page
        if t % 3 == 1:
            case.v.view(torch.uint8)[at] = 0
        case.scales[1][at] = dr.LEAST if t % 3 == 1 else 2.0 ** 12
    got, (want, bound) = case.run(), case.want()
    check(got, want, bound)
    one = paged_attention(*dev(case.q[:, :, -1].contiguous(), case.k, case.v, case.table), numbers([70 + nodes - 1]), scales=dev(case.scales)[0])
    check(one, want[:, :, -1], bound[:, :, -1])
    _native.poll_status(DEV)
