"""Drafted tokens over a paged cache against plain forms in 64 bits: attention of a tree, its accepted path moved together."""

import math

import pytest
import torch

import paged_drafts_reference as dr
import paged_reference as pr
from titanmac_b200 import PagedCache, _native, draft_tree, paged_attention, paged_keep, paged_tree_attention

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32
I8, E4 = torch.int8, torch.float8_e4m3fn
# How much of itself a weight may be off by, as the operand of the product with the values: in 16-bit types it goes in as two numbers
# of the type, 16 bits in bf16 and 22 in fp16, 2^-36 of the largest weight at the least
WEIGHT = {BF: 2.0 ** -16, HF: 2.0 ** -22, FF: 0.0}


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
    assert (off <= allowed).all(), (off / allowed).max().item()


class Case:
    """Sequences of ``start`` tokens with ``counts`` drafted ones behind them, in a pool whose other slots hold infinities and NaN."""

    def __init__(self, start, counts, nodes, heads, kv_heads, dh, page, dtype, form=None, window=None, n_p=0, seed=0, branch=2, shape="tree"):
        g = torch.Generator().manual_seed(seed + 1)
        self.start, self.counts, self.window, self.dtype = torch.tensor(start), torch.tensor(counts), window, dtype
        lengths = [max(s, 0) + max(c, 0) for s, c in zip(start, counts)]
        self.scales = self.pers_scales = (None, None)
        if form is None:
            self.k, self.v, self.table = pr.pool(lengths, page, kv_heads, dh, dtype, seed, fill="wild")
        else:
            self.k, self.v, self.table, self.scales = dr.pool8(lengths, page, kv_heads, dh, form, seed)
        B = len(start)
        self.q = torch.randn(B, nodes, heads, dh, generator=g).to(dtype).permute(0, 2, 1, 3)
        self.pers = (None, None)
        if n_p:
            self.pers = tuple(torch.randn(kv_heads, n_p, dh, generator=g).to(dtype) for _ in range(2))
            if form is not None:
                (kp, ks), (vp, vs) = (dr.coded(t, form) for t in self.pers)
                self.pers, self.pers_scales = (kp, vp), (ks, vs)
        if shape == "tree":
            parents = [-1] + [(i - 1) // branch for i in range(1, nodes)]
            seen, depth = dr.ancestors(parents)
            self.seen, self.positions = seen.repeat(B, 1), (self.start.clamp(min=0)[:, None] + depth).to(torch.int32)
        else:  # any node may see any other one, and nothing
            bits = torch.rand(B, nodes, nodes, generator=g) < 0.4
            bits[:, 0] = False
            self.seen = (bits.long() << torch.arange(nodes)).sum(-1)
            self.positions = (self.start[:, None] + torch.randint(-3, 90, (B, nodes), generator=g)).to(torch.int32)

    def run(self, **kw):
        args = dict(counts=numbers(self.counts.tolist()), positions=self.positions.to(DEV), window=self.window, k_pers=dev(self.pers[0])[0],
                    v_pers=dev(self.pers[1])[0], scales=dev(self.scales)[0] if self.scales[0] is not None else None,
                    pers_scales=dev(self.pers_scales)[0] if self.pers_scales[0] is not None else None)
        args.update(kw)
        return paged_tree_attention(*dev(self.q, self.k, self.v, self.table), numbers(self.start.tolist()), self.seen.to(DEV), **args)

    def want(self, scale=0.0):
        off = WEIGHT[HF] if self.scales[0] is not None and self.dtype != FF else WEIGHT[self.dtype]
        return dr.tree_attention(self.q, self.k, self.v, self.table, self.start, self.seen, self.counts, self.positions, self.window,
                                 *self.pers, scale, self.scales, self.pers_scales, weight_off=off)


TREES = [
    ([0], [1], 1, 1, 1, 64, 16, None, 0),                                # one token alone
    ([700], [8], 8, 10, 10, 64, 64, 512, 16),                            # the default geometry
    ([15, 16, 17, 31, 1, 0], [1, 2, 3, 5, 16, 16], 16, 4, 4, 64, 16, None, 0),  # drafts that begin and end everywhere
    ([300, 3, 50], [16, 16, 9], 16, 8, 2, 128, 24, None, 3),             # shared heads, pages that end inside tiles
    ([513, 77, 20], [33, 7, 33], 33, 14, 2, 64, 7, 100, 5),              # a window that begins inside a tile, seven heads on one
    ([40, 100], [64, 63], 64, 16, 2, 128, 16, None, 0),                  # every bit of the mask
    ([90, 33], [5, 2], 5, 40, 2, 32, 64, None, 1),                       # twenty heads on one
    ([150, 20], [12, 6], 12, 6, 2, 256, 16, None, 17),                   # wide heads
    ([65, 200], [20, 1], 20, 4, 2, 96, 20, 30, 2),
    ([50, 9], [3, 3], 3, 2, 1, 64, 1, 0, 0),                             # the tree alone, pages of one token
    ([70, 45], [9, 9], 9, 2, 2, 144, 16, None, 1),                       # head sizes of no tile
    ([45, 100], [31, 4], 31, 3, 1, 80, 9, 60, 0),
]


@pytest.mark.parametrize("dtype,form", [(BF, None), (HF, None), (FF, None), (BF, I8), (HF, E4), (BF, E4), (FF, I8)])
@pytest.mark.parametrize("start,counts,nodes,heads,kv_heads,dh,page,window,n_p", TREES)
def test_trees_against_64_bits(start, counts, nodes, heads, kv_heads, dh, page, window, n_p, dtype, form):
    case = Case(start, counts, nodes, heads, kv_heads, dh, page, dtype, form, window, n_p, seed=dh + nodes)
    got = case.run()
    _native.poll_status(DEV)
    check(got, *case.want())


@pytest.mark.parametrize("dtype,form", [(BF, None), (HF, I8), (FF, None)])
@pytest.mark.parametrize("start,counts,nodes,heads,dh,window,n_p", [
    ([0, 30, 100], [40, 40, 17], 40, 4, 64, None, 0), ([0, 5], [64, 9], 64, 8, 128, None, 2), ([200, 61], [20, 20], 20, 2, 64, 50, 0)])
def test_any_mask(start, counts, nodes, heads, dh, window, n_p, dtype, form):
    """Nodes that see later ones, not themselves, or nothing at all; positions in front of the start and far behind it."""
    case = Case(start, counts, nodes, heads, 2, dh, 16, dtype, form, window, n_p, seed=nodes, shape="any")
    got = case.run()
    _native.poll_status(DEV)
    want, bound = case.want()
    check(got, want, bound)
    if start[0] == 0 and not n_p:
        assert (got[0, :, 0] == 0).all()


@pytest.mark.parametrize("dtype,dh", [(BF, 64), (HF, 128), (FF, 64), (BF, 144)])
def test_what_a_node_does_not_see_does_not_matter(dtype, dh):
    """Infinities and NaN in the keys and values of one branch, and in front of the window of the deeper nodes."""
    case = Case([70], [15], 15, 4, 2, dh, 16, dtype, window=40, seed=1)
    before, (want, bound) = case.run(), case.want()
    page = case.k.shape[2]
    for t, what in ((2, math.nan), (5, math.inf)):  # node 2 and, below it, node 5
        at = int(case.table[0, (70 + t) // page]), slice(None), (70 + t) % page
        case.k[at] = what
        case.v[at] = -what
    low = 70 - 40  # seen by the root alone
    case.v[int(case.table[0, low // page]), :, low % page] = math.inf
    got = case.run().cpu()
    _native.poll_status(DEV)
    touched = [i for i in range(15) if i == 0 or int(case.seen[0, i]) & 0b100100]
    free = [i for i in range(15) if i not in touched]
    assert len(free) >= 6 and not torch.isfinite(got[:, :, touched]).any()
    assert torch.isinf(got[:, :, 0]).all()
    check(got[:, :, free], want[:, :, free], bound[:, :, free])
    assert torch.isfinite(before).all()


def test_rows_that_are_not_there_are_left_as_they_are():
    case = Case([40, -1, 9], [3, 5, 0], 5, 4, 2, 64, 16, BF, seed=2)
    wide = torch.full((3, 5, 4, 70), 7.0, dtype=BF, device=DEV)
    out = wide.permute(0, 2, 1, 3)[..., 3:67]
    assert case.run(out=out) is out
    _native.poll_status(DEV)
    want, bound = case.want()
    check(out[:1, :, :3], want[:1, :, :3], bound[:1, :, :3])
    assert (out[0, :, 3:] == 7).all() and (out[1:] == 7).all() and (wide[..., :3] == 7).all() and (wide[..., 67:] == 7).all()


@pytest.mark.parametrize("dtype,heads,dh", [(BF, 4, 64), (HF, 16, 128), (FF, 2, 64)])
def test_what_has_no_place(dtype, heads, dh):
    case = Case([40, 40, 20, 3, 4], [8] * 5, 8, heads, 2, dh, 16, dtype, seed=3, branch=1)
    want, bound = case.want()
    case.table[0, 1] = -1           # context that every node sees
    case.table[1, 2] = 1 << 30      # nodes 0 .. 7
    case.start[2] = 48 * 1000       # behind the table
    case.counts[3] = 9
    got = case.run()
    reported()
    assert torch.isnan(got[:4]).all()
    check(got[4:], want[4:], bound[4:])
    case = Case([40], [16], 16, heads, 2, dh, 8, dtype, seed=4, branch=1)
    want, bound = case.want()
    case.table[0, 6] = -3           # nodes 8 .. 15
    got = case.run()
    reported()
    assert torch.isnan(got[:, :, 8:]).all()
    check(got[:, :, :8], want[:, :, :8], bound[:, :, :8])


@pytest.mark.parametrize("dtype,form", [(BF, None), (BF, I8), (FF, None)])
def test_many_sequences_of_every_size(dtype, form):
    start = [(37 * b) % 150 for b in range(120)]
    counts = [(5 * b) % 11 for b in range(120)]
    case = Case(start, counts, 10, 4, 2, 64, 16, dtype, form, seed=5)
    got = case.run()
    _native.poll_status(DEV)
    check(got, *case.want())


@pytest.mark.parametrize("dtype,form,dh,heads,kv_heads,nodes", [(BF, None, 64, 2, 2, 16), (HF, None, 128, 8, 1, 40), (BF, I8, 128, 8, 1, 12), (FF, None, 64, 2, 1, 8)])
def test_one_long_sequence(dtype, form, dh, heads, kv_heads, nodes):
    """Every CTA has a part of the same items, which are joined."""
    case = Case([6000], [nodes], nodes, heads, kv_heads, dh, 64, dtype, form, seed=6)
    got = case.run()
    again = case.run()
    assert torch.equal(got, again)
    check(got, *case.want())


@pytest.mark.parametrize("dtype", [BF, FF])
def test_a_chain_is_token_after_token(dtype):
    """Node i of a chain is what the attention of one token gives at its place."""
    case = Case([77], [9], 9, 8, 2, 64, 16, dtype, window=30, seed=7, branch=1)
    tree = draft_tree(torch.arange(-1, 8)[None], torch.tensor([77]), 30)
    assert torch.equal(tree.positions, case.positions) and torch.equal(tree.seen, case.seen)
    got = case.run()
    want, bound = case.want()
    for i in range(9):
        one = paged_attention(*dev(case.q[:, :, i].contiguous(), case.k, case.v, case.table), numbers([77 + i]), 30)
        check(one, want[:, :, i], bound[:, :, i])
    check(got, want, bound)


def test_two_streams_and_graphs():
    cases = [Case([700, 3], [16, 2], 16, 8, 2, 64, 16, BF, seed=8), Case([50] * 9, [5] * 9, 5, 4, 4, 128, 16, BF, seed=9)]
    want = [c.run() for c in cases]
    streams, graphs, outs = [torch.cuda.Stream(DEV) for _ in cases], [], []
    args = []
    for c in cases:  # what a captured call reads has to stay
        args.append((dev(c.q, c.k, c.v, c.table) + [numbers(c.start.tolist()), c.seen.to(DEV)], numbers(c.counts.tolist())))
    torch.cuda.synchronize(DEV)
    for (a, n), s in zip(args, streams):
        with torch.cuda.stream(s):
            paged_tree_attention(*a, n)
        torch.cuda.synchronize(DEV)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(paged_tree_attention(*a, n))
        graphs.append(graph)
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize(DEV)
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


def test_a_cache_takes_a_tree():
    """Drafts rotated by their depth, appended, attended to; the accepted path kept; the next token on top, as if it had come alone."""
    B, H, KV, dh = 2, 4, 2, 64
    g = torch.Generator().manual_seed(3)
    inv_freq = (100.0 ** (-torch.arange(32) / 32)).float().to(DEV)
    table = torch.randperm(12, generator=g).view(2, 6).to(torch.int32).to(DEV)
    parents = torch.tensor([[-1, 0, 0, 2, 2, 4], [-1, 0, 1, 0, 3, 4]])
    path = [[0, 2, 4, 5], [0, 3, 4, 5]]  # of each tree
    prompt = [torch.randn(B, KV, 30, dh, generator=g).to(BF).to(DEV) for _ in range(2)]
    drafts = [torch.randn(B, n, 6, dh, generator=g).to(BF).to(DEV) for n in (H, KV, KV)]
    last = [torch.randn(B, n, dh, generator=g).to(BF).to(DEV) for n in (H, KV, KV)]
    lengths = numbers([30, 21])
    tree = draft_tree(parents.to(DEV), lengths)

    def cache():
        c = PagedCache(table, 12, 8, KV, dh, None, 0, BF, inv_freq=inv_freq)
        c.append(*prompt, numbers([0, 0]), lengths)
        return c

    a, b = cache(), cache()
    outs = a.decode_tree(*drafts, lengths, tree)
    a.keep(lengths, numbers(path), numbers([4, 4]))
    for i in range(4):  # the same path, token by token
        pick = [torch.stack([t[n, :, path[n][i]] for n in range(B)]) for t in drafts]
        one = b.decode(*pick, lengths + i)
        for n in range(B):
            assert (outs[n, :, path[n][i]].float() - one[n].float()).abs().max() <= 2.0 ** -7 * one[n].float().abs().max()
    got, want = a.decode(*last, lengths + 4), b.decode(*last, lengths + 4)
    assert torch.equal(got, want)  # the same keys in the same places
    _native.poll_status(DEV)


# ---- keep -----------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,form,dh,page", [(BF, None, 64, 16), (FF, None, 256, 5), (HF, None, 8, 3), (BF, I8, 64, 16), (BF, E4, 128, 7)])
@pytest.mark.parametrize("start,kept", [([0, 17], [[0, 1, 2], [1, 2, 3]]), ([9], [[5]]), ([3, -1, 60], [[0, 7, 40, 63], [1, 2, 3, 4], [2, 3, 4]]),
                                        ([12], [list(range(1, 64))]), ([12], [list(range(64))]), ([4], [[]])])
def test_keep_moves_tokens(start, kept, dtype, form, dh, page):
    lengths = [max(s, 0) + 64 for s in start]
    if form is None:
        k, v, table = pr.pool(lengths, page, 3, dh, dtype, 4)
        scales = None
    else:
        k, v, table, scales = dr.pool8(lengths, page, 3, dh, form, 4)
    most = max(1, max(len(x) for x in kept))
    rows = [x + [-9] * (most - len(x)) for x in kept]
    d = dev(k, v, table, scales)
    paged_keep(*d[:3], numbers(start), numbers(rows), numbers([len(x) for x in kept]), scales=d[3])
    _native.poll_status(DEV)
    for got, t in zip((d[0], d[1], *(d[3] or ())), (k, v, *(scales or ()))):
        want = t.clone() if t.dtype != E4 else t.clone()
        for b, x in enumerate(kept):
            for i, j in enumerate(x if start[b] >= 0 else []):
                to, source = ((int(table[b, (start[b] + n) // page]), (start[b] + n) % page) for n in (i, j))
                want[to[0], :, to[1]] = t[source[0], :, source[1]]
        assert torch.equal(got.cpu().contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))


@pytest.mark.parametrize("rows,count,start,break_page", [([1, 1], 2, 0, None), ([2, 1], 2, 0, None), ([0, -1], 2, 0, None), ([1, 2], 3, 0, None),
                                                         ([1, 2], -1, 0, None), ([1, 2], 2, -2, None), ([1, 60], 2, 10, None), ([1, 20], 2, 0, 1)])
def test_keep_leaves_alone_what_does_not_hold(rows, count, start, break_page):
    k, v, table = pr.pool([64, 64], 16, 2, 32, BF, 4)
    if break_page is not None:
        table[0, break_page] = -1
    d = dev(k, v, table)
    paged_keep(*d, numbers([start, 5]), numbers([rows, [1, 2]]), numbers([count, 1]))
    reported()
    want_k = k.clone()
    want_k[int(table[1, 0]), :, 5] = k[int(table[1, 0]), :, 6]
    assert torch.equal(d[0].cpu(), want_k)


# ---- many rows to a key head ------------------------------------------------------------------------------------------------

MANY = [
    ([300, 3, 50], [33, 33, 17], 33, 8, 2, 128, 32, None, 3),             # 132 rows: one block of 128 and a small one
    ([513, 77, 20, 0], [64, 1, 40, 64], 64, 4, 4, 64, 64, 100, 5),        # 64 rows, a window, a tree without tokens in front
    ([1000], [64], 64, 8, 1, 64, 16, None, 0),                            # 512 rows: four blocks
    ([129, 64, 63, 1], [40, 40, 40, 40], 40, 4, 2, 128, 8, 37, 0),        # runs of eight, windows that begin in tiles
    ([700], [20], 20, 10, 5, 64, 128, None, 100),                         # more persistent keys than a tile
    ([90, 200], [50, 12], 50, 3, 1, 128, 24, None, 64),
]


@pytest.mark.parametrize("dtype,form", [(BF, None), (HF, None), (BF, I8), (HF, E4)])
@pytest.mark.parametrize("start,counts,nodes,heads,kv_heads,dh,page,window,n_p", MANY)
def test_many_rows_against_64_bits(start, counts, nodes, heads, kv_heads, dh, page, window, n_p, dtype, form):
    case = Case(start, counts, nodes, heads, kv_heads, dh, page, dtype, form, window, n_p, seed=dh + nodes)
    got = case.run()
    _native.poll_status(DEV)
    check(got, *case.want())


@pytest.mark.parametrize("dtype,dh,start", [(BF, 64, 70), (HF, 128, 70), (BF, 128, 200), (HF, 64, 3), (BF, 128, 0)])
def test_what_many_rows_do_not_see_does_not_matter(dtype, dh, start):
    """As above with 40 nodes of a chain and a half: infinities and NaN in nodes that some see, in one tile and across two."""
    nodes, page = 40, 16
    case = Case([start], [nodes], nodes, 4, 2, dh, page, dtype, seed=1)
    parents = [-1] + [0 if i == 20 else i - 1 for i in range(1, nodes)]  # 1 .. 19 and 20 .. 39 are two branches
    case.seen = dr.ancestors(parents)[0][None]
    want, bound = case.want()
    for node, what in ((10, math.inf), (30, math.nan)):
        at = int(case.table[0, (start + node) // page]), slice(None), (start + node) % page
        case.v[at] = what
    case.v[int(case.table[0, (start + 35) // page]), :, (start + 35) % page, ::2] = -math.inf
    got = case.run().cpu()
    _native.poll_status(DEV)
    assert torch.isinf(got[:, :, 10:20]).all() and (got[:, :, 10:20] > 0).all() and torch.isnan(got[:, :, 30:]).all()
    free = list(range(10)) + list(range(20, 30))
    check(got[:, :, free], want[:, :, free], bound[:, :, free])


@pytest.mark.parametrize("dtype,form", [(BF, None), (HF, None), (BF, I8)])
def test_many_rows_with_any_mask(dtype, form):
    case = Case([0, 130, 64], [64, 40, 64], 64, 4, 2, 64, 16, dtype, form, 70, 0, seed=3, shape="any")
    got = case.run()
    _native.poll_status(DEV)
    check(got, *case.want())
    assert (got[0, :, 0] == 0).all()


@pytest.mark.parametrize("dtype,dh", [(BF, 64), (HF, 128)])
def test_many_rows_and_what_has_no_place(dtype, dh):
    case = Case([150, 40, 40], [40] * 3, 40, 4, 2, dh, 16, dtype, seed=3, branch=1)
    want, bound = case.want()
    case.table[0, 3] = -1           # context that every node sees
    case.table[1, 4] = 1 << 30      # nodes 24 .. 39
    got = case.run()
    reported()
    assert torch.isnan(got[0]).all() and torch.isnan(got[1, :, 24:]).all()
    check(got[1, :, :24], want[1, :, :24], bound[1, :, :24])
    check(got[2:], want[2:], bound[2:])


@pytest.mark.parametrize("dtype,dh,heads,nodes", [(BF, 64, 4, 48), (HF, 128, 8, 33)])
def test_many_rows_of_a_long_sequence_and_of_many(dtype, dh, heads, nodes):
    case = Case([9000], [nodes], nodes, heads, 1, dh, 64, dtype, seed=6)
    got = case.run()
    assert all(torch.equal(got, case.run()) for _ in range(3))
    check(got, *case.want())
    case = Case([(37 * b) % 200 for b in range(90)], [(5 * b) % (nodes + 1) for b in range(90)], nodes, heads, 1, dh, 16, dtype, n_p=3, seed=7)
    got = case.run()
    _native.poll_status(DEV)
    check(got, *case.want())


def test_many_rows_with_strides():
    case = Case([140], [40], 40, 2, 2, 64, 16, BF, seed=2)
    q, out = torch.zeros(1, 40, 2, 67, dtype=BF), torch.zeros(1, 40, 2, 71, dtype=BF, device=DEV)
    q[..., 1:65] = case.q.permute(0, 2, 1, 3)
    got = paged_tree_attention(q.to(DEV).permute(0, 2, 1, 3)[..., 1:65], *dev(case.k, case.v, case.table), numbers([140]), case.seen.to(DEV),
                               out=out.permute(0, 2, 1, 3)[..., 3:67])
    check(got, *case.want())
    assert (out[..., :3] == 0).all() and (out[..., 67:] == 0).all()


@pytest.mark.parametrize("dtype,form", [(BF, None), (HF, None), (BF, I8), (HF, E4)])
@pytest.mark.parametrize("page", [16, 12])
@pytest.mark.parametrize("dh,nodes,group", [(128, 8, 1), (128, 9, 1), (128, 4, 4), (128, 31, 1), (128, 8, 4), (128, 33, 1), (64, 16, 2), (64, 33, 1),
                                            (64, 12, 4), (64, 49, 1), (64, 7, 7)])
def test_rows_on_both_sides_of_what_tcgen05_takes(dh, nodes, group, page, dtype, form):
    case = Case([210, 0, 65], [nodes, nodes, 1], nodes, 2 * group, 2, dh, page, dtype, form, 90, 3, seed=nodes)
    got = case.run()
    _native.poll_status(DEV)
    check(got, *case.want())
