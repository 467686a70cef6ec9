"""Calls over pages of 8 bits and of drafted trees that lie at the edge of what is allowed: empty pools, scales and tables that are views,
shared pages, no nodes, forward-mode derivatives."""

import pytest
import torch
from torch.autograd import forward_ad

from titanmac_b200 import (TitanMAC, TitanMACConfig, _native, draft_tree, paged_append, paged_attention, paged_keep, paged_read,
                           paged_tree_attention)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, FF, I8, E4 = torch.bfloat16, torch.float32, torch.int8, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _fresh_status():
    _native.poll_status(DEV)
    yield


def numbers(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def pool(pages, kv_heads, page, dh, held, gen):
    shape = (pages, kv_heads, page, dh)
    if held is BF:
        return (torch.randn(shape, generator=gen).to(BF).to(DEV), torch.randn(shape, generator=gen).to(BF).to(DEV)), None
    codes = tuple((torch.randint(-127, 128, shape, generator=gen).to(I8) if held is I8 else torch.randn(shape, generator=gen).mul(100).to(E4)).to(DEV)
                  for _ in range(2))
    return codes, tuple((torch.rand(shape[:3], generator=gen) * 0.02 + 0.001).to(DEV) for _ in range(2))


def tree_of(B, nodes, start):
    parents = torch.tensor([[-1] + [(i - 1) // 2 for i in range(1, nodes)]] * B, device=DEV)
    return draft_tree(parents, start)


@pytest.mark.parametrize("held,heads,nodes,page", [(BF, 2, 5, 16), (BF, 2, 40, 16), (I8, 2, 40, 16), (E4, 2, 5, 16), (I8, 2, 5, 12)])
@pytest.mark.parametrize("n_p", [0, 3])
def test_a_pool_of_no_pages(held, heads, nodes, page, n_p):
    g = torch.Generator().manual_seed(0)
    (k, v), scales = pool(0, heads, page, 64, held, g)
    (kp, vp), pers = pool(1, heads, 3, 64, held, g)
    more = dict(scales=scales)
    if n_p:
        more.update(k_pers=kp[0], v_pers=vp[0], pers_scales=pers and tuple(t[0] for t in pers))
    table, start = torch.zeros(2, 5, dtype=torch.int32, device=DEV), numbers([7, -1])
    q = torch.randn(2, heads, nodes, 64, generator=g).to(BF).to(DEV)
    tree = tree_of(2, nodes, start)
    out = paged_tree_attention(q, k, v, table, start, tree.seen, positions=tree.positions, **more)
    assert torch.isnan(out[0]).all() and (out[1] == 0).all()
    with pytest.raises(_native.TmwError):
        _native.poll_status(DEV)
    out = paged_attention(q[:, :, 0], k, v, table, start, **more)
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()
    with pytest.raises(_native.TmwError):
        _native.poll_status(DEV)


@pytest.mark.parametrize("held", [I8, E4])
@pytest.mark.parametrize("heads,kv_heads,nodes", [(4, 4, 9), (8, 2, 17), (8, 1, 3)])
def test_scales_and_tables_that_are_views(held, heads, kv_heads, nodes):
    """Scales that begin four bytes behind sixteen, rows of a wider table: the same numbers by other copies.  Both results are rounded
    from sums that agree to a few 2^-20 of the largest value; they may be neighbours in bf16, 2^-7 apart."""
    g = torch.Generator().manual_seed(1)
    (k, v), scales = pool(24, kv_heads, 16, 128, held, g)
    wide = torch.randperm(24, generator=g).to(torch.int32).view(2, 12).to(DEV)
    other = [torch.empty(t.numel() + 1, device=DEV)[1:].view(t.shape).copy_(t) for t in scales]
    assert all(t.data_ptr() % 16 == 4 and t.is_contiguous() for t in other)
    start, q = numbers([60, 25]), torch.randn(2, heads, nodes, 128, generator=g).to(BF).to(DEV)
    tree = tree_of(2, nodes, start)
    both = [(paged_tree_attention(q, k, v, t, start, tree.seen, scales=s), paged_attention(q[:, :, 0].contiguous(), k, v, t, start, scales=s))
            for s, t in ((scales, wide[:, :6].contiguous()), (tuple(other), wide[:, :6]))]
    for a, b in zip(*both):
        nan = torch.isnan(a)  # (e4m3 codes may be NaN: the same outputs are)
        assert torch.equal(nan, torch.isnan(b)) and not nan.all()
        a, b = (t.float().masked_fill(nan, 0) for t in (a, b))
        assert bool((a - b).abs().max() <= 2.0 ** -7 * a.abs().max())
    codes, dense = (paged_read(k, v, wide[:, :6], start, 20, dtype=FF, scales=s) for s in (scales, other))
    assert all(bool(((x == y) | (torch.isnan(x) & torch.isnan(y))).all()) for x, y in zip(codes, dense))
    _native.poll_status(DEV)


@pytest.mark.parametrize("held", [BF, I8])
def test_sequences_that_share_the_pages_in_front_of_their_drafts(held):
    """A prompt's pages belong to three sequences, each with a page of its own behind them: what each says is what it says with a copy."""
    g = torch.Generator().manual_seed(2)
    (k, v), scales = pool(16, 2, 16, 64, held, g)
    shared = torch.tensor([[0, 1, 2], [0, 1, 3], [0, 1, 4]], dtype=torch.int32, device=DEV)
    apart = torch.tensor([[0, 1, 2], [5, 6, 3], [7, 8, 4]], dtype=torch.int32, device=DEV)
    for t in (k, v) + (scales or ()):
        for a, b in ((5, 0), (6, 1), (7, 0), (8, 1)):
            t.view(torch.uint8 if t.dtype is I8 else t.dtype)[a] = t.view(torch.uint8 if t.dtype is I8 else t.dtype)[b]
    start, q = numbers([32, 32, 32]), torch.randn(3, 2, 11, 64, generator=g).to(BF).to(DEV)
    tree = tree_of(3, 11, start)
    a, b = (paged_tree_attention(q, k, v, t, start, tree.seen, scales=scales) for t in (shared, apart))
    assert torch.equal(a, b)
    before = [t.clone() for t in (k, v)]
    paged_keep(k, v, shared, start, numbers([[0, 3, 7]] * 3), numbers([3, 3, 3]), scales=scales)
    for t, old in zip((k, v), before):
        assert torch.equal(t[:2].float(), old[:2].float()) and torch.equal(t[2:5, :, [0, 1, 2]].float(), old[2:5, :, [0, 3, 7]].float())
    _native.poll_status(DEV)


def test_no_nodes_and_no_sequences():
    cfg = TitanMACConfig(vocab_size=64, d_model=128, n_heads=2, n_layers=1, d_ff=256, max_seq_len=64, window_size=16, n_persistent=2,
                         use_block_sparse=False)
    model = TitanMAC(cfg).to(device=DEV, dtype=BF).eval()
    table = torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4)
    caches = model.prefill(torch.randint(0, 64, (2, 9), device=DEV), model.new_paged_caches(table, 8, 8, BF, I8))[1]
    none = torch.zeros(2, 0, dtype=torch.int64, device=DEV)
    assert model.decode_tree(none, none, numbers([9, 9]), caches).shape == (2, 0, 64)
    model.keep_drafts(caches, numbers([9, 9]), torch.zeros(2, 0, dtype=torch.int32, device=DEV), numbers([0, 0]))
    before = caches[0].k_pages.clone()
    one = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    out = model.decode_tree(one, one - 1, numbers([-1, -1]), caches)
    assert out.shape == (2, 3, 64) and torch.equal(before, caches[0].k_pages)
    _native.poll_status(DEV)


def test_reading_and_keeping_refuse_forward_mode():
    k = torch.zeros(2, 1, 8, 16, device=DEV)
    table = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(k, torch.ones_like(k))
        with pytest.raises(NotImplementedError):
            paged_read(dual, k, table, numbers([0]), 1)
        with pytest.raises(NotImplementedError):
            paged_keep(dual, k, table, numbers([0]), numbers([[0]]), numbers([1]))
    # (nothing is refused outside)
    paged_append(k[:1, :, :1], k[:1, :, :1], k, k.clone(), table, numbers([0]))
    _native.poll_status(DEV)
