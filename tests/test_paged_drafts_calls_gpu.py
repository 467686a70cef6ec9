"""Calls over pages of 8 bits and drafted trees that took, or dropped, something without a word."""

import pytest
import torch
from torch.autograd import forward_ad

from test_model_drafts_gpu import BF, DEV, E4, FF, I8, build, numbers
from titanmac_b200 import (PagedCache, _native, paged_append, paged_attention, paged_keep, paged_read, paged_tree_attention)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _fresh_status():
    _native.poll_status(DEV)
    yield


@pytest.mark.parametrize("which", ["k_scales", "v_scales", "k_pers_scales", "v_pers_scales"])
def test_scales_with_a_forward_mode_derivative_are_refused(which):
    codes, pers = torch.zeros(2, 1, 8, 16, dtype=I8, device=DEV), torch.zeros(1, 3, 16, dtype=I8, device=DEV)
    table, x = torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.zeros(1, 1, 1, 16, device=DEV)
    seen = torch.ones(1, 1, dtype=torch.int64, device=DEV)
    s = {n: torch.ones(2, 1, 8, device=DEV) if "pers" not in n else torch.ones(1, 3, device=DEV)
         for n in ("k_scales", "v_scales", "k_pers_scales", "v_pers_scales")}

    def calls():
        scales, more = (s["k_scales"], s["v_scales"]), dict(k_pers=pers, v_pers=pers, pers_scales=(s["k_pers_scales"], s["v_pers_scales"]))
        yield lambda: paged_attention(x[:, :, 0], codes, codes, table, numbers([0]), scales=scales, **more)
        yield lambda: paged_tree_attention(x, codes, codes, table, numbers([0]), seen, scales=scales, **more)
        if "pers" not in which:
            yield lambda: paged_append(x, x, codes, codes.clone(), table, numbers([0]), scales=scales)
            yield lambda: paged_read(codes, codes, table, numbers([0]), 1, dtype=FF, scales=scales)
            yield lambda: paged_keep(codes, codes.clone(), table, numbers([0]), numbers([[0]]), numbers([1]), scales=scales)

    for call in calls():  # nothing is refused outside
        call()
    with forward_ad.dual_level():
        s[which] = forward_ad.make_dual(s[which], torch.ones_like(s[which]))
        for call in calls():
            with pytest.raises(NotImplementedError):
                call()
    _native.poll_status(DEV)


def test_angles_with_a_forward_mode_derivative_are_refused():
    pages, table = torch.zeros(2, 1, 8, 16, device=DEV), torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    x, inv_freq = torch.zeros(1, 1, 1, 16, device=DEV), torch.ones(8, device=DEV)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            paged_append(x, x, pages, pages.clone(), table, numbers([0]), inv_freq=forward_ad.make_dual(inv_freq, torch.ones_like(inv_freq)))


@pytest.mark.parametrize("page_dtype", [None, I8, E4])
def test_persistent_rows_of_any_strides(page_dtype):
    """Keys and values whose numbers are not neighbours in memory, as a cache in the model's type takes them."""
    g = torch.Generator().manual_seed(0)
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    k, v = (torch.randn(32, 2, 5, generator=g).to(BF).to(DEV).permute(1, 2, 0) for _ in range(2))
    caches = [PagedCache(table, 1, 8, 2, 32, None, 5, BF, page_dtype=page_dtype) for _ in range(2)]
    caches[0].set_persistent(k, v)
    caches[1].set_persistent(k.contiguous(), v.contiguous())
    for name in ("k_pers", "v_pers"):
        a, b = (getattr(c, name).float() for c in caches)
        assert torch.equal(a, b) and a.abs().max() > 0
    if page_dtype is not None:
        assert all(torch.equal(a, b) for a, b in zip(caches[0].pers_scales, caches[1].pers_scales))
    _native.poll_status(DEV)


def test_a_tree_goes_through_every_layer():
    """Fewer or more caches than layers: not a model's answer that leaves layers out."""
    model = build(FF)
    table = torch.arange(2 * 8).view(2, 8).to(torch.int32).to(DEV)
    _, caches = model.prefill(torch.randint(0, 64, (2, 9), device=DEV), model.new_paged_caches(table, 16, 8, FF))
    drafts, parents = torch.zeros(2, 3, dtype=torch.int64, device=DEV), torch.tensor([[-1, 0, 0]] * 2, device=DEV)
    before = [c.k_pages.clone() for c in caches]
    for some in (caches[:1], caches + caches[:1], []):
        with pytest.raises(ValueError):
            model.decode_tree(drafts, parents, numbers([9, 9]), some)
        with pytest.raises(ValueError):
            model.keep_drafts(some, numbers([9, 9]), numbers([[0]] * 2), numbers([1, 1]))
    assert all(torch.equal(c.k_pages, b) for c, b in zip(caches, before))
    _native.poll_status(DEV)


@pytest.mark.parametrize("dtype,nodes", [(FF, 4), (BF, 4), (BF, 40)])
def test_a_tree_that_does_not_end_within_its_pages(dtype, nodes):
    """Its nodes are NaN, all of them, and that is reported; the other sequence's are as they are alone, and so are the pages."""
    model = build(dtype, positions=200)
    table = torch.arange(2 * 8).view(2, 8).to(torch.int32).to(DEV)  # room for 64 tokens
    _, caches = model.prefill(torch.randint(0, 64, (2, 62), device=DEV), model.new_paged_caches(table, 16, 8, dtype))
    drafts, parents = torch.randint(0, 64, (2, nodes), device=DEV), torch.arange(-1, nodes - 1, device=DEV).expand(2, nodes).contiguous()
    alone = model.decode_tree(drafts, parents, numbers([20, -1]), caches)
    _native.poll_status(DEV)
    before = [c.k_pages[8:14].clone() for c in caches]
    got = model.decode_tree(drafts, parents, numbers([20, 62]), caches)
    with pytest.raises(_native.TmwError):
        _native.poll_status(DEV)
    assert torch.isnan(got[1]).all() and torch.equal(got[0], alone[0])
    assert all(torch.equal(c.k_pages[8:14], b) for c, b in zip(caches, before))
