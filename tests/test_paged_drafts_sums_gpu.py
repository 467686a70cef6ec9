"""Drafted trees where their sums are delicate: what single numbers of a value do to the rows that see them and to those that do not."""

import pytest
import torch

import paged_drafts_reference as dr
from test_paged_drafts_gpu import BF, DEV, E4, FF, HF, Case, check
from titanmac_b200 import _native

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
