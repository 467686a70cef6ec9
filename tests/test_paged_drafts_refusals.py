"""What the entries of pages in 8 bits and of drafted tokens refuse before anything is launched, the layout of their descriptions, and
the trees that the package makes."""

import os
import subprocess
import tempfile

import pytest
import torch

from conftest import ROOT
from paged_drafts_reference import ancestors
from test_operator_refusals import APPEND, ATTENTION, FAKE, PAGES, PAGES_REFUSED, packed
from titanmac_b200 import _native, draft_tree, paged_cache, paged_keep, paged_read, paged_tree_attention

OK, BAD, UNSUPPORTED, LARGE = (_native.TMW_OK, _native.TMW_ERR_INVALID_ARGUMENT, _native.TMW_ERR_UNSUPPORTED, _native.TMW_ERR_TOO_LARGE)
SCALES = dict(format=1, reserved=0, k_scales=FAKE, v_scales=FAKE, k_pers_scales=FAKE, v_pers_scales=FAKE)
READ = dict(PAGES, rows=3, reserved2=0, k=FAKE, v=0x2000, **{f"{n}{i}": 64 for n in ("ks", "vs") for i in range(3)}, start=FAKE, counts=0)
TREE = dict(PAGES, heads=4, nodes=8, n_persistent=1, window=-1, scale=0.0, reserved2=0, q=FAKE, k_pers=FAKE, v_pers=FAKE, o=0x2000,
            **{f"{n}{i}": 64 for n in ("qs", "os") for i in range(3)}, start=FAKE, counts=0, positions=0, seen=FAKE)
KEEP = dict(PAGES, rows=4, reserved2=0, start=FAKE, kept=FAKE, counts=FAKE)
SCALES_REFUSED = [(dict(format=3), UNSUPPORTED), (dict(format=-1), UNSUPPORTED), (dict(k_scales=0), BAD), (dict(v_scales=0x1002), BAD)]


def scales(**changes):
    return packed(paged_cache._SCALES, SCALES, **changes)


def test_layouts_match_the_header():
    src = r"""
    #include <stdio.h>
    #include <stddef.h>
    #include "tmw.h"
    int main(void) {
        printf("%zu %zu %zu %zu\n", sizeof(tmw_paged_read_desc), sizeof(tmw_paged_tree_desc), sizeof(tmw_paged_keep_desc), sizeof(tmw_page_scales));
        printf("%zu %zu %zu\n", offsetof(tmw_paged_read_desc, k), offsetof(tmw_paged_read_desc, v_stride), offsetof(tmw_paged_read_desc, start));
        printf("%zu %zu %zu %zu\n", offsetof(tmw_paged_tree_desc, nodes), offsetof(tmw_paged_tree_desc, o), offsetof(tmw_paged_tree_desc, o_stride), offsetof(tmw_paged_tree_desc, seen));
        printf("%zu %zu\n", offsetof(tmw_paged_keep_desc, kept), offsetof(tmw_page_scales, k_pers_scales));
        return 0;
    }
    """
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "t.c"), os.path.join(d, "t")
        open(c, "w").write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        lines = [[int(v) for v in line.split()] for line in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines()]
    assert lines[0] == [s.size for s in (paged_cache._READ, paged_cache._TREE, paged_cache._KEEP, paged_cache._SCALES)]

    def at(layout, fields, name):  # where a mark put into the field comes out
        zeros, marked = layout.pack(*[0] * len(fields)), layout.pack(*[(1 if n == name else 0) for n in fields])
        return next(i for i in range(len(zeros)) if zeros[i] != marked[i])

    assert lines[1] == [at(paged_cache._READ, READ, n) for n in ("k", "vs0", "start")]
    assert lines[2] == [at(paged_cache._TREE, TREE, n) for n in ("nodes", "o", "os0", "seen")]
    assert lines[3] == [at(paged_cache._KEEP, KEEP, "kept"), at(paged_cache._SCALES, SCALES, "k_pers_scales")]


@pytest.mark.parametrize("change,status", PAGES_REFUSED + [(dict(head_dim=72), UNSUPPORTED), (dict(rows=-1), BAD), (dict(k=0), BAD), (dict(ks1=-64), BAD)])
def test_scaled_append_refuses(change, status):
    assert _native.lib().tmw_paged_append_scaled(packed(paged_cache._APPEND, APPEND, **change), scales(), None, None) == status


@pytest.mark.parametrize("change,status", PAGES_REFUSED + [
    (dict(head_dim=72), UNSUPPORTED), (dict(rows=-1), BAD), (dict(k=0), BAD), (dict(v=0), BAD), (dict(start=0), BAD), (dict(k=0x1001), BAD),
    (dict(vs2=-1), BAD), (dict(ks0=0), BAD), (dict(vs1=0), BAD), (dict(v=FAKE), BAD)])
def test_read_refuses(change, status):
    assert _native.lib().tmw_paged_read(packed(paged_cache._READ, READ, **change), scales(), None) == status


@pytest.mark.parametrize("change,status", PAGES_REFUSED + [
    (dict(head_dim=72), UNSUPPORTED), (dict(heads=3), BAD), (dict(window=-2), BAD), (dict(q=0), BAD), (dict(pos=0), BAD), (dict(o=FAKE), BAD)])
def test_scaled_attention_refuses(change, status):
    lib, desc = _native.lib(), packed(paged_cache._ATTENTION, ATTENTION, **change)
    assert lib.tmw_paged_attention_scaled(desc, scales(), FAKE, 1 << 30, None) == status


@pytest.mark.parametrize("change,status", PAGES_REFUSED + [
    (dict(heads=3), BAD), (dict(heads=-2), BAD), (dict(nodes=-1), BAD), (dict(nodes=65), LARGE), (dict(n_persistent=-1), BAD), (dict(window=-2), BAD),
    (dict(window=5), BAD), (dict(scale=-1.0), BAD), (dict(scale=float("nan")), BAD), (dict(q=0), BAD), (dict(o=0), BAD), (dict(start=0), BAD),
    (dict(seen=0), BAD), (dict(seen=0x1004), BAD), (dict(k_pers=0), BAD), (dict(qs2=-1), BAD), (dict(os2=-1), BAD), (dict(os2=0), BAD),
    (dict(os1=0), BAD), (dict(o=FAKE), BAD), (dict(q=0x1001), BAD)])
def test_tree_refuses(change, status):
    lib, desc = _native.lib(), packed(paged_cache._TREE, TREE, **change)
    assert lib.tmw_paged_tree_attention(desc, None, FAKE, 1 << 30, None) == status
    assert lib.tmw_paged_tree_attention(desc, scales(), FAKE, 1 << 30, None) == status


@pytest.mark.parametrize("change,status", PAGES_REFUSED + [(dict(rows=-1), BAD), (dict(rows=65), LARGE), (dict(start=0), BAD), (dict(kept=0), BAD), (dict(counts=0), BAD)])
def test_keep_refuses(change, status):
    assert _native.lib().tmw_paged_keep(packed(paged_cache._KEEP, KEEP, **change), None, None) == status


@pytest.mark.parametrize("change,status", SCALES_REFUSED)
def test_scales_are_checked(change, status):
    lib, s = _native.lib(), scales(**change)
    assert lib.tmw_paged_append_scaled(packed(paged_cache._APPEND, APPEND), s, None, None) == status
    assert lib.tmw_paged_read(packed(paged_cache._READ, READ), s, None) == status
    assert lib.tmw_paged_attention_scaled(packed(paged_cache._ATTENTION, ATTENTION), s, FAKE, 1 << 30, None) == status
    assert lib.tmw_paged_tree_attention(packed(paged_cache._TREE, TREE), s, FAKE, 1 << 30, None) == status
    assert lib.tmw_paged_keep(packed(paged_cache._KEEP, KEEP), s, None) == status


def test_scales_of_persistent_keys_and_scratch_are_checked():
    lib = _native.lib()
    attention, tree = packed(paged_cache._ATTENTION, ATTENTION), packed(paged_cache._TREE, TREE)
    assert lib.tmw_paged_attention_scaled(attention, scales(k_pers_scales=0), FAKE, 1 << 30, None) == BAD
    assert lib.tmw_paged_tree_attention(tree, scales(v_pers_scales=0), FAKE, 1 << 30, None) == BAD
    assert lib.tmw_paged_attention_scaled(attention, None, FAKE, 1 << 30, None) == BAD
    assert lib.tmw_paged_attention_scaled(attention, scales(format=0), FAKE, 1 << 30, None) == BAD
    for at in (None, 0x1008):
        assert lib.tmw_paged_attention_scaled(attention, scales(), at, 1 << 30, None) == BAD
        assert lib.tmw_paged_tree_attention(tree, scales(), at, 1 << 30, None) == BAD
    for call in (lib.tmw_paged_attention_scaled, lib.tmw_paged_tree_attention):
        assert call(None, scales(), FAKE, 1 << 30, None) == BAD
    assert lib.tmw_paged_read(None, None, None) == lib.tmw_paged_keep(None, None, None) == BAD
    assert lib.tmw_paged_append_scaled(None, None, None, None) == BAD


def test_nothing_to_do_is_fine():
    lib, nothing = _native.lib(), dict(k_pages=0, v_pages=0, page_table=0)
    empty = scales(k_scales=0, v_scales=0, k_pers_scales=0, v_pers_scales=0)
    for change in (dict(batch=0), dict(rows=0)):
        assert lib.tmw_paged_append_scaled(packed(paged_cache._APPEND, APPEND, **nothing, **change), empty, None, None) == OK
        assert lib.tmw_paged_read(packed(paged_cache._READ, READ, **nothing, **change), empty, None) == OK
        assert lib.tmw_paged_keep(packed(paged_cache._KEEP, KEEP, **nothing, **change), empty, None) == OK
    for change in (dict(batch=0), dict(heads=0), dict(nodes=0)):
        assert lib.tmw_paged_tree_attention(packed(paged_cache._TREE, TREE, **nothing, **change), empty, None, 0, None) == OK
    assert lib.tmw_paged_attention_scaled(packed(paged_cache._ATTENTION, ATTENTION, batch=0, **nothing), empty, None, 0, None) == OK


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("form", [0, 1, 2])
@pytest.mark.parametrize("head_dim", [16, 64, 96, 128, 240, 256])
def test_scratch_grows_with_the_work_up_to_the_gpu(head_dim, form, dtype):
    def size(**kw):
        desc = packed(paged_cache._TREE, TREE, head_dim=head_dim, dtype=dtype, **kw)
        return _native.lib().tmw_paged_tree_attention_scratch_bytes(desc, scales(format=form))

    assert 0 < size(columns=1, batch=1) <= size(columns=100) <= size(columns=10000) == size(columns=1 << 20)
    assert size(batch=0) == size(heads=0) == size(nodes=0) == size(heads=3) == 0


def test_there_is_no_cpu_path():
    pages, table, pos = torch.zeros(4, 2, 16, 64), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        paged_read(pages, pages, table, pos, 3)
    with pytest.raises(RuntimeError):
        paged_tree_attention(torch.zeros(2, 2, 3, 64), pages, pages, table, pos, torch.zeros(2, 3, dtype=torch.int64))
    with pytest.raises(RuntimeError):
        paged_keep(pages, pages, table, pos, torch.zeros(2, 1, dtype=torch.int32), pos)


@pytest.mark.parametrize("nodes", [0, 1, 2, 3, 5, 17, 63, 64])
@pytest.mark.parametrize("window", [None, 0, 1, 3, 100])
def test_trees_are_walked_to_their_roots(nodes, window):
    g = torch.Generator().manual_seed(nodes)
    chain, bushy = list(range(-1, nodes - 1)), [max(-1, int(torch.randint(-2, max(i, 1), (), generator=g))) if i else -1 for i in range(nodes)]
    tree = draft_tree(torch.tensor([chain, bushy], dtype=torch.int64).view(2, nodes), torch.tensor([0, 1000], dtype=torch.int32), window)
    assert tree.seen.dtype == torch.int64 and tree.positions.dtype == torch.int32
    for row, (parents, start) in enumerate(((chain, 0), (bushy, 1000))):
        seen, depth = ancestors(parents)
        assert tree.positions[row].tolist() == [start + int(d) for d in depth]
        for i in range(nodes):
            bits = [j for j in range(nodes) if int(seen[i]) >> j & 1 and (window is None or depth[i] - depth[j] <= window)]
            assert [j for j in range(nodes) if int(tree.seen[row, i]) >> j & 1] == bits


def test_trees_that_are_none():
    start = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        draft_tree(torch.zeros(1, 65, dtype=torch.int64), start)
    with pytest.raises(ValueError):
        draft_tree(torch.zeros(4, dtype=torch.int64), start)
    with pytest.raises(ValueError):
        draft_tree(torch.zeros(1, 4), start)
    with pytest.raises(ValueError):
        draft_tree(torch.zeros(1, 4, dtype=torch.int64), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        draft_tree(torch.zeros(1, 4, dtype=torch.int64), start, -1)
    tree = draft_tree(torch.tensor([[0, 1, 9, -7]]), start)  # a node that is no earlier one is nobody's parent
    assert tree.seen.tolist() == [[1, 2, 4, 8]] and tree.positions.tolist() == [[0, 0, 0, 0]]
