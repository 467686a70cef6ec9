"""What the C entries of the paged cache and of the token log-probabilities refuse on the host, before anything is launched, and
the layout of the descriptions that the package packs for them."""

import os
import subprocess
import tempfile

import pytest

from conftest import ROOT
from titanmac_b200 import _native, logprobs, paged_cache

OK, BAD, UNSUPPORTED, LARGE = (_native.TMW_OK, _native.TMW_ERR_INVALID_ARGUMENT, _native.TMW_ERR_UNSUPPORTED, _native.TMW_ERR_TOO_LARGE)
FAKE = 0x1000  # never dereferenced: validation fails first

PAGES = dict(dtype=1, batch=2, kv_heads=2, head_dim=64, page_size=16, pages=8, columns=4, reserved=0, table_stride=4, k_pages=FAKE,
             v_pages=FAKE, page_table=FAKE)
APPEND = dict(PAGES, rows=3, heads=4, rotated=64, interleaved=0, k=FAKE, v=FAKE, q=FAKE, q_out=FAKE,
              **{f"{n}{i}": 64 for n in ("ks", "vs", "qs", "os") for i in range(3)}, start=FAKE, counts=0, inv_freq=FAKE)
ATTENTION = dict(PAGES, heads=4, n_persistent=1, window=-1, scale=0.0, q=FAKE, k_pers=FAKE, v_pers=FAKE, o=0x2000, qs0=64, qs1=64,
                 os0=64, os1=64, pos=FAKE)
LOGPROBS = dict(dtype=1, batch=2, tokens=3, vocab=100, top=4, reserved=0, logits=FAKE, s0=300, s1=100, targets=FAKE, logprobs=FAKE,
                entropy=FAKE, lse=FAKE, top_logprobs=FAKE, top_ids=FAKE)


def packed(layout, fields, **changes):
    assert set(changes) <= set(fields)
    return layout.pack(*{**fields, **changes}.values())


def test_layouts_match_the_header():
    src = r"""
    #include <stdio.h>
    #include <stddef.h>
    #include "tmw.h"
    int main(void) {
        printf("%zu %zu %zu\n", sizeof(tmw_paged_append_desc), sizeof(tmw_paged_attention_desc), sizeof(tmw_logprobs_desc));
        printf("%zu %zu %zu %zu\n", offsetof(tmw_pages, table_stride), offsetof(tmw_paged_append_desc, k),
               offsetof(tmw_paged_append_desc, k_stride), offsetof(tmw_paged_append_desc, start));
        printf("%zu %zu %zu\n", offsetof(tmw_paged_attention_desc, scale), offsetof(tmw_paged_attention_desc, o),
               offsetof(tmw_paged_attention_desc, pos));
        printf("%zu %zu %zu\n", offsetof(tmw_logprobs_desc, stride), offsetof(tmw_logprobs_desc, logprobs), offsetof(tmw_logprobs_desc, top_ids));
        return 0;
    }
    """
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "t.c"), os.path.join(d, "t")
        open(c, "w").write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        lines = [[int(v) for v in line.split()] for line in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines()]
    assert lines[0] == [paged_cache._APPEND.size, paged_cache._ATTENTION.size, logprobs._DESC.size]

    def at(layout, fields, name):  # where a mark put into the field comes out
        zeros = layout.pack(*[0] * len(fields))
        marked = layout.pack(*[(1 if n == name else 0) for n in fields])
        return next(i for i in range(len(zeros)) if zeros[i] != marked[i])

    assert lines[1] == [at(paged_cache._APPEND, APPEND, n) for n in ("table_stride", "k", "ks0", "start")]
    scale = next(i for i, (a, b) in enumerate(zip(packed(paged_cache._ATTENTION, ATTENTION), packed(paged_cache._ATTENTION, ATTENTION, scale=1.0)))
                 if a != b) // 4 * 4
    assert lines[2] == [scale] + [at(paged_cache._ATTENTION, ATTENTION, n) for n in ("o", "pos")]
    assert lines[3] == [at(logprobs._DESC, LOGPROBS, n) for n in ("s0", "logprobs", "top_ids")]


PAGES_REFUSED = [(dict(dtype=7), UNSUPPORTED), (dict(head_dim=12), UNSUPPORTED), (dict(head_dim=264), UNSUPPORTED), (dict(batch=-1), BAD),
                 (dict(kv_heads=0), BAD), (dict(page_size=0), BAD), (dict(pages=-1), BAD), (dict(columns=-1), BAD), (dict(table_stride=-4), BAD),
                 (dict(columns=1 << 27), LARGE), (dict(batch=70000), LARGE), (dict(k_pages=0), BAD), (dict(v_pages=0x1008), BAD),
                 (dict(page_table=0), BAD)]


@pytest.mark.parametrize("change,status", PAGES_REFUSED + [
    (dict(rows=-1), BAD), (dict(heads=-1), BAD), (dict(heads=70000), LARGE), (dict(rotated=63), BAD), (dict(rotated=66), BAD), (dict(k=0), BAD),
    (dict(v=0), BAD), (dict(q=0), BAD), (dict(q_out=0), BAD), (dict(start=0), BAD), (dict(inv_freq=0), BAD), (dict(k=0x1001), BAD), (dict(ks1=-64), BAD),
    (dict(os2=-1), BAD)])
def test_append_refuses(change, status):
    assert _native.lib().tmw_paged_append(packed(paged_cache._APPEND, APPEND, **change), None) == status


@pytest.mark.parametrize("change,status", PAGES_REFUSED + [
    (dict(heads=3), BAD), (dict(heads=-2), BAD), (dict(n_persistent=-1), BAD), (dict(window=-2), BAD), (dict(scale=-1.0), BAD),
    (dict(scale=float("nan")), BAD), (dict(heads=70000), LARGE), (dict(n_persistent=1 << 25), LARGE), (dict(q=0), BAD), (dict(o=0), BAD),
    (dict(pos=0), BAD), (dict(k_pers=0), BAD), (dict(v_pers=0x1008), BAD), (dict(q=0x1001), BAD), (dict(qs1=-1), BAD), (dict(os0=-1), BAD),
    (dict(o=FAKE), BAD)])
def test_attention_refuses(change, status):
    lib, desc = _native.lib(), packed(paged_cache._ATTENTION, ATTENTION, **change)
    assert lib.tmw_paged_attention(desc, FAKE, 1 << 30, None) == status


def test_attention_refuses_its_scratch():
    lib, desc = _native.lib(), packed(paged_cache._ATTENTION, ATTENTION)
    assert lib.tmw_paged_attention(desc, None, 1 << 30, None) == BAD
    assert lib.tmw_paged_attention(desc, 0x1008, 1 << 30, None) == BAD
    assert lib.tmw_paged_attention(None, FAKE, 1 << 30, None) == BAD
    assert lib.tmw_paged_attention_scratch_bytes(packed(paged_cache._ATTENTION, ATTENTION, heads=3)) == 0


@pytest.mark.parametrize("change,status", [
    (dict(dtype=3), UNSUPPORTED), (dict(batch=-1), BAD), (dict(tokens=-1), BAD), (dict(vocab=0), BAD), (dict(top=-1), BAD), (dict(top=33), LARGE),
    (dict(vocab=3), BAD), (dict(vocab=(1 << 26) + 1), LARGE), (dict(batch=1 << 20, tokens=1 << 10), LARGE), (dict(logits=0), BAD),
    (dict(targets=0), BAD), (dict(entropy=0), BAD), (dict(s0=-1), BAD), (dict(s1=-1), BAD), (dict(logits=0x1001), BAD)])
def test_logprobs_refuse(change, status):
    lib, desc = _native.lib(), packed(logprobs._DESC, LOGPROBS, **change)
    assert lib.tmw_token_logprobs(desc, None) == status
    assert lib.tmw_token_logprobs_backward(desc, FAKE, FAKE, FAKE, 0x2000, logprobs._STRIDES.pack(300, 100), None) == status


def test_logprobs_refuse_their_outputs():
    lib, strides = _native.lib(), logprobs._STRIDES.pack(300, 100)
    for change in (dict(logprobs=0), dict(top_ids=0), dict(top_logprobs=0)):
        assert lib.tmw_token_logprobs(packed(logprobs._DESC, LOGPROBS, **change), None) == BAD
    back = lib.tmw_token_logprobs_backward
    desc = packed(logprobs._DESC, LOGPROBS)
    assert back(packed(logprobs._DESC, LOGPROBS, lse=0), FAKE, FAKE, FAKE, 0x2000, strides, None) == BAD
    assert back(desc, FAKE, FAKE, FAKE, None, strides, None) == BAD
    assert back(desc, FAKE, FAKE, FAKE, FAKE, strides, None) == BAD  # in place
    assert back(desc, FAKE, FAKE, FAKE, 0x2000, None, None) == BAD
    assert back(desc, FAKE, FAKE, FAKE, 0x2000, logprobs._STRIDES.pack(-1, 100), None) == BAD
    assert back(packed(logprobs._DESC, LOGPROBS, top_ids=0), FAKE, FAKE, FAKE, 0x2000, strides, None) == BAD


def test_nothing_to_do_is_fine():
    lib = _native.lib()
    nothing = dict(k_pages=0, v_pages=0, page_table=0)
    assert lib.tmw_paged_append(packed(paged_cache._APPEND, APPEND, batch=0, **nothing), None) == OK
    assert lib.tmw_paged_append(packed(paged_cache._APPEND, APPEND, rows=0, **nothing), None) == OK
    assert lib.tmw_paged_attention(packed(paged_cache._ATTENTION, ATTENTION, batch=0, **nothing), None, 0, None) == OK
    assert lib.tmw_paged_attention(packed(paged_cache._ATTENTION, ATTENTION, heads=0, **nothing), None, 0, None) == OK
    assert lib.tmw_token_logprobs(packed(logprobs._DESC, LOGPROBS, batch=0, logits=0), None) == OK
    assert lib.tmw_token_logprobs(packed(logprobs._DESC, LOGPROBS, tokens=0, logits=0), None) == OK


def test_there_is_no_cpu_path():
    import torch

    from titanmac_b200 import PagedCache, paged_append, paged_attention, token_logprobs

    pages, table, pos = torch.zeros(4, 2, 16, 64), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    k = torch.zeros(2, 2, 1, 64)
    with pytest.raises(RuntimeError):
        paged_append(k, k, pages, pages, table, pos)
    with pytest.raises(RuntimeError):
        paged_attention(k[:, :, 0], pages, pages, table, pos)
    with pytest.raises(RuntimeError):
        PagedCache(table, 4, 16, 2, 64, None, 0, torch.float32)
    with pytest.raises(RuntimeError):
        token_logprobs(torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64))


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("head_dim", [8, 64, 96, 128, 200, 256])
def test_attention_scratch_grows_with_the_work_up_to_the_gpu(head_dim, dtype):
    def size(**kw):
        desc = packed(paged_cache._ATTENTION, ATTENTION, head_dim=head_dim, dtype=dtype, **kw)
        return _native.lib().tmw_paged_attention_scratch_bytes(desc)

    assert 0 < size(columns=1, batch=1) <= size(columns=100) <= size(columns=10000) == size(columns=1 << 20)
    assert size(columns=10000, window=20) <= size(columns=10000)
    assert size(batch=0) == size(heads=0) == 0
