"""Paged attention where many heads read one key head, and where sequences read the same pages."""

import pytest
import torch

import paged_reference as pr
from titanmac_b200 import _native, paged_append, paged_attention
from test_paged_cache_gpu import attend, check, dev, numbers

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("dh", [32, 64, 80, 96, 192, 256])
@pytest.mark.parametrize("heads,kv_heads", [(9, 1), (16, 1), (33, 1), (22, 2)])
def test_nine_heads_and_more_on_one(heads, kv_heads, dh, dtype):
    check(*attend([70, 1, 45, 0, 300], heads, kv_heads, dh, 16, dtype, window=200, n_p=3, seed=heads + dh))


@pytest.mark.parametrize("dtype", [BF, HF, FF])
def test_sequences_that_share_a_prefix(dtype):
    """Whole pages of one prefix under five sequences, each with pages of its own behind it: a step of all of them at once is what
    each is alone, and the shared pages stay as they are."""
    page, KV, dh, H, prefix = 16, 2, 64, 6, 48
    g = torch.Generator().manual_seed(4)
    lengths = [48, 49, 60, 75, 130]  # the new token is the last of each
    columns = [-(-n // page) for n in lengths]
    pages = 3 + sum(c - 3 for c in columns) + 2
    order = torch.randperm(pages, generator=g).tolist()
    shared, free = order[:3], order[3:]
    table = torch.full((5, max(columns)), -9, dtype=torch.int32)
    for b, c in enumerate(columns):
        table[b, :c] = torch.tensor(shared + [free.pop() for _ in range(c - 3)])
    k, v = (torch.randn(pages, KV, page, dh, generator=g).to(dtype) for _ in range(2))
    q, new_k, new_v = (torch.randn(5, heads, dh, generator=g).to(dtype) for heads in (H, KV, KV))
    k_dev, v_dev, table_dev = dev(k, v, table)
    start = [-1] + [n - 1 for n in lengths[1:]]  # (the first has nothing but the prefix)
    paged_append(*dev(new_k[:, :, None], new_v[:, :, None]), k_dev, v_dev, table_dev, numbers(start))
    pos = torch.tensor(lengths) - 1
    got = paged_attention(q.to(DEV), k_dev, v_dev, table_dev, numbers(pos.tolist()))
    _native.poll_status(DEV)
    for b, n in enumerate(lengths[1:], 1):
        k[table[b, (n - 1) // page], :, (n - 1) % page], v[table[b, (n - 1) // page], :, (n - 1) % page] = new_k[b], new_v[b]
    assert torch.equal(k_dev.cpu(), k) and torch.equal(v_dev.cpu(), v)
    check(got, *pr.attention(q, k, v, table, pos))
    for b in range(5):
        alone = paged_attention(q[b:b + 1].to(DEV), k_dev, v_dev, table_dev[b:b + 1], numbers([lengths[b] - 1]))
        check(alone, *(t[b:b + 1] for t in pr.attention(q, k, v, table, pos)))


@pytest.mark.parametrize("dtype", [BF, HF, FF])
def test_one_page_named_many_times(dtype):
    """Every column of every sequence names the same page: nothing but reads."""
    page, dh = 8, 96
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(1, 1, page, dh, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(3, 4, dh, generator=g).to(dtype)
    table, pos = torch.zeros(3, 40, dtype=torch.int32), torch.tensor([7, 133, 319])
    got = paged_attention(*dev(q, k, v, table), numbers(pos.tolist()))
    check(got, *pr.attention(q, k, v, table, pos))
