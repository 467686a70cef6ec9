"""Outputs that have no places of their own are refused on the host: rows that lie on one another, a buffer that is an input under
other strides."""

import pytest
import torch

from titanmac_b200 import _native, logprobs, paged_append, paged_cache
from test_operator_refusals import APPEND, ATTENTION, BAD, FAKE, LOGPROBS, packed


@pytest.mark.parametrize("change", [dict(os0=0), dict(os1=0), dict(os2=0), dict(os0=128), dict(qs2=128), dict(q_out=0x2000, os1=0)])
def test_append(change):
    assert _native.lib().tmw_paged_append(packed(paged_cache._APPEND, APPEND, **change), None) == BAD


@pytest.mark.gpu
def test_append_in_place_of_one_row_asks_nothing_of_its_stride():
    dev = torch.device("cuda:0")
    k, q = torch.randn(2, 2, 1, 64, device=dev), torch.randn(2, 4, 1, 64, device=dev)
    pages, table = torch.zeros(2, 2, 16, 64, device=dev), torch.tensor([[0], [1]], dtype=torch.int32, device=dev)
    at, inv_freq = torch.tensor([3, 5], dtype=torch.int32, device=dev), torch.linspace(0, 1, 32, device=dev)
    want = paged_append(k, k, pages, pages.clone(), table, at, q=q.clone(), inv_freq=inv_freq)
    got = paged_append(k, k, pages, pages.clone(), table, at, q=q, q_out=q.as_strided(q.shape, (256, 64, 999, 1)), inv_freq=inv_freq)
    _native.poll_status(dev)
    assert torch.equal(got, want) and torch.equal(q, want)


@pytest.mark.parametrize("change", [dict(os0=0), dict(os1=0)])
def test_attention(change):
    desc = packed(paged_cache._ATTENTION, ATTENTION, **change)
    assert _native.lib().tmw_paged_attention(desc, FAKE, 1 << 30, None) == BAD


@pytest.mark.parametrize("strides", [(0, 100), (300, 0)])
def test_the_gradient_of_logprobs(strides):
    back = _native.lib().tmw_token_logprobs_backward
    assert back(packed(logprobs._DESC, LOGPROBS), FAKE, FAKE, FAKE, 0x2000, logprobs._STRIDES.pack(*strides), None) == BAD
