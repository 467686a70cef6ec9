"""Forward-mode derivatives: refused by the calls that have none, instead of lost."""

import pytest
import torch
from torch.autograd import forward_ad

from titanmac_b200 import PagedCache, _native, paged_append, paged_attention, token_logprobs

DEV = torch.device("cuda:0")


def test_tangents_are_found():
    x = torch.zeros(3)
    _native.refuse_tangents("call", x, None)
    with forward_ad.dual_level():
        _native.refuse_tangents("call", x, None)
        with pytest.raises(NotImplementedError):
            _native.refuse_tangents("call", x, forward_ad.make_dual(x, torch.ones(3)))
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda t: (_native.refuse_tangents("call", t), t)[1], (x,), (torch.ones(3),))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_logprobs(dtype):
    x, y = torch.randn(4, 50, device=DEV).to(dtype), torch.randint(0, 50, (4,), device=DEV)
    want = token_logprobs(x, y, 3)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            token_logprobs(forward_ad.make_dual(x, torch.ones_like(x)), y)
        with pytest.raises(NotImplementedError):
            token_logprobs(forward_ad.make_dual(x.clone().requires_grad_(True), torch.ones_like(x)), y)
        assert torch.equal(token_logprobs(x, y, 3).logprobs, want.logprobs)  # nothing to lose
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda t: token_logprobs(t, y).logprobs, (x,), (torch.ones_like(x),))


@pytest.mark.gpu
def test_paged_calls():
    table, at = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    cache = PagedCache(table, 1, 16, 2, 64, None, 0, torch.float32)
    k = torch.randn(1, 2, 1, 64, device=DEV)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(k, torch.ones_like(k))
        for args in ((dual, k), (k, dual)):
            with pytest.raises(NotImplementedError):
                paged_append(*args, cache.k_pages, cache.v_pages, table, at)
        with pytest.raises(NotImplementedError):
            paged_append(k, k, cache.k_pages, cache.v_pages, table, at, q=dual)
        assert (cache.k_pages == 0).all()
        with pytest.raises(NotImplementedError):
            paged_attention(dual[:, :, 0], cache.k_pages, cache.v_pages, table, at)
    cache.append(k, k, at)
    assert torch.equal(cache.attend(k[:, :, 0], at), k[:, :, 0])
