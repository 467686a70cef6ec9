"""The weights of paged attention: how many bits they have, and where infinite values meet small ones."""

import math

import pytest
import torch

import paged_reference as pr
from titanmac_b200 import _native, paged_attention

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


def attend(q, k, v, table, pos):
    got = paged_attention(*[t.to(DEV) for t in (q, k, v, table)], pos.to(torch.int32).to(DEV))
    _native.poll_status(DEV)
    return got


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("heads,kv_heads,dh", [(8, 1, 64), (2, 2, 32), (16, 1, 128), (4, 1, 256), (12, 1, 64)])
def test_weights_are_held_in_32_bits(heads, kv_heads, dh, dtype):
    """Two keys of nearly equal scores whose values cancel: what is left of the output, tanh(d / 2) of scores d apart, shows what
    the weights lost.  d is below 2^-13, so the output's own rounding is below 2^-22 in every type, and the bound of an fp32
    evaluation is 2 (2 + 8) 2^-23 and next to nothing for the score (its one product, of numbers of 8 bits, is exact); a weight of
    16 bits is off by up to 2^-17 here, the output by half of that."""
    B, page = 64, 16
    k, v, table = pr.pool([2] * B, page, kv_heads, dh, dtype, 1)
    g = torch.Generator().manual_seed(dh + heads)
    q = torch.zeros(B, heads, dh, dtype=dtype)
    q[..., 5] = (1 + torch.randint(0, 128, (B, heads), generator=g) / 128.0).to(dtype)
    k[...] = 0
    k[:, :, 1, 5] = -(2.0 ** (math.ceil(math.log2(dh) / 2) - 15))
    v[:, :, 0], v[:, :, 1] = 1, -1
    pos = torch.ones(B, dtype=torch.int64)
    got = attend(q, k, v, table, pos)
    want, bound = pr.attention(q, k, v, table, pos)
    assert want.min() > 0 and want.max() < 2.0 ** -14
    step = torch.finfo(dtype).eps / 2 if dtype != FF else 0.0
    allowed = bound + step * (want + bound) + (2.0 ** -25 if dtype == HF else 0.0)  # (fp16 has steps of 2^-24 below 2^-14)
    off = (got.double().cpu() - want).abs()
    assert (off <= allowed).all(), (off / allowed).max().item()
