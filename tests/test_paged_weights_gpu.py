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


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads,dh", [(8, 64), (1, 128), (16, 128), (4, 256)])
def test_long_sums_are_rounded_not_cut_off(heads, dh, dtype):
    """One key of value -1 against 65,000 of value 1 with as much weight together: the sum of the many passes through hundreds of
    additions in each warp, and what is left of the output, nearly nothing, shows what they lost.

    Relative to the weights A on either side: the scores are below 18 in powers of two and rounded three times, 3 * 18 * 2^-24 ln 2,
    the exponential is off by 2^-22; a tile's sum of at most six cut-off products by 8 * 2^-23; each of a warp's tiles is added with
    2^-24 of the sum before; joining parts costs 2^-22.  The output is half of the difference.  (All products cut off in one chain:
    6e-5 to 1.3e-4 towards the single key.)"""
    page, n, B, pages = 128, 65536, 384, 8
    g = torch.Generator().manual_seed(dh)
    k, v = torch.zeros(pages + 1, 1, page, dh, dtype=dtype), torch.ones(pages + 1, 1, page, dh, dtype=dtype)
    k[:pages, 0, :, 0] = (8 * torch.randn(pages, page, generator=g)).to(dtype)
    k[pages, 0, :, 0] = torch.tensor([64.0] + [-6e4] * (page - 1), dtype=dtype)
    v[pages, 0, 1:], v[pages, 0, 0] = 0, -1
    columns = torch.arange(n // page - 1) % pages
    many = k[:pages, 0, :, 0].double()[columns]

    def sides(scale):  # over e^(64 scale)
        return torch.exp((many - 64) * scale).sum().item()

    low, high = 0.01, 1.0
    for _ in range(60):
        low, high = ((low + high) / 2, high) if sides((low + high) / 2) > 1 else (low, (low + high) / 2)
    scale = torch.tensor(low, dtype=torch.float32).item()
    A = sides(scale)
    want = (A - 1) / (A + 1)
    assert abs(want) < 1e-5 and 64 * scale * math.log2(math.e) < 18
    q = torch.zeros(B, heads, dh, dtype=dtype)
    q[..., 0] = 1
    table = torch.cat((torch.tensor([pages]), columns)).to(torch.int32).expand(B, -1).contiguous()
    got = paged_attention(*[t.to(DEV) for t in (q, k, v, table)], torch.full((B,), n - 1, dtype=torch.int32, device=DEV), scale=scale)
    _native.poll_status(DEV)
    tiles = B * n / (16 if dh > 128 else 32) / torch.cuda.get_device_properties(DEV).multi_processor_count / 6  # of a warp, six to an SM
    allowed = 0.5 * (3 * 18 * 2.0 ** -24 * math.log(2) + 2 * 2.0 ** -22 + 8 * 2.0 ** -23 + tiles * 2.0 ** -24) + 1e-5 * torch.finfo(dtype).eps
    off = (got.double() - want).abs().max().item()
    assert off <= allowed + 2.0 ** -25, (off, allowed)


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("heads,dh", [(2, 64), (12, 64), (4, 256), (4, 40)])
@pytest.mark.parametrize("behind", [0.0, 5.0, 17.0, 25.0, 30.0, 60.0, 85.0])
def test_an_infinite_value_behind_the_largest_score(behind, heads, dh, dtype):
    """Its weight, e^-behind, is a normal number of fp32: the output is that infinity in its dimension, and nothing else changes.  A
    key of no weight at all, a score of -inf, makes it NaN (0 times infinity)."""
    n = 40
    k, v, table = pr.pool([n, n], 16, 1, dh, dtype, 3)
    q = torch.zeros(2, heads, dh, dtype=dtype)
    q[..., 0] = 1
    k[..., 0] = 0
    for t in (3, 21):  # one value in each direction, of different dimensions
        k[table[0, t // 16], 0, t % 16, 0] = -behind
        v[table[0, t // 16], 0, t % 16, t] = math.inf if t == 3 else -math.inf
    k[table[1, 0], 0, 7, 0] = -math.inf
    v[table[1, 0], 0, 7, 5] = math.inf
    got = paged_attention(*[t.to(DEV) for t in (q, k, v, table)], torch.full((2,), n - 1, dtype=torch.int32, device=DEV), scale=1.0)
    _native.poll_status(DEV)
    got = got.double().cpu()
    v[v.isinf()] = 0
    k[k.isinf()] = -1000  # (no weight in 64 bits either)
    want, bound = pr.attention(q, k, v, table, torch.tensor([n - 1] * 2), scale=1.0)
    assert (got[0, :, 3] == math.inf).all() and (got[0, :, 21] == -math.inf).all() and torch.isnan(got[1, :, 5]).all()
    got[0, :, [3, 21]], got[1, :, 5] = want[0, :, [3, 21]], want[1, :, 5]
    step = torch.finfo(dtype).eps / 2
    off = (got - want).abs()
    bound = 2 * v.double().abs().max() * (n + 8 + 85) * 2.0 ** -23  # (the scores are exact, their multiples below 85 / ln 2 rounded)
    assert (off <= bound + step * (want.abs() + bound)).all(), off.max()
