"""Gradients of token log-probabilities for views of logits: rows that begin at other places of their vectors than the gradient's."""

import pytest
import torch

from titanmac_b200 import _native, logprobs, token_logprobs

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32

VIEWS = {
    "all_but_the_last": lambda t: t[:, :-1],
    "behind_the_first": lambda t: t[:, 1:],
    "of_part_of_the_ids": lambda t: t[:, :, 3:],
    "every_other": lambda t: t[:, ::2, 1:],
    "one_row_each": lambda t: t[:, 2],
}


def wanted(x, y, ids, g, h, a):
    """``(gradient, bound)`` in 64 bits.  The bound: log p is off by 100 * 2^-23 of its differences and chains of 512 sums, an
    exponential by 2^-21, which p carries with what it is multiplied by - all incoming gradients, and for the entropy's log p + H,
    off by three times that."""
    lp = torch.log_softmax(x.double(), -1)
    p = lp.exp()
    seen = torch.where(p > 0, lp, 0.0)
    H = -(p * seen).sum(-1, keepdim=True)
    incoming = torch.zeros_like(p)
    if a is not None:
        incoming.scatter_add_(-1, ids, a.double())
    counted = y >= 0
    incoming.scatter_add_(-1, y.clamp(0)[..., None], torch.where(counted, g.double(), 0.0)[..., None])
    h = torch.zeros_like(H) if h is None else h.double()[..., None]
    want = incoming - p * (incoming.sum(-1, keepdim=True) + h * (seen + H))
    most = 100 * 2.0 ** -23 + 512 * 2.0 ** -24 + 2.0 ** -21
    bound = p * (incoming.abs().sum(-1, keepdim=True) * (most + 34 * 2.0 ** -24) + h.abs() * (seen.abs() + H) * 4 * most) \
        + 2.0 ** -21 * incoming.abs()
    return want, bound


def held(got, want, bound):
    rounding = torch.finfo(got.dtype).eps / 2 if got.dtype != FF else 2.0 ** -23
    off = (got.double() - want).abs()
    allowed = bound + rounding * (want.abs() + bound) + (2.0 ** -24 if got.dtype == HF else 2.0 ** -126)
    assert (off <= allowed).all(), (off / allowed).max().item()


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("view", list(VIEWS))
@pytest.mark.parametrize("V", [37, 5003, 40001])
@pytest.mark.parametrize("n_top,entropy", [(0, False), (0, True), (6, False), (32, True)])
def test_views(n_top, entropy, V, view, dtype):
    gen = torch.Generator(device=DEV).manual_seed(V)
    whole = (3 * torch.randn(3, 5, V, generator=gen, device=DEV)).to(dtype)
    whole[..., V - 4:] = -float("inf")
    with torch.enable_grad():
        leaf = whole.clone().requires_grad_(True)
        x = VIEWS[view](leaf)
        rows = x.shape[:-1]
        y = torch.randint(0, x.shape[-1] - 4, rows, generator=gen, device=DEV)
        y.view(-1)[0] = -100
        out = token_logprobs(x, y, n_top)
        g = torch.randn(rows, generator=gen, device=DEV)
        h = torch.randn(rows, generator=gen, device=DEV) if entropy else None
        a = torch.randn(*rows, n_top, generator=gen, device=DEV) if n_top else None
        pairs = [(o, d) for o, d in ((out.logprobs, g), (out.entropy, h), (out.top_logprobs, a)) if d is not None]
        (got,) = torch.autograd.grad([o for o, _ in pairs], leaf, [d for _, d in pairs])
    _native.poll_status(DEV)
    held(VIEWS[view](got), *wanted(VIEWS[view](whole), y, out.top_ids, g, h, a))
    outside = torch.ones_like(whole, dtype=torch.bool)
    VIEWS[view](outside)[...] = False
    assert (got[outside] == 0).all()


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("n_top,entropy", [(0, False), (32, False), (5, True), (32, True)])
@pytest.mark.parametrize("shift", [0, 1, 5])
def test_the_entry_writes_rows_anywhere_and_nothing_else(shift, n_top, entropy, dtype):
    """tmw_token_logprobs_backward into rows further apart than they are long, at the logits' places of their vectors or others."""
    gen = torch.Generator(device=DEV).manual_seed(n_top)
    B, T, V = 2, 3, 4999
    x = (3 * torch.randn(B, T, V, generator=gen, device=DEV)).to(dtype)
    y = torch.randint(0, V, (B, T), generator=gen, device=DEV)
    lp, H, ids, _, lse = logprobs._forward(x, y, n_top, True)
    g, h = (torch.randn(B, T, generator=gen, device=DEV) for _ in range(2))
    a = torch.randn(B, T, n_top, generator=gen, device=DEV) if n_top else None
    buffer = torch.full((B, T + 1, V + 17), 7.0, dtype=dtype, device=DEV)
    d = buffer[:, 1:, shift:shift + V]
    desc = logprobs._DESC.pack(_native._DTYPES[dtype], B, T, V, n_top, 0, x.data_ptr(), *x.stride()[:2], y.data_ptr(), 0, H.data_ptr(),
                               lse.data_ptr(), 0, ids.data_ptr() if n_top else 0)
    _native.launch(0, _native.lib().tmw_token_logprobs_backward, desc, g.data_ptr(), h.data_ptr() if entropy else None,
                   a.data_ptr() if n_top else None, d.data_ptr(), logprobs._STRIDES.pack(*d.stride()[:2]))
    _native.poll_status(DEV)
    held(d, *wanted(x, y, ids, g, h if entropy else None, a))
    d.fill_(7.0)
    assert (buffer == 7).all()
