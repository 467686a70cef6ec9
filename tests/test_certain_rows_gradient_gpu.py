"""The gradient of token log-probabilities where one id has nearly all of a row: what is left of 1 - p keeps its digits."""

import math

import pytest
import torch

from titanmac_b200 import _native, token_logprobs

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


def certain_rows(rows, V, dtype):
    """Logits and, for every row, the id that is ahead of all others: by e^8 to e^20 of all of them together."""
    g = torch.Generator(device=DEV).manual_seed(V + rows)
    x = (2 * torch.randn(rows, V, generator=g, device=DEV)).to(dtype)
    c = torch.randint(0, V, (rows,), generator=g, device=DEV)
    ahead = torch.linspace(8.0, 20.0, rows, device=DEV) + math.log(V)
    x.scatter_(1, c[:, None], (x.float().amax(-1) + ahead).to(dtype)[:, None])
    return x, c, g


def expected(x, c, ids, a, y, g, h):
    """``(gradient, bound on an fp32 evaluation's error)`` in 64 bits, with 1 - p of the id ahead from the others' weights, never by
    a subtraction.

    The bound: a log-probability's argument is below 100 and a sum has chains of at most 512, so the rest of the row, log p of the id
    ahead and the other ids' probabilities are off by `most` of themselves, the entropy by twice that; e^d - 1 and 2^d by 2^-21 with
    what they are multiplied by; 33 incoming gradients are added with 2^-24 each."""
    x, rows = x.double(), torch.arange(x.shape[0], device=DEV)
    d = x - x[rows, c][:, None]
    w = torch.exp(d)
    w[rows, c] = 0
    rest = w.sum(-1, keepdim=True)
    log_s = torch.log1p(rest)
    p = w / (1 + rest)
    H = log_s + (p * -d).sum(-1, keepdim=True)
    log_p = d - log_s
    incoming = torch.zeros_like(x)
    if a is not None:
        incoming.scatter_add_(1, ids, a.double())
    counted = y >= 0
    incoming[rows[counted], y[counted]] += g[counted].double()
    h = torch.zeros_like(rest) if h is None else h.double()[:, None]
    total, size = incoming.sum(-1, keepdim=True), incoming.abs().sum(-1, keepdim=True)
    want = incoming - p * (total + h * (log_p + H))
    most, u = 100 * 2.0 ** -23 + 512 * 2.0 ** -24 + 2.0 ** -21, 2.0 ** -21
    spread = h.abs() * (log_p.abs() + H)
    bound = u * incoming.abs() + p * (size * (most + u + 34 * 2.0 ** -24) + spread * (3 * most + u))
    mine = incoming[rows, c][:, None]
    others = incoming.clone()
    others[rows, c] = 0
    of_others = others.sum(-1, keepdim=True)
    p_c, lp_c = 1 / (1 + rest), -log_s
    want[rows, c] = (mine * rest * p_c - p_c * (of_others + h * (lp_c + H)))[:, 0]
    bound[rows, c] = (mine.abs() * rest * (most + u) + others.abs().sum(-1, keepdim=True) * (34 * 2.0 ** -24 + u)
                      + h.abs() * (lp_c.abs() + H) * (2 * most + u))[:, 0]
    return want, bound


@pytest.mark.parametrize("dtype", [FF, BF, HF])
@pytest.mark.parametrize("rows,V", [(5, 60), (3, 40000), (1, 128000), (2000, 900), (900, 5000)])
@pytest.mark.parametrize("kind,n_top", [("target", 0), ("target", 5), ("target", 32), ("likely", 5), ("likely", 32), ("target_and_likely", 4),
                                        ("elsewhere", 3), ("elsewhere", 32), ("entropy", 0), ("all", 7), ("all", 32)])
def test_the_gradient_of_the_id_ahead(kind, n_top, rows, V, dtype):
    x, c, gen = certain_rows(rows, V, dtype)
    y = c if kind in ("target", "target_and_likely", "entropy", "all") else torch.full_like(c, -100)
    if kind == "elsewhere":  # the id ahead is a likely one, the target another
        y = (c + 7) % V
    g = torch.randn(rows, generator=gen, device=DEV)
    a = h = None
    if kind != "target" and n_top:
        a = torch.randn(rows, n_top, generator=gen, device=DEV)
        if kind != "all":
            a[:, 1:] = 0
    if kind in ("entropy", "all"):
        h = torch.randn(rows, generator=gen, device=DEV)
    with torch.enable_grad():
        logits = x.clone().requires_grad_(True)
        out = token_logprobs(logits, y, n_top)
        outputs, grads = [out.logprobs], [g]
        if a is not None:
            outputs.append(out.top_logprobs), grads.append(a)
        if h is not None:
            outputs.append(out.entropy), grads.append(h)
        (got,) = torch.autograd.grad(outputs, logits, grads)
    _native.poll_status(DEV)
    if n_top:
        assert torch.equal(out.top_ids[:, 0], c)
    want, bound = expected(x, c, out.top_ids, a, y, g, h)
    rounding = torch.finfo(dtype).eps / 2 if dtype != FF else 2.0 ** -23
    least = {FF: 2.0 ** -126, BF: 2.0 ** -126, HF: 2.0 ** -24}[dtype]  # (what a type or the exponential flushes to zero)
    off = (got.double() - want).abs()
    allowed = bound + rounding * (want.abs() + bound) + least
    assert (off <= allowed).all(), (off / allowed).max().item()


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("rows,V,n_top", [(7, 1001, 5), (300, 8003, 0), (3, 40003, 32)])
def test_ordinary_rows_without_the_entropys_share(rows, V, n_top, dtype):
    """Gradients of log-probabilities alone, against the formula: none of what the entropy's factor, log p + H, allows."""
    gen = torch.Generator(device=DEV).manual_seed(V)
    x = (3 * torch.randn(rows, V, generator=gen, device=DEV)).to(dtype)
    y = torch.randint(0, V, (rows,), generator=gen, device=DEV)
    g = torch.randn(rows, generator=gen, device=DEV)
    with torch.enable_grad():
        logits = x.clone().requires_grad_(True)
        out = token_logprobs(logits, y, n_top)
        a = torch.randn(rows, n_top, generator=gen, device=DEV) if n_top else None
        (got,) = torch.autograd.grad([out.logprobs] + ([out.top_logprobs] if n_top else []), logits, [g] + ([a] if n_top else []))
    p = torch.softmax(x.double(), -1)
    incoming = torch.zeros_like(p).scatter_add_(1, y[:, None], g.double()[:, None])
    if n_top:
        incoming.scatter_add_(1, out.top_ids, a.double())
    want = incoming - p * incoming.sum(-1, keepdim=True)
    # log p is off by 100 * 2^-23 of its differences, the sum by chains of 512, the exponential by 2^-21, as is p of itself
    most = 100 * 2.0 ** -23 + 512 * 2.0 ** -24 + 2.0 ** -21
    bound = p * incoming.abs().sum(-1, keepdim=True) * (most + 34 * 2.0 ** -24) + 2.0 ** -22 * incoming.abs()
    rounding = torch.finfo(dtype).eps / 2 if dtype != FF else 2.0 ** -23
    off = (got.double() - want).abs()
    allowed = bound + rounding * (want.abs() + bound) + (2.0 ** -24 if dtype == HF else 2.0 ** -126)
    assert (off <= allowed).all(), (off / allowed).max().item()
