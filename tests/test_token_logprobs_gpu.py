"""Token log-probabilities, entropy and alternatives against 64 bits, and their gradients against the formula and differences."""

import math

import pytest
import torch

from titanmac_b200 import TitanMAC, TitanMACConfig, _native, token_logprobs

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32
INF = float("inf")


@pytest.fixture(autouse=True)
def _grad_mode():
    _native.poll_status(DEV)
    with torch.enable_grad():  # (other tests may have turned it off)
        yield


def reference(x, y, n_top):
    """In 64 bits: logprobs, entropy, ids, their log-probabilities; rows without a distribution have NaN and -1."""
    x = x.double()
    logp = torch.log_softmax(x, -1)
    fine = ~torch.isnan(logp).any(-1)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, torch.where(torch.isnan(p), p, 0.0)).sum(-1)
    picked = logp.gather(-1, y.clamp(0)[..., None])[..., 0]
    picked = torch.where(y == -100, 0.0, picked)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :n_top]
    top = logp.gather(-1, order)
    return picked, entropy, torch.where(fine[..., None], order, -1), top, logp


def allowed(x, want):
    """fp32 sums of V terms in chains of at most 512, exponentials to 2^-22 and their arguments to 2^-23 of a difference that
    matters only down to -100: what a log-probability, or the entropy, is off by at most."""
    return (want.abs() + 100.0) * 2.0 ** -23 + (512 + 16) * 2.0 ** -24 + 2.0 ** -21


def run(x, y, n_top=0):
    with torch.no_grad():
        return token_logprobs(x, y, n_top)


def check(x, y, n_top):
    got = run(x, y, n_top)
    picked, entropy, ids, top, _ = reference(x, y, n_top)
    for a, b in ((got.logprobs, picked), (got.entropy, entropy)) + (((got.top_logprobs, top),) if n_top else ()):
        assert a.dtype == FF and a.shape == b.shape
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.isinf(a), torch.isinf(b))
        ok = torch.isfinite(b)
        assert ((a.double() - b)[ok].abs() <= allowed(x, b[ok])).all(), (a.double() - b)[ok].abs().max()
    if n_top:
        assert torch.equal(got.top_ids, ids)
    else:
        assert got.top_ids is None and got.top_logprobs is None


def data(rows, V, dtype, seed=0, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed + V)
    x = (torch.randn(*rows, V, generator=g, device=DEV) * spread).to(dtype)
    return x, torch.randint(0, V, rows, generator=g, device=DEV)


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("rows,V,n_top", [
    ((1,), 1, 1), ((3,), 2, 2), ((5, 2), 7, 5), ((), 50, 3), ((4,), 33, 32), ((2, 3), 1000, 20), ((2, 3, 2), 4099, 32),
    ((700,), 2048, 5), ((3,), 20001, 32), ((1,), 128000, 20), ((300,), 5003, 0),
])
def test_against_64_bits(rows, V, n_top, dtype):
    x, y = data(rows, V, dtype)
    check(x, y, n_top)
    _native.poll_status(DEV)


@pytest.mark.parametrize("dtype", [BF, FF])
def test_rows_at_any_address(dtype):
    """Views whose rows begin anywhere in a vector, further apart than their length, or all at one place."""
    whole, _ = data((3, 9), 1200, dtype)
    for x in (whole[:, 1:, 5:1000], whole[:, ::2, 3:], whole[1, :, 1:8], whole[:1].expand(4, -1, -1)[..., 7:], whole.transpose(0, 1)[..., 2:],
              whole.transpose(1, 2)):
        y = torch.randint(0, x.shape[-1], x.shape[:-1], device=DEV)
        check(x, y, min(6, x.shape[-1]))


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("V", [5, 700, 9001, 70001])
@pytest.mark.parametrize("kind", ["equal", "few_values", "rising", "falling", "one_thread", "zeros", "masked", "mostly_masked", "lowest"])
def test_alternatives_in_order(kind, V, dtype):
    """Ties go to the lower id, wherever the likely ids stand."""
    x, y = data((3,), V, dtype)
    if kind == "equal":
        x[:] = 1.5
    elif kind == "few_values":
        x = (x * 0.3).round()
    elif kind == "rising":
        x = torch.arange(V, device=DEV).expand(3, -1).div(64).to(dtype).contiguous()
    elif kind == "falling":
        x = torch.arange(V, 0, -1, device=DEV).expand(3, -1).div(64).to(dtype).contiguous()
    elif kind == "one_thread":  # the likely ids at distances of whole turns of a CTA's threads
        x[:, 3::2048] += 20
        x[:, 4::1024] += 20
    elif kind == "zeros":  # 0 and -0 are equal
        x = torch.where(torch.arange(V, device=DEV) % 3 == 0, -0.0, 0.0).to(dtype).expand(3, -1).contiguous()
    elif kind == "masked":
        x[:, V // 2:] = -INF
    elif kind == "mostly_masked":
        x[:] = -INF
        x[:, V - 2:] = torch.tensor([1.0, 2.0], dtype=dtype)
    elif kind == "lowest":
        x[:, : V - 2] = torch.finfo(dtype).min
    y = x.argmax(-1)
    check(x, y, min(32, V))


@pytest.mark.parametrize("dtype", [BF, FF])
@pytest.mark.parametrize("V", [40, 30000])
def test_rows_without_a_distribution(V, dtype):
    x, y = data((5,), V, dtype)
    x[0, 7] = float("nan")
    x[1, V - 1] = INF
    x[2] = -INF
    x[3, 0], x[3, 1] = INF, float("nan")
    check(x, y, 4)
    y[:] = -100
    got = run(x, y)
    assert (got.logprobs == 0).all() and torch.isnan(got.entropy).tolist() == [True] * 4 + [False]
    _native.poll_status(DEV)


def test_targets_outside():
    x, y = data((4,), 100, BF)
    y[1], y[2], y[3] = 100, -1, -100
    got = run(x, y, 3)
    with pytest.raises(_native.TmwError):
        _native.poll_status(DEV)
    assert torch.isnan(got.logprobs).tolist() == [False, True, True, False] and got.logprobs[3] == 0
    assert torch.isfinite(got.entropy).all() and (got.top_ids >= 0).all()


def test_far_apart_and_large_logits():
    """Differences count, not magnitudes: the same distribution 10,000 up, and one token ahead of all others."""
    x = torch.randint(-20, 20, (3, 5000), device=DEV).float()
    y = torch.randint(0, 5000, (3,), device=DEV)
    for up in (0.0, 10000.0, -30000.0):
        check(x + up, y, 5)
    x[:, 4] = 90.0
    check(x, y, 5)


@pytest.mark.parametrize("rows", [1, 100, 700, 4000])
@pytest.mark.parametrize("V,n_top", [(300, 7), (1030, 32), (5001, 1), (16500, 20), (40000, 32)])
def test_every_number_of_warps(V, n_top, rows):
    """One to eight warps to a row, clusters of them, by the number of rows and their length."""
    if rows * V > 3e7:
        rows = int(3e7 / V)
    check(*data((rows,), V, BF, seed=rows), n_top)


def test_more_than_2_to_the_31_logits():
    x = torch.zeros(67200, 32003, dtype=BF, device=DEV)
    last = data((3,), 32003, BF)[0]
    x[-3:] = last
    y = torch.zeros(67200, dtype=torch.int64, device=DEV)
    y[-3:] = torch.tensor([5, 32002, 77])
    a = x.requires_grad_(True)
    out = token_logprobs(a, y, 4)
    picked, entropy, ids, top, _ = reference(last, y[-3:], 4)
    assert torch.equal(out.top_ids[-3:], ids) and torch.equal(out.top_ids[:2], torch.arange(4, device=DEV).expand(2, -1))
    assert ((out.logprobs[-3:].double() - picked).abs() <= allowed(last, picked)).all()
    (g,) = torch.autograd.grad(out.logprobs[-3:].sum(), a)
    want = -torch.softmax(last.double(), -1)
    want[torch.arange(3), y[-3:]] += 1
    assert ((g[-3:].double() - want).abs() <= 2.0 ** -8 * want.abs() + 5e-5).all() and (g[:67197:999] == 0).all()


@pytest.mark.parametrize("dtype", [BF, FF])
@pytest.mark.parametrize("rows,V", [((5,), 60), ((3,), 40000), ((1,), 128000), ((2000,), 900), ((900,), 5000)])
def test_tokens_that_are_nearly_certain(rows, V, dtype):
    """Log-probabilities and entropies of almost nothing, to their own size: ln(1 + rest) with the rest summed up by itself, weights to
    2^-22 and their arguments, below 100, to 2^-23 of themselves, chains of at most 512 sums.  (The 64-bit reference sums V weights
    up next to 1, each sum off by 2^-53 at most: V 2^-53 is what its own logarithm may be off by.)"""
    x, y = data(rows, V, dtype, seed=3, spread=2.0)
    ahead = torch.linspace(8.0, 20.0, x.shape[0], device=DEV) + math.log(V)
    x.scatter_(1, y[:, None], (x.float().amax(-1) + ahead).to(dtype)[:, None])
    got, (picked, entropy, _, _, _) = run(x, y), reference(x, y, 1)
    most = 100 * 2.0 ** -23 + 512 * 2.0 ** -24 + 2.0 ** -21
    assert ((got.logprobs.double() - picked).abs() <= most * picked.abs() + V * 2.0 ** -53).all(), ((got.logprobs.double() / picked) - 1).abs().max()
    assert ((got.entropy.double() - entropy).abs() <= 2 * most * entropy + V * 2.0 ** -53).all(), ((got.entropy.double() / entropy) - 1).abs().max()


# ---- gradients ---------------------------------------------------------------------------------------------------------------------


def gradients(x, y, n_top, weights):
    """The kernel's gradient and, in 64 bits, autograd's of the definition."""
    a = x.clone().requires_grad_(True)
    out = token_logprobs(a, y, n_top)
    sum((w * o).sum() for w, o in zip(weights, (out.logprobs, out.entropy, out.top_logprobs)) if w is not None).backward()
    b = x.double().requires_grad_(True)
    logp = torch.log_softmax(b, -1)
    p = logp.exp()
    hidden = p == 0
    entropy = -(p * logp.masked_fill(hidden, 0.0)).sum(-1)
    counted = (y >= 0) & (y < x.shape[-1])
    picked = logp.gather(-1, y.masked_fill(~counted, 0)[..., None])[..., 0].masked_fill(~counted, 0.0)
    top = logp.gather(-1, out.top_ids) if n_top else None
    sum((w.double() * o).sum() for w, o in zip(weights, (picked, entropy, top)) if w is not None).backward()
    return a.grad, b.grad


def check_gradients(got, want, weights, x):
    """One rounding, and fp32 arithmetic: log p is off by 5e-5 at most (``allowed``), p by as much of itself, and what it is
    multiplied with - incoming gradients, the entropy's times log p + H - stays below 13 times their size where p counts."""
    size = sum(w.abs().sum(-1) if w.dim() == want.dim() else w.abs() for w in weights if w is not None).double()[..., None]
    step = torch.finfo(got.dtype).eps / 2
    p = torch.softmax(x.double(), -1)
    bound = step * want.abs() + size * (13 * 5e-5 * p + 2.0 ** -23) + torch.finfo(got.dtype).tiny
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (off / bound).max()


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("which", ["logprobs", "entropy", "top", "all"])
@pytest.mark.parametrize("rows,V,n_top", [((3,), 9, 4), ((2, 5), 1001, 8), ((4,), 40003, 32)])
def test_gradients_against_64_bits(rows, V, n_top, which, dtype):
    x, y = data(rows, V, dtype, seed=1)
    if V > 100:
        x[..., V - 5:] = -INF  # hidden ids get no gradient
        y.clamp_(max=V - 6)
    y.view(-1)[0] = -100
    g = torch.Generator(device=DEV).manual_seed(V)
    weights = [torch.randn(rows, generator=g, device=DEV) if which in (n, "all") else None for n in ("logprobs", "entropy")]
    weights.append(torch.randn(*rows, n_top, generator=g, device=DEV) if which in ("top", "all") else None)
    got, want = gradients(x, y, n_top, weights)
    assert torch.isfinite(got).all() and got.shape == x.shape and got.dtype == dtype
    if V > 100:
        assert (got[..., V - 5:] == 0).all()
    check_gradients(got, want, weights, x)
    _native.poll_status(DEV)


def test_gradient_against_differences():
    """The change of the outputs along a direction, in fp32 with a step of 2^-7: off by its third-order term and the rounding."""
    x, y = data((6,), 300, FF, seed=2, spread=1.0)
    a = x.clone().requires_grad_(True)
    out = token_logprobs(a, y, 3)
    (out.logprobs.sum() + out.entropy.sum() - out.top_logprobs.sum()).backward()
    g = torch.Generator(device=DEV).manual_seed(5)
    for _ in range(4):
        d = torch.randn(x.shape, generator=g, device=DEV)
        eps = 2.0 ** -7
        f = []
        for s in (eps, -eps):
            o = run(x + s * d, y)
            picked = torch.log_softmax((x + s * d).double(), -1).gather(-1, out.top_ids)  # (the same ids on both sides)
            f.append(o.logprobs.double().sum() + o.entropy.double().sum() - picked.sum())
        got = (a.grad.double() * d.double()).sum()
        assert abs((f[0] - f[1]) / (2 * eps) - got) <= 5e-3 * (1 + abs(got))


def test_gradient_of_strided_and_repeated_logits():
    """Views: every row's gradient reaches the tensor behind them; rows used twice add up."""
    whole, _ = data((3, 8), 501, FF)
    for cut in (lambda t: t[:, 1:-1, 3:], lambda t: t[1:2].expand(3, -1, -1), lambda t: t.transpose(0, 1)):
        a, b = whole.clone().requires_grad_(True), whole.double().requires_grad_(True)
        x, z = cut(a), cut(b)
        y = torch.randint(0, x.shape[-1], x.shape[:-1], device=DEV)
        token_logprobs(x, y).logprobs.sum().backward()
        torch.log_softmax(z, -1).gather(-1, y[..., None]).sum().backward()
        assert ((a.grad.double() - b.grad).abs() <= 1e-5).all()


def test_rows_that_nothing_comes_back_to():
    """Not counted, or unused: zeros, whatever the logits are."""
    x, y = data((4,), 64, BF)
    x[1] = float("nan")
    y[0] = y[1] = -100
    a = x.clone().requires_grad_(True)
    token_logprobs(a, y).logprobs.sum().backward()
    assert (a.grad[:2] == 0).all() and (a.grad[2:] != 0).any()
    a.grad = None
    out = token_logprobs(a, y, 2)
    out.logprobs[2].backward()
    assert (a.grad[[0, 1, 3]] == 0).all()
    assert not out.top_ids.requires_grad


def test_captured_forward_and_backward():
    """A training step's pass in a graph, replayed with new logits and targets."""
    x, y = data((37,), 3001, BF, seed=3)
    held = x.clone().requires_grad_(True)
    targets = y.clone()

    def step():
        out = token_logprobs(held, targets, 4)
        (g,) = torch.autograd.grad(out.logprobs.sum() + out.entropy.sum(), held)
        return out, g

    side = torch.cuda.Stream(DEV)
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grad = step()
    for seed in (4, 5):
        x2, y2 = data((37,), 3001, BF, seed=seed)
        with torch.no_grad():
            held.copy_(x2)
        targets.copy_(y2)
        graph.replay()
        eager = x2.clone().requires_grad_(True)
        o = token_logprobs(eager, y2, 4)
        (g,) = torch.autograd.grad(o.logprobs.sum() + o.entropy.sum(), eager)
        assert torch.equal(o.logprobs, out.logprobs) and torch.equal(o.top_ids, out.top_ids) and torch.equal(g, grad)


@pytest.mark.parametrize("dtype", [FF, BF])
def test_model_scores_and_trains(dtype):
    """TitanMAC.token_logprobs: the mean is the loss, and so is its gradient; alternatives of a greedy continuation lead it."""
    cfg = TitanMACConfig(vocab_size=200, d_model=128, n_heads=2, n_layers=2, d_ff=256, max_seq_len=64, window_size=16, n_persistent=4,
                         use_block_sparse=False)
    torch.manual_seed(1)
    model = TitanMAC(cfg).to(device=DEV, dtype=dtype)
    ids = torch.randint(0, 200, (3, 20), device=DEV)
    out = model.token_logprobs(ids, n_top=5)
    assert out.logprobs.shape == (3, 20) and out.top_ids.shape == (3, 20, 5) and (out.logprobs[:, -1] == 0).all()
    (-out.logprobs[:, :-1].mean()).backward()
    mine = {n: p.grad.double() for n, p in model.named_parameters()}
    model.zero_grad(set_to_none=True)
    loss = model(ids, labels=ids)["loss"]
    loss.backward()
    step = torch.finfo(dtype).eps
    assert abs(-out.logprobs[:, :-1].double().mean() - loss.double()) <= 4 * step * loss.double() + 1e-5
    for n, p in model.named_parameters():  # (16-bit: the loss's gradient is rounded before and behind the factor 1 / n)
        a, b = mine[n], p.grad.double()
        assert (a - b).norm() <= (1e-4 if dtype == FF else 4 * step) * b.norm() + 1e-9, n
    if dtype == FF:  # (in 16 bits two likely tokens may be nearer than the paths' roundings)
        with torch.no_grad():
            assert torch.equal(model.token_logprobs(ids, n_top=1).top_ids[:, -1, 0], model.generate(ids, 2)[:, 20])


def test_refusals():
    x, y = data((4,), 100, BF)
    for error, args in [(RuntimeError, (x.cpu(), y.cpu())), (RuntimeError, (x, y.cpu())), (TypeError, (x.double(), y)),
                        (TypeError, (x, y.int())), (ValueError, (x, y[:2])), (ValueError, (x[:, :0], y)), (ValueError, (x, y, 33)),
                        (ValueError, (x, y, -1)), (ValueError, (x[:, :3], y, 4))]:
        with pytest.raises(error):
            token_logprobs(*args)
    none = token_logprobs(x[:0], y[:0], 2)
    assert none.logprobs.shape == (0,) and none.top_ids.shape == (0, 2)
    a = x[:0].clone().requires_grad_(True)
    token_logprobs(a, y[:0]).logprobs.sum().backward()
    assert a.grad.shape == (0, 100)
