"""A model serving from pages in 8 bits, and checking drafted trees: the calls together, as a serving loop makes them."""

import pytest
import torch

from titanmac_b200 import TitanMAC, TitanMACConfig, _native, token_logprobs

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, FF, I8, E4 = torch.bfloat16, torch.float32, torch.int8, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _fresh_status():
    _native.poll_status(DEV)
    yield


def build(dtype, vocab=64, window=24, n_p=4, positions=128, seed=0):
    cfg = TitanMACConfig(vocab_size=vocab, d_model=128, n_heads=2, n_layers=2, d_ff=256, max_seq_len=positions, window_size=window,
                         n_persistent=n_p, use_block_sparse=False)
    torch.manual_seed(seed)
    return TitanMAC(cfg).to(device=DEV, dtype=dtype).eval()


def numbers(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# As for the serving loop from pages: fp32 sums in another order, twice over; in bf16 some 24 roundings of half a step on either side, of
# logits below 2 (with the pages the same the cached numbers are the same)
MOST = {FF: 2e-5, BF: 2 * 24 * 2.0 ** -8 * 2.0}


@pytest.mark.parametrize("dtype,page_dtype", [(FF, None), (BF, None), (FF, I8), (BF, I8), (BF, E4)])
@pytest.mark.parametrize("nodes", [7, 40])
def test_a_tree_says_what_its_paths_say(dtype, page_dtype, nodes):
    """Every node's logits are those of the step that would come to it token by token, and behind a kept path everything goes on
    as if it had come alone."""
    model = build(dtype)
    g = torch.Generator().manual_seed(nodes)
    B, T = 2, 33
    ids = torch.randint(0, 64, (B, T), generator=g).to(DEV)
    table = torch.randperm(2 * 12, generator=g).view(2, 12).to(torch.int32).to(DEV)
    first = model.prefill(ids, model.new_paged_caches(table, 24, 8, dtype, page_dtype))[1]
    drafts = torch.randint(0, 64, (B, nodes), generator=g).to(DEV)
    parents = torch.tensor([[-1] + [(i - 1) // 2 for i in range(1, nodes)], [-1] + [max(0, i - 3) for i in range(1, nodes)]], device=DEV)
    start = numbers([T, T])
    logits = model.decode_tree(drafts, parents, start, first)
    _native.poll_status(DEV)
    path = [[], []]
    for b in range(B):
        i = nodes - 1
        while i >= 0:
            path[b].insert(0, i)
            i = int(parents[b, i])
    most = min(len(p) for p in path)
    second = model.prefill(ids, model.new_paged_caches(table, 24, 8, dtype, page_dtype))[1]
    for step in range(most):
        token = torch.stack([drafts[b, path[b][step]] for b in range(B)])
        want = model.decode_step(token, start + step, second)
        got = torch.stack([logits[b, path[b][step]] for b in range(B)])
        assert (got.float() - want.float()).abs().max() <= MOST[dtype] * (1 + want.float().abs().max())
    kept = numbers([p[:most] for p in path])
    model.keep_drafts(first, start, kept, numbers([most] * B))
    token = torch.randint(0, 64, (B,), generator=g).to(DEV)
    got, want = (model.decode_step(token, start + most, caches) for caches in (first, second))
    _native.poll_status(DEV)
    # a kept key was rounded once more or less than the other's: in 8 bits a code may be the next one, a step of 2^-7 or 2^-4 of a number
    step = {None: 0.0, I8: 2.0 ** -7, E4: 2.0 ** -4}[page_dtype]
    assert (got.float() - want.float()).abs().max() <= (MOST[dtype] + step) * (1 + want.float().abs().max())


@pytest.mark.parametrize("page_dtype,off", [(I8, 2.0 ** -8), (E4, 2.0 ** -4)])
def test_pages_in_8_bits_change_little(page_dtype, off):
    """Prompt and decoding with keys and values of 8 bits against rings: a number is off by half a step, 2^-8 of its row's largest or 2^-4 of
    itself; two layers of averages of such numbers and what becomes of them in the residual stream, whose logits are below 2."""
    model = build(FF)
    ids = torch.randint(0, 64, (2, 40), device=DEV)
    table = torch.randperm(2 * 8).view(2, 8).to(torch.int32).to(DEV)
    want, rings = model.prefill(ids)
    got, paged = model.prefill(ids, model.new_paged_caches(table, 16, 16, FF, page_dtype))
    assert torch.equal(got, want)  # (the prompt itself does not go through the pages)
    token = want.argmax(-1)
    for i in range(20):
        pos = numbers([40 + i] * 2)
        want, got = model.decode_step(token, pos, rings), model.decode_step(token, pos, paged)
        assert (got - want).abs().max() <= 4 * off * (1 + want.abs().max())
        token = want.argmax(-1)
    _native.poll_status(DEV)


@pytest.mark.parametrize("dtype,page_dtype", [(FF, None), (BF, I8)])
def test_speculative_greedy_decoding(dtype, page_dtype):
    """Trees with one right branch and wrong ones beside it: what is accepted is what greedy decoding says, token for token."""
    model = build(dtype, seed=3)
    g = torch.Generator().manual_seed(1)
    B, T, new = 2, 20, 24
    ids = torch.randint(0, 64, (B, T), generator=g).to(DEV)
    table = torch.arange(2 * 12).view(2, 12).to(torch.int32).to(DEV)

    logits, caches = model.prefill(ids, model.new_paged_caches(table, 24, 8, dtype, page_dtype))
    token = logits.argmax(-1)
    greedy = [token]
    for i in range(new):
        token = model.decode_step(token, numbers([T + i] * B), caches).argmax(-1)
        greedy.append(token)
    greedy = torch.stack(greedy, 1)

    logits, caches = model.prefill(ids, model.new_paged_caches(table, 24, 8, dtype, page_dtype))
    said, start, parents = [[int(logits[b].argmax())] for b in range(B)], [T] * B, [-1, 0, 0, 1, 1, 3]
    while min(len(s) for s in said) <= new:
        drafts = torch.randint(0, 64, (B, 6), generator=g)
        for b in range(B):  # node 0 is the last token said; of its drafts one path is right for one to three tokens
            at = len(said[b]) - 1
            drafts[b, 0] = said[b][-1]
            right = [int(x) for x in greedy[b, at + 1:at + 4]]
            for node, x in zip((2, 1, 3)[at % 2:], right if at % 2 else right[:1]):
                drafts[b, node] = x
        out = model.decode_tree(drafts.to(DEV), torch.tensor([parents] * B, device=DEV), numbers(start), caches)
        lp = token_logprobs(out, out.argmax(-1), n_top=1)
        assert torch.equal(lp.top_ids[..., 0], out.argmax(-1))
        choice = out.argmax(-1).cpu()
        kept = []
        for b in range(B):
            path, node = [0], 0
            while True:
                node = next((i for i in range(6) if parents[i] == node and int(drafts[b, i]) == int(choice[b, node])), -1)
                if node < 0:
                    break
                path.append(node)
            said[b] += [int(choice[b, i]) for i in path]
            kept.append(path)
        most = max(len(p) for p in kept)
        model.keep_drafts(caches, numbers(start), numbers([p + [-1] * (most - len(p)) for p in kept]), numbers([len(p) for p in kept]))
        start = [s + len(p) for s, p in zip(start, kept)]
    _native.poll_status(DEV)
    steps = [torch.tensor(s[: new + 1]) for s in said]
    if dtype == FF:  # (in bf16 two nearly equal logits may change places)
        assert all(torch.equal(s, greedy[b].cpu()) for b, s in enumerate(steps))
    assert max(start) > T + 8


def test_ids_and_positions_outside_their_tables():
    model = build(FF, positions=40)
    table = torch.arange(3 * 8).view(3, 8).to(torch.int32).to(DEV)
    ids = torch.randint(0, 64, (3, 30), device=DEV)
    _, caches = model.prefill(ids, model.new_paged_caches(table, 24, 8, FF))
    drafts, parents = torch.randint(0, 64, (3, 4), device=DEV), torch.tensor([[-1, 0, 0, 2]] * 3, device=DEV)
    clean = model.decode_tree(drafts, parents, numbers([30, 30, -1]), caches)
    _native.poll_status(DEV)
    drafts[0, 2] = 64
    got = model.decode_tree(drafts, parents, numbers([30, 30, -1]), caches, numbers([4, 3, 4]))
    with pytest.raises(_native.TmwError):
        _native.poll_status(DEV)
    assert torch.isnan(got[0, 2:]).all() and torch.equal(got[0, :2], clean[0, :2]) and torch.equal(got[1, :3], clean[1, :3])
    got = model.decode_tree(drafts[:, :2], parents[:, :2], numbers([-1, 39, -1]), caches)  # node 1 would be at position 40
    with pytest.raises(_native.TmwError):
        _native.poll_status(DEV)
    assert torch.isfinite(got[1, 0]).all() and torch.isnan(got[1, 1]).all()
    with pytest.raises(TypeError):
        model.decode_tree(drafts, parents, numbers([30, 30, -1]), model.new_caches(3, DEV, FF))
