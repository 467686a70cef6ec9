"""TitanMAC with paged caches and ids or positions outside their tables: met on the device, in every type, row by row."""

import pytest
import torch

from titanmac_b200 import PagedCache, TitanMAC, TitanMACConfig, _native

DEV = torch.device("cuda:0")
V, MAX = 96, 64


def make(device, dtype, n_layers=2):
    cfg = TitanMACConfig(vocab_size=V, d_model=128, n_heads=2, n_layers=n_layers, d_ff=256, max_seq_len=MAX, window_size=16,
                         n_persistent=3, use_block_sparse=False)
    torch.manual_seed(0)
    return TitanMAC(cfg).to(device=device, dtype=dtype).eval()


@pytest.mark.parametrize("token,pos", [(V, 5), (-1, 5), (1 << 40, 5), (3, MAX), (3, -2), (3, (1 << 31) - 1)])
def test_nothing_outside_a_table_is_looked_up(token, pos):
    """On the CPU the embedding's own check is an IndexError.  The step gets past it: the wrong row's keys are NaN, and it attends
    nowhere; the other one is as it would be."""
    model = make("cpu", torch.float32, 1)
    steps = []

    class Held(PagedCache):
        def __init__(self):
            pass

        def decode(self, q, k_new, v_new, at, out=None, seen=None):
            steps.append((k_new, at, seen))
            return torch.zeros_like(q)

    for row in ((3, 5), (token, pos)):
        model.decode_step(torch.tensor([2, row[0]]), torch.tensor([1, row[1]], dtype=torch.int32), [Held()])
    (sound, _, first), (k_new, at, seen) = steps
    assert first.tolist() == [1, 5] and at.tolist() == [1, pos] and seen.tolist() == [1, -2]
    assert torch.isfinite(sound).all() and torch.isnan(k_new[1]).all() and torch.equal(k_new[0], sound[0])


@pytest.mark.parametrize("token", [V, -1, 1 << 40])
def test_nothing_outside_the_vocabulary_is_looked_up_for_a_prompt(token):
    model = make("cpu", torch.float32)
    caches = [object.__new__(PagedCache) for _ in model.layers]
    ids = torch.ones(2, 9, dtype=torch.int64)
    ids[1, 4] = token
    with pytest.raises(RuntimeError, match="no CPU path"):
        model.prefill(ids, caches)


def test_a_prompt_longer_than_the_positions_is_refused():
    model = make("cpu", torch.float32)
    with pytest.raises(ValueError, match="max_seq_len"):
        model.prefill(torch.ones(1, MAX + 1, dtype=torch.int64), [object.__new__(PagedCache) for _ in model.layers])


def reported():
    with pytest.raises(_native.TmwError):
        _native.poll_status(DEV)


def prepared(dtype, n_layers, T=20, B=4):
    model = make(DEV, dtype, n_layers)
    ids = torch.randint(0, V, (B, T), generator=torch.Generator().manual_seed(1)).to(DEV)
    table = torch.randperm(B * 8, generator=torch.Generator().manual_seed(2)).view(B, 8).to(torch.int32).to(DEV)
    return model, ids, lambda: model.new_paged_caches(table, B * 8, 13, dtype)  # (pages for more positions than the model has)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("token,pos,later", [(V, 20, True), (-1, 20, True), (3, MAX, False), (3, 200, False), (3, -2, False)])
def test_a_step_outside_the_tables(token, pos, later, dtype):
    _native.poll_status(DEV)
    model, ids, new = prepared(dtype, 2)
    rest = [0, 1, 3]
    good = [torch.tensor([5, 6, 7, 8], device=DEV), torch.full((4,), 20, dtype=torch.int32, device=DEV)]
    _, sound = model.prefill(ids, new())
    want = model.decode_step(*good, sound)
    next_want = model.decode_step(good[0], good[1] + 1, sound)
    _native.poll_status(DEV)
    _, caches = model.prefill(ids, new())
    tokens, at = good[0].clone(), good[1].clone()
    tokens[2], at[2] = token, pos
    got = model.decode_step(tokens, at, caches)
    reported()
    assert torch.isnan(got[2]).all() and torch.equal(got[rest], want[rest])
    got = model.decode_step(good[0], good[1] + 1, caches)
    _native.poll_status(DEV)
    assert torch.equal(got[rest], next_want[rest])
    assert not later or torch.isnan(got[2]).all()  # it sees the key that the wrong token has left


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n_layers", [1, 2])
@pytest.mark.parametrize("row", [0, 2])
def test_a_prompt_outside_the_vocabulary(row, n_layers, dtype):
    _native.poll_status(DEV)
    model, ids, new = prepared(dtype, n_layers)
    rest = [b for b in range(4) if b != row]
    want, sound = model.prefill(ids, new())
    step = [torch.tensor([5, 6, 7, 8], device=DEV), torch.full((4,), 20, dtype=torch.int32, device=DEV)]
    next_want = model.decode_step(*step, sound)
    _native.poll_status(DEV)
    ids[row, 19] = V
    got, caches = model.prefill(ids, new())
    reported()
    assert torch.isnan(got[row]).all() and torch.equal(got[rest], want[rest])
    got = model.decode_step(*step, caches)
    _native.poll_status(DEV)
    assert torch.isnan(got[row]).all() and torch.equal(got[rest], next_want[rest])


@pytest.mark.gpu
def test_a_row_without_a_sequence_may_hold_any_token():
    _native.poll_status(DEV)
    model, ids, new = prepared(torch.bfloat16, 2)
    _, caches = model.prefill(ids, new())
    pages = [c.k_pages.clone() for c in caches]
    at = torch.tensor([20, 20, -1, 20], dtype=torch.int32, device=DEV)
    got = model.decode_step(torch.tensor([5, 6, V + 7, 8], device=DEV), at, caches)
    _native.poll_status(DEV)
    assert torch.isfinite(got[[0, 1, 3]]).all()
    held = caches[0].page_table[2].long()
    assert all(torch.equal(c.k_pages[held], p[held]) for c, p in zip(caches, pages))


@pytest.mark.gpu
def test_a_captured_step_meets_them_too():
    _native.poll_status(DEV)
    model, ids, new = prepared(torch.bfloat16, 2)
    _, caches = model.prefill(ids, new())
    token, at = torch.tensor([5, 6, 7, 8], device=DEV), torch.full((4,), 20, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream(DEV)
    with torch.cuda.stream(side):
        model.decode_step(token, at, caches)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = model.decode_step(token, at, caches)
    at += 1
    graph.replay()
    _native.poll_status(DEV)
    assert torch.isfinite(logits).all()
    at += 1
    token[1] = V
    graph.replay()
    reported()
    assert torch.isnan(logits[1]).all() and torch.isfinite(logits[[0, 2, 3]]).all()
