"""CPU: the paged history's page accounting -- pages are taken as sequences
grow, given back behind the window and on reset, never shared; the index
tensors say what the accounting says; refusals change nothing."""

import random

import pytest
import torch

from fast_moss_b200 import PagedHistory


def history(sequences=3, pages=40, max_positions=400, page_size=16, context=None):
    return PagedHistory(2, sequences, 2, 64, "cpu", pages=pages, max_positions=max_positions,
                        page_size=page_size, context=context)


def check(h, low):
    """Every position from low[s] on has a page, no page has two owners, and
    the table holds exactly the pages in use."""
    size = h.page_size
    table = h.page_table.tolist()
    used = [p for row in table for p in row if p >= 0]
    assert len(used) == len(set(used)) and len(used) + h.free_pages == h.k_pages[0].shape[0]
    for s, row in enumerate(table):
        have = h.lengths[s]
        assert h.kv_len[s] == have
        want = set(range(low[s] // size, -(-have // size))) if have > low[s] else set()
        assert {c for c, p in enumerate(row) if p >= 0} >= want
        assert all(p < 0 for c, p in enumerate(row) if c * size >= have)


@pytest.mark.parametrize("seed,context,page_size", [(0, None, 16), (1, 20, 16), (2, 1, 32), (3, 100, 16)])
def test_pages_follow_the_sequences(seed, context, page_size):
    rng = random.Random(seed)
    h = history(sequences=4, pages=60, max_positions=5000, page_size=page_size, context=context)
    for _ in range(120):
        new = [rng.choice([0, 1, 1, 4, rng.randint(0, 40)]) for _ in range(4)]
        before = list(h.lengths)
        if rng.random() < 0.1:
            s = rng.randrange(4)
            h.reset([s])
            before[s] = 0
        try:
            rows = h.advance(new)
        except RuntimeError:
            assert h.lengths == before
            h.reset([max(range(4), key=lambda s: h.lengths[s])])
            continue
        assert rows == sum(new) == h.q_start[-1]
        assert h.lengths == [a + b for a, b in zip(before, new)]
        assert (h.q_start[1:] - h.q_start[:-1]).tolist() == new
        check(h, [0 if context is None else max(0, a - context + 1) for a in before])
        if context is not None:  # nothing is kept that no later token attends to
            held = [sum(p >= 0 for p in row) for row in h.page_table.tolist()]
            for s, a in enumerate(before):
                low = max(0, a - context + 1)
                assert held[s] <= -(-h.lengths[s] // page_size) - low // page_size


def test_refusals_change_nothing():
    h = history(pages=4, max_positions=100)
    h.advance([20, 10, 0])
    state = (h.page_table.clone(), h.kv_len.clone(), h.q_start.clone(), list(h.lengths), h.free_pages)
    for new, error in (([81, 0, 0], ValueError), ([0, 0, 40], RuntimeError), ([1, 2], ValueError),
                       ([1, -1, 0], ValueError)):
        with pytest.raises(error):
            h.advance(new)
        assert torch.equal(h.page_table, state[0]) and torch.equal(h.kv_len, state[1])
        assert torch.equal(h.q_start, state[2])
        assert (h.lengths, h.free_pages) == state[3:]
    h.reset([0])
    assert h.advance([0, 0, 40]) == 40
    with pytest.raises(ValueError):
        h.reset([3])
    h.reset()
    assert h.free_pages == 4
    for kw in (dict(page_size=24), dict(pages=0), dict(context=0), dict(sequences=0)):
        with pytest.raises(ValueError):
            history(**kw)


def test_a_full_table_and_a_pool_to_the_last_page():
    h = history(sequences=1, pages=3, max_positions=48)
    h.advance([48])
    assert h.free_pages == 0 and sorted(h.page_table[0].tolist()) == [0, 1, 2]
    with pytest.raises(ValueError):
        h.advance([1])
    assert h.advance([0]) == 0


def test_stack_config_weight_names():
    from fast_moss_b200.transformer import StackConfig, WEIGHT_NAMES, init_weights

    plain = StackConfig(layers=1, dim=128, heads=2, ffn=256, context=8)
    normed = StackConfig(layers=1, dim=128, heads=2, ffn=256, context=8, qk_norm=True)
    assert plain.weight_names == WEIGHT_NAMES
    assert set(init_weights(plain)[0]) == set(WEIGHT_NAMES)
    assert set(init_weights(normed)[0]) == set(WEIGHT_NAMES) | {"q_norm_w", "k_norm_w"}
    a, b = init_weights(plain, seed=4)[0], init_weights(normed, seed=4)[0]
    assert all(torch.equal(a[k], b[k]) for k in WEIGHT_NAMES)


def test_a_step_takes_at_least_the_rows_that_were_made_room_for():
    """Fewer rows than advance() announced would leave positions of the history
    unwritten: refused before anything runs; a captured step takes the history
    as it is at its replays."""
    from unittest import mock

    from fast_moss_b200 import transformer

    # a stack without its weights, which live on a GPU: nothing here comes to them
    cfg = transformer.StackConfig(layers=2, dim=128, heads=2, ffn=128, context=8)
    stack = object.__new__(transformer.StreamingTransformer)
    stack.cfg, stack.device = cfg, torch.device("cpu")
    stack.layers = [{"norm1_w": None, "norm1_b": None}] * 2
    h = stack.paged_history(2, pages=6, max_positions=64)
    h.advance([5, 1])
    ran = RuntimeError("the step ran")
    with mock.patch.object(transformer, "layer_norm", side_effect=ran), \
            mock.patch.object(torch.cuda, "is_current_stream_capturing", return_value=False):
        for rows in (0, 1, 5):
            with pytest.raises(ValueError, match="rows"):
                stack.step_paged(torch.zeros(rows, 128), h)
        for rows in (6, 7):
            with pytest.raises(RuntimeError, match="the step ran"):
                stack.step_paged(torch.zeros(rows, 128), h)
        with mock.patch.object(torch.cuda, "is_current_stream_capturing", return_value=True):
            with pytest.raises(RuntimeError, match="the step ran"):
                stack.step_paged(torch.zeros(2, 128), h)
        h.advance([0, 1])
        with pytest.raises(RuntimeError, match="the step ran"):
            stack.step_paged(torch.zeros(1, 128), h)
    with pytest.raises(RuntimeError, match="pages"):
        h.advance([59, 62])
    assert h.rows == 1


def test_a_refused_reset_changes_nothing():
    h = history(pages=6, max_positions=64)
    h.advance([20, 10, 33])
    state = (list(h.lengths), h.free_pages)
    for bad in ([0, 3], [1, -1], [2, 0, 99], iter([0, 5])):
        with pytest.raises(ValueError):
            h.reset(bad)
        assert (h.lengths, h.free_pages) == state
    h.reset(iter([2, 0, 2]))  # the same one twice
    assert h.lengths == [0, 10, 0] and h.free_pages == 5
    h.advance([0, 1, 0])
    check(h, [0, 0, 0])
