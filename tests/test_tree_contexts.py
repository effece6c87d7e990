"""Which tree contexts can still be ended: the last forward begun of sequences that are the ones it was begun for."""
import pytest
import torch

from test_tree_cache import CPU, HKV, HQ, L, D, Model, make, prefill, rows

BACKENDS = pytest.mark.parametrize("backend", ["paged", "contiguous"])


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def _write(cache, ctx, S, value):
    for i in range(L):
        x = torch.full((ctx.batch_size, S, HQ, D), value)
        ctx.attend(i, x, x[:, :, :HKV], x[:, :, :HKV], HQ, HKV)


def _refused(cache, ctx):
    V = 60
    S = max(ctx.new_token_counts)
    B = ctx.batch_size
    with pytest.raises(ValueError, match="has changed"):
        cache.end_tree(ctx, _i32([list(range(S))] * B), _i32(ctx.new_token_counts))
    with pytest.raises(ValueError, match="has changed"):
        cache.accept_tree(ctx, torch.zeros(B, S).long(), torch.full((B, S, V), 1 / V), torch.zeros(B, S), torch.zeros(B))
    with pytest.raises(ValueError, match="have changed"):
        _write(cache, ctx, S, 9.0)


@BACKENDS
@pytest.mark.parametrize("release", [True, False])
def test_another_sequence_of_the_same_id_and_length(backend, release):
    """Its pages are other pages; those of the old one may be anyone's."""
    cache = make(backend, "cpu", CPU)
    cache.allocate_sequence("a")
    if backend == "contiguous":  # (a slot is given again once all are free)
        cache.begin_forward(["a"], [1])
    ctx = cache.begin_tree(["a"], [[-1, 0, 0, 2]])
    _write(cache, ctx, 4, 1.0)
    if release:
        cache.release_sequence("a")
        cache.allocate_sequence("b")
        one = cache.begin_forward(["b"], [4])
        _write(cache, one, 4, 2.0)
        cache.end_forward(one)
    cache.allocate_sequence("a")
    before = cache._kv_pools.k.clone()
    _refused(cache, ctx)
    assert torch.equal(cache._kv_pools.k, before) and cache._states["a"].num_tokens == 0
    if release:
        assert (rows(cache, "b", 0)[0] == 2).all()


@BACKENDS
def test_two_open_trees_of_one_sequence(backend):
    cache, model = make(backend, "cpu", CPU), Model("cpu")
    ids, _ = prefill(cache, model, [[1, 2, 3], [4, 5], [6]], "cpu")
    first = cache.begin_tree(ids, [[-1, 0], [-1, 0], [-1]])
    alone = cache.begin_tree(ids[1:2], [[-1, 0, 0]])  # (of one of them: the other two's nodes cannot be kept without it)
    _write(cache, alone, 3, 3.0)
    _refused(cache, first)
    assert cache.end_tree(alone, _i32([[0, 2]]), _i32([2])) == [2]
    _refused(cache, first)
    assert [cache._states[s].num_tokens for s in ids] == [3, 4, 1]
    # trees of different sequences stay open side by side
    x, y = cache.begin_tree(ids[:1], [[-1, 0]]), cache.begin_tree(ids[1:], [[-1], [-1]])
    assert cache.end_tree(x, _i32([[0, 1]]), _i32([2])) == [2] and cache.end_tree(y, _i32([[0], [0]]), _i32([1, 1])) == [1, 1]
    assert not cache._open_trees


@BACKENDS
@pytest.mark.parametrize("n", [1, 3])
def test_a_plain_forward_begun_and_not_ended(backend, n):
    cache, model = make(backend, "cpu", CPU), Model("cpu")
    ids, _ = prefill(cache, model, [[1, 2, 3], [4, 5]], "cpu")
    for _ in range(2):  # (decode steps, so that the next one may take the steady path)
        step = cache.begin_forward(ids, [1, 1])
        _write(cache, step, 1, 4.0)
        cache.end_forward(step)
    ctx = cache.begin_tree(ids, [[-1, 0, 1], [-1]])
    cache.begin_forward(ids if n == 1 else ids[1:], [n] * (2 if n == 1 else 1))
    _refused(cache, ctx)
    ctx = cache.begin_tree(ids, [[-1], [-1]])
    cache.begin_forward(ids, [1, 1])
    _refused(cache, ctx)


@BACKENDS
def test_forwards_that_do_not_begin_leave_a_tree_open(backend):
    cache, model = make(backend, "cpu", CPU, pages=12), Model("cpu")
    ids, _ = prefill(cache, model, [[1, 2, 3], [4, 5]], "cpu")
    ctx = cache.begin_tree(ids, [[-1, 0, 1], [-1]])
    with pytest.raises((RuntimeError, AssertionError)):
        cache.begin_forward(ids[:1], [200])
    with pytest.raises(ValueError):
        cache.begin_tree(ids[:1], [[-1, 5]])
    assert cache.end_tree(ctx, _i32([[0, 1, 2], [0, -1, -1]]), _i32([3, 1])) == [3, 1]
