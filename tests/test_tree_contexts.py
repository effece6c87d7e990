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


@BACKENDS
@pytest.mark.parametrize("rope", [True, False])
def test_a_forward_on_another_stream_holds_what_it_reads(backend, rope, monkeypatch):
    """Every tensor of the context that a kernel is given on another stream than begin_tree's is recorded there, once for each
    stream and width; on begin_tree's own nothing is."""
    from types import SimpleNamespace

    from nanoslg_amd import tree_cache
    given, held, now = [], [], [7]
    calls = SimpleNamespace(**vars(CPU))
    for name in ("paged_tree_attention", "rope_append"):
        def call(*a, _f=getattr(CPU, name), **kw):
            given.extend(t.data_ptr() for t in (*a, *kw.values()) if isinstance(t, torch.Tensor) and t.dtype == torch.int32)
            return _f(*a, **kw)
        setattr(calls, name, call)
    monkeypatch.setattr(tree_cache, "_raw_stream", lambda device: now[0])
    monkeypatch.setattr(tree_cache, "_current_stream", lambda index: now[0])
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, stream: held.append((t.data_ptr(), stream)))
    cache, model = make(backend, "cpu", calls), Model("cpu")
    ids, _ = prefill(cache, model, [[1, 2, 3], [4, 5]], "cpu")
    ctx = cache.begin_tree(ids, [[-1, 0, 0], [-1]])
    held.clear()

    def forward(S):
        given.clear()
        model(torch.zeros(2, S, dtype=torch.long), ctx, rope)

    forward(3)
    assert not held
    for now[0], S in ((8, 3), (8, 5), (9, 5), (7, 6), (8, 6)):
        before = len(held)
        forward(S)
        assert given and {(p, now[0]) for p in given} <= set(held) and len(held) > before
        before = len(held)
        forward(S)
        assert len(held) == before


def test_trees_of_roots_have_a_plan_of_their_own():
    """Later decode steps, of any sequences, do not write the plan of an open tree."""
    cache, model = make("paged", "cpu", CPU), Model("cpu")
    ids, _ = prefill(cache, model, [[1, 2, 3], [4, 5]], "cpu")
    for _ in range(2):
        step = cache.begin_forward(ids, [1, 1])
        _write(cache, step, 1, 4.0)
        cache.end_forward(step)
    assert cache._dev_plan is not None
    seen = []
    begin = cache._begin_steady_decode
    cache._begin_steady_decode = lambda *a: seen.append(a) or begin(*a)
    ctx = cache.begin_tree(ids, [[-1], [-1]])
    assert not seen
    assert cache.end_tree(ctx, _i32([[0], [0]]), _i32([1, 1])) == [1, 1]


@pytest.mark.gpu
@BACKENDS
def test_a_context_dropped_while_its_forward_runs_elsewhere(backend):
    """What is allocated meanwhile does not take the memory that the waiting kernels will read."""
    from nanoslg_amd import kernels
    dev = "cuda:0"
    g = torch.Generator(device=dev).manual_seed(0)
    cache, model = make(backend, dev, kernels), Model(dev)
    ids, _ = prefill(cache, model, [[1, 2, 3] * 9, [4, 5]], dev)
    trees = [[-1, 0, 0, 1, 3, 3], [-1, 0]]
    q, k, v = (torch.randn(2, 6, h, D, generator=g, device=dev) for h in (HQ, HKV, HKV))
    ctx = cache.begin_tree(ids, trees)
    want = ctx.attend(0, q, k, v, HQ, HKV).clone()
    side = torch.cuda.Stream()
    for _ in range(2):
        ctx = cache.begin_tree(ids, trees)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)
            got = ctx.attend(0, q, k, v, HQ, HKV)
        del ctx
        taken = [torch.zeros(n, dtype=torch.int32, device=dev) for n in (1, 60, 120, 500, 1000, 5000) for _ in range(20)]
        torch.cuda.synchronize()
        assert torch.equal(got, want) and not any(t.any() for t in taken)


@BACKENDS
@pytest.mark.parametrize("nodes", [1, 3])
def test_numbers_and_tokens_as_parts_of_wider_tensors(backend, nodes):
    """A column of one tensor of uniform numbers, tokens of a longer buffer: the call takes them as their values."""
    from types import SimpleNamespace
    V, B = 60, 2
    calls, strided = SimpleNamespace(**vars(CPU)), []

    def verify(tokens, parents, qo, total, max_q, probs, u_accept, u_next, **kw):
        strided.extend(not t.is_contiguous() for t in (tokens, parents, u_accept, u_next))
        return CPU.verify_tree(tokens, parents, qo, total, max_q, probs, u_accept, u_next, **kw)

    calls.verify_tree = verify
    done = []
    for parts in (False, True):
        cache, model = make(backend, "cpu", calls), Model("cpu")
        ids, _ = prefill(cache, model, [[1, 2, 3], [4, 5]], "cpu")
        g = torch.Generator().manual_seed(1)
        u = torch.rand(B, 2 * nodes + 2, generator=g)
        tokens = torch.randint(0, 3, (B, 2 * nodes), generator=g, dtype=torch.int32)
        probs = torch.zeros(B, nodes, V)
        probs[:, :, :3] = 1 / 3
        ctx = cache.begin_tree(ids, [[-1] + [0] * (nodes - 1)] * B)
        args = (tokens[:, ::2], u[:, :2 * nodes:2], u[:, -1])
        tok, ua, un = args if parts else (a.clone(memory_format=torch.contiguous_format) for a in args)
        done.append(cache.accept_tree(ctx, tok, probs, ua, un))
    assert not any(strided)
    assert torch.equal(done[0].path, done[1].path) and torch.equal(done[0].next_tokens, done[1].next_tokens)


@BACKENDS
@pytest.mark.parametrize("uniform,wide", [(True, 0), (True, 2), (False, 0), (False, 3)])
def test_what_the_attention_call_is_told(backend, uniform, wide):
    """The pages of the call's block table, always; with q_rows the rows of a grid, without them the ragged rows alone."""
    from types import SimpleNamespace
    calls, seen = SimpleNamespace(**vars(CPU)), []

    def attention(q, mask, qo, total, max_q, k, v, indptr, indices, lpl, pages, **kw):
        seen.append(kw.get("q_rows") is not None)
        assert pages == int(indptr[-1]) == indices[:pages].numel() and total == int(qo[-1])
        rows = (len(qo) - 1) * kw["grid_width"] if seen[-1] else total
        assert q.shape[0] == rows and (kw.get("k_new") is None or kw["k_new"].shape[:-2].numel() == rows)
        return CPU.paged_tree_attention(q, mask, qo, total, max_q, k, v, indptr, indices, lpl, pages, **kw)

    calls.paged_tree_attention = attention
    cache, model = make(backend, "cpu", calls), Model("cpu")
    ids, _ = prefill(cache, model, [list(range(9)), [4, 5]], "cpu")
    ctx = cache.begin_tree(ids, [[-1, 0, 0], [-1, 0, 1] if uniform else [-1]])
    for rope in (True, False):
        model(torch.zeros(2, 3 + wide, dtype=torch.long), ctx, rope)
    assert len(seen) == 2 * L and all(s == (wide > 0 or not uniform) for s in seen)


@pytest.mark.gpu
def test_a_graph_step_drops_an_open_tree():
    from nanoslg_amd import kernels
    from nanoslg_amd import kv_cache as KC
    dev = "cuda:0"
    cache, model = make("paged", dev, kernels), Model(dev)
    ids, _ = prefill(cache, model, [[1, 2, 3], [4, 5]], dev)
    q, k, v = (torch.zeros(2, 1, h, D, device=dev) for h in (HQ, HKV, HKV))
    graph = KC.DecodeGraph(cache, ids, lambda ctx: [ctx.attend(i, q, k, v, HQ, HKV) for i in range(L)])
    ctx = cache.begin_tree(ids[:1], [[-1, 0]])
    graph.step()
    torch.cuda.synchronize()
    x = torch.zeros(1, 2, HQ, D, device=dev)
    with pytest.raises(ValueError, match="have changed"):
        ctx.attend(0, x, x[:, :, :HKV], x[:, :, :HKV], HQ, HKV)
    with pytest.raises(ValueError, match="has changed"):
        cache.end_tree(ctx, torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev))


@pytest.mark.gpu
@BACKENDS
def test_a_tree_forward_in_a_graph(backend):
    """Captured on the capture's own stream, replayed over other rows, the context dropped behind the last replay."""
    from nanoslg_amd import kernels
    dev = "cuda:0"
    g = torch.Generator(device=dev).manual_seed(0)
    cache, model = make(backend, dev, kernels), Model(dev)
    ids, _ = prefill(cache, model, [[1, 2, 3] * 9, [4, 5]], dev)
    ctx = cache.begin_tree(ids, [[-1, 0, 0, 1, 3, 3], [-1, 0]])
    q, k, v = (torch.randn(2, 6, h, D, generator=g, device=dev) for h in (HQ, HKV, HKV))

    def forward():
        return [ctx.attend_rope(i, q, k, v, model.cos, model.sin, HQ, HKV) for i in range(L)]

    forward()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = forward()
    for _ in range(3):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g, device=dev))
        want = [o.clone() for o in forward()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    counts = cache.end_tree(ctx, _i32([[0, 2, -1], [0, 1, -1]]).to(dev), _i32([2, 2]).to(dev))
    assert counts == [2, 2]
    del ctx, graph
    torch.cuda.synchronize()
