"""Speculative decoding through the cache managers (begin_tree, accept_tree, end_tree): a small model that drafts trees and
verifies them greedily decodes the tokens that it decodes one at a time. On the CPU with stand-ins of the kernels that
follow the 64-bit oracle, on the GPU with the kernels themselves.

The model is fp32; its logits are compared as tokens only, so the weights are the first ones with which the two largest
logits of no step of the plain run are closer than 1e-4 (the errors of three layers' fp32 sums are below 1e-5 at logits
of order 1)."""
import random
import types

import numpy as np
import pytest
import torch

import fake_kernels as FK
from nanoslg_amd import kv_cache as KC
from nanoslg_amd.tree_cache import TreeCacheContext
from oracle import kv_oracle
from oracle import tree_oracle as O

L, HQ, HKV, D, V, H = 3, 4, 2, 64, 60, 48
CPU = types.SimpleNamespace(**{k: v for k, v in vars(FK).items() if not k.startswith("__")})


# ---- the kernels' stand-ins ------------------------------------------------------------------


def _split(x, qo):
    qo = qo.tolist()
    return [x[a:b] for a, b in zip(qo, qo[1:])]


def tree_plan(parents, qo_indptr, start, total_q, max_q, q_rows=None, grid_width=0):
    trees = [t.tolist() for t in _split(parents, qo_indptr)]
    assert sum(map(len, trees)) == total_q and max(map(len, trees)) <= max_q
    pos = torch.tensor([s + d for s, t in zip(start.tolist(), trees) for d in O.depths(t)], dtype=torch.int32)
    if q_rows is not None:
        grid = torch.zeros(len(trees) * grid_width, dtype=torch.int32)
        grid[q_rows[:total_q].long()] = pos
        pos = grid
    return O.mask_words(trees, max_q), pos


def _slots(pool, indptr, indices, lpl):
    ps, out = pool.shape[-3], []
    for pages, last in zip(_split(indices, indptr), lpl.tolist()):
        n = (len(pages) - 1) * ps + last if len(pages) else 0
        out.append([int(pages[i // ps]) * ps + i % ps for i in range(n)])
    return out


def paged_tree_attention(q, mask, qo_indptr, total_q, max_q, k_layer, v_layer, kv_indptr, kv_indices, kv_last_page_len,
                         total_pages, k_new=None, v_new=None, sm_scale=None, out=None, workspace=None, q_rows=None, grid_width=0):
    Hkv, D = k_layer.shape[-2:]
    assert total_pages == int(kv_indptr[-1]) and q.shape[0] == (len(qo_indptr) - 1) * grid_width if q_rows is not None else True
    rows = torch.arange(total_q) if q_rows is None else q_rows[:total_q].long()
    out = torch.zeros_like(q)
    k, v = k_layer.view(-1, Hkv, D), v_layer.view(-1, Hkv, D)
    for at, r, m in zip(_slots(k_layer, kv_indptr, kv_indices, kv_last_page_len), _split(rows, qo_indptr), _split(mask, qo_indptr)):
        n = len(r)
        at = torch.tensor(at)
        if k_new is not None:
            k[at[len(at) - n:]], v[at[len(at) - n:]] = k_new.reshape(-1, Hkv, D)[r], v_new.reshape(-1, Hkv, D)[r]
        see = torch.tensor([[bool(int(m[i, j // 32]) >> (j % 32) & 1) for j in range(n)] for i in range(n)])
        out[r] = O.attention(q[r], k[at], v[at], see, sm_scale)[0].to(q.dtype)
    return out


def verify_tree(tokens, parents, qo_indptr, total_q, max_q, target_probs, u_accept, u_next, draft_probs=None, q_rows=None,
                workspace=None):
    assert tokens.dtype == torch.int32 and len(tokens) == len(parents) == len(u_accept) == total_q
    rows = (torch.arange(total_q) if q_rows is None else q_rows[:total_q]).int()
    path, count, token = [], [], []
    for b, (t, x, r, u) in enumerate(zip(*(_split(y, qo_indptr) for y in (parents, tokens, rows, u_accept)))):
        p, nxt = O.verify(t.tolist(), x.tolist(), target_probs, u.tolist(), float(u_next[b]), draft_probs, r.tolist())
        path.append(p + [-1] * (max_q - len(p)))
        count.append(len(p))
        token.append(nxt)
    return tuple(torch.tensor(y, dtype=torch.int32) for y in (path, count, token))


def move_accepted(k_pool, v_pool, path, count, qo_indptr, kv_indptr, kv_indices, kv_last_page_len):
    for b, at in enumerate(_slots(k_pool, kv_indptr, kv_indices, kv_last_page_len)):
        n = int(qo_indptr[b + 1] - qo_indptr[b])
        for pool in (k_pool, v_pool):
            O.move(pool.view(pool.shape[0], -1, *pool.shape[-2:]), at[len(at) - n:], path[b, :int(count[b])].tolist())


for f in (tree_plan, paged_tree_attention, verify_tree, move_accepted):
    setattr(CPU, f.__name__, f)
CPU.MAX_TREE_NODES = 1024


# ---- a model -----------------------------------------------------------------------------------


class Model:
    def __init__(self, dev, seed=0, max_pos=512):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g)
        self.E = r(V, H).to(dev)
        self.W = [[w.to(dev) for w in (r(H, HQ * D) / H ** 0.5, r(H, HKV * D) / H ** 0.5, r(H, HKV * D) / H ** 0.5,
                                       r(HQ * D, H) * (2 / (HQ * D) ** 0.5))] for _ in range(L)]
        self.out = (r(H, V) / H ** 0.5).to(dev)
        self.cos, self.sin = (t.to(dev) for t in kv_oracle.rope_tables(D, max_pos, 10000.0))

    def __call__(self, tokens, ctx, rope=True):
        """Logits [B, S, V] of a [B, S] grid of tokens."""
        B, S = tokens.shape
        x = self.E[tokens.long()]
        for i, (wq, wk, wv, wo) in enumerate(self.W):
            h = x / x.square().mean(-1, keepdim=True).sqrt()
            q, k, v = (h @ wq).view(B, S, HQ, D), (h @ wk).view(B, S, HKV, D), (h @ wv).view(B, S, HKV, D)
            if rope:
                o = ctx.attend_rope(i, q, k, v, self.cos, self.sin, HQ, HKV)
            else:
                q, k = kv_oracle.rope_forward_ref(q, k, self.cos, self.sin, ctx.get_position_ids(S))
                o = ctx.attend(i, q, k, v, HQ, HKV)
            x = x + o @ wo
        return x / x.square().mean(-1, keepdim=True).sqrt() @ self.out


def make(backend, dev, kern, ps=4, pages=96, **kw):
    cfg = KC.KVCacheConfig(num_layers=L, num_kv_heads=HKV, num_qo_heads=HQ, head_dim=D, page_size=ps, max_pages=pages,
                           dtype=kw.pop("dtype", torch.float32), device=dev, backend=backend, max_batch_size=5, max_seq_len=160,
                           enable_prefix_caching=True, share_partial_pages=True, **kw)
    return (KC.PagedKVCache if backend == "paged" else KC.ContiguousKVCache)(cfg, kernels=kern)


def prefill(cache, model, prompts, dev):
    ids = [f"s{b}" for b in range(len(prompts))]
    first = []
    for sid, p in zip(ids, prompts):
        done = cache.allocate_sequence(sid, token_ids=p) if cache.cfg.backend == "paged" else cache.allocate_sequence(sid)
        if cache.cfg.backend == "paged":
            cache.seqs[sid].num_tokens = done
        ctx = cache.begin_forward([sid], [len(p) - done])
        logits = model(torch.tensor([p[done:]], device=dev), ctx)
        cache.end_forward(ctx)
        first.append(int(logits[0, -1].argmax()))
    return ids, first


def plain(backend, dev, kern, model, prompts, steps):
    cache = make(backend, dev, kern)
    ids, last = prefill(cache, model, prompts, dev)
    out = [[t] for t in last]
    for _ in range(steps):
        ctx = cache.begin_forward(ids, [1] * len(ids))
        logits = model(torch.tensor([[o[-1]] for o in out], device=dev), ctx)[:, 0]
        cache.end_forward(ctx)
        top = logits.topk(2).values
        if (top[:, 0] - top[:, 1]).min() < 1e-4:
            return None
        for o, t in zip(out, logits.argmax(-1).tolist()):
            o.append(t)
    return out


def drafted(rng, n, known):
    """A tree of n nodes whose tokens are often the ones to come (known: [0] the root's)."""
    parents, tokens, depth = [-1], [known[0]], [0]
    for j in range(1, n):
        p = max(0, j - 1 - int(rng.expovariate(0.8)))
        right = depth[p] + 1 < len(known) and rng.random() < 0.75
        parents.append(p)
        depth.append(depth[p] + 1)
        tokens.append(known[depth[j]] if right else rng.randrange(V))
    return parents, tokens


def speculative(backend, dev, kern, seed=0, rope=True, draw=False, wide=0, on_device=False, steps=24):
    """Decode with drafted trees; every token is the plain run's."""
    rng = random.Random(seed)
    prompts = [[rng.randrange(V) for _ in range(n)] for n in (9, 1, 14, 30)]
    prompts[3][:14] = prompts[2]  # a shared prefix
    for weights in range(seed, seed + 50, 5):
        model = Model(dev, weights)
        want = plain(backend, dev, kern, model, prompts, steps + 20)
        if want:
            break
    cache = make(backend, dev, kern)
    ids, last = prefill(cache, model, prompts, dev)
    got = [[t] for t in last]
    lengths, accepted = [len(p) for p in prompts], []
    for step in range(steps):
        batch = [b for b in range(4) if len(got[b]) < steps and (rng.random() < 0.8 or b == step % 4)]
        if not batch:
            break
        if step % 5 == 4:  # a plain step between
            ctx = cache.begin_forward([ids[b] for b in batch], [1] * len(batch))
            logits = model(torch.tensor([[got[b][-1]] for b in batch], device=dev), ctx, rope)
            cache.end_forward(ctx)
            for b, t in zip(batch, logits[:, 0].argmax(-1).tolist()):
                got[b].append(t)
                lengths[b] += 1
            continue
        same = rng.randint(1, 13) if on_device or step % 5 == 3 else 0
        trees = [drafted(rng, same or rng.randint(1, 13), want[b][len(got[b]) - 1:]) for b in batch]
        S = max(len(t[0]) for t in trees) + wide
        tokens = torch.tensor([t[1] + [0] * (S - len(t[1])) for t in trees], device=dev)
        parents = torch.tensor([t[0] for t in trees], dtype=torch.int32, device=dev) if on_device else [t[0] for t in trees]
        ctx = cache.begin_tree([ids[b] for b in batch], parents)
        assert isinstance(ctx, TreeCacheContext) and ctx.get_start_pos(0) == lengths[batch[0]]
        pos = ctx.get_position_ids(S).tolist()
        for row, (t, _), b in zip(pos, trees, batch):
            assert row == [lengths[b] + d for d in O.depths(t)] + [0] * (S - len(t))
        logits = model(tokens, ctx, rope)
        if step % 7 == 6:  # the forward is dropped
            continue
        probs = torch.zeros(len(batch), S, V, device=dev).scatter_(2, logits.argmax(-1, keepdim=True), 1.0)
        u, un = torch.rand(len(batch), S).to(dev), torch.rand(len(batch)).to(dev)
        if step % 5 == 2:  # the paths by hand
            paths = [O.verify(t, x, probs[i], [0] * S, 0, None)[0] for i, (t, x) in enumerate(trees)]
            path = torch.tensor([p + [-1] * (S - len(p)) for p in paths], dtype=torch.int32, device=dev)
            counts = cache.end_tree(ctx, path, torch.tensor([len(p) for p in paths], dtype=torch.int32, device=dev))
            after = [int(probs[i, p[-1]].argmax()) for i, p in enumerate(paths)]
        else:
            q = None
            if draw:  # (drafts drawn from rows that are certain: greedy all the same)
                q = torch.zeros(len(batch), S, V)
                for i, (t, x) in enumerate(trees):
                    for j, p in enumerate(t):
                        if p >= 0 and not q[i, p].any():
                            q[i, p, x[j]] = 1
                q = q.to(dev)
            done = cache.accept_tree(ctx, tokens, probs, u, un, q)
            counts, after = done.counts, done.next_tokens.tolist()
            paths = [p[:c] for p, c in zip(done.path.tolist(), counts)]
        for i, b in enumerate(batch):
            got[b] += [trees[i][1][j] for j in paths[i][1:]] + [after[i]]
            lengths[b] += counts[i]
            assert counts[i] == len(paths[i]) and cache._states[ids[b]].num_tokens == lengths[b]
            accepted.append(counts[i] - 1)
        with pytest.raises(ValueError, match="open context"):
            cache.end_tree(ctx, *(done.path, done.path[:, 0]) if step % 5 != 2 else (path, path[:, 0]))
    for _ in range(12):  # plain steps in a row, over pages that rejected nodes opened
        ctx = cache.begin_forward(ids, [1] * 4)
        logits = model(torch.tensor([[o[-1]] for o in got], device=dev), ctx, rope)
        cache.end_forward(ctx)
        for o, t in zip(got, logits[:, 0].argmax(-1).tolist()):
            o.append(t)
    for w, o in zip(want, got):
        assert o[:len(w)] == w[:len(o)]
    assert max(accepted) >= 3 and 0 in accepted
    return cache, ids, got, prompts


CASES = [(b, kw) for b in ("paged", "contiguous")
         for kw in ({}, {"seed": 1, "rope": False}, {"seed": 2, "wide": 3}, {"seed": 3, "on_device": True},
                    {"seed": 4, "draw": True, "rope": False, "wide": 1})]


@pytest.mark.parametrize("backend,kw", CASES)
def test_speculative_decoding_is_plain_decoding(backend, kw):
    cache, ids, got, prompts = speculative(backend, "cpu", CPU, **kw)
    if backend == "paged":  # no page is lost
        for sid, p, o in zip(ids, prompts, got):
            cache.seqs[sid].token_ids = (p + o)[:cache.seqs[sid].num_tokens]
        cache.reset()
        assert cache.pool.num_free + cache.tree.cached_pages == cache.cfg.max_pages - 1


@pytest.mark.gpu
@pytest.mark.parametrize("backend,kw", CASES)
def test_speculative_decoding_is_plain_decoding_gpu(backend, kw):
    from nanoslg_amd import kernels
    speculative(backend, "cuda:0", kernels, **kw)


def rows(cache, sid, layer):
    st = cache._states[sid]
    k, v = cache._kv_layer(layer)
    if cache.cfg.backend != "paged":
        return k[st.slot, :st.num_tokens], v[st.slot, :st.num_tokens]
    at = torch.tensor([int(st.bt[i // cache.cfg.page_size]) * cache.cfg.page_size + i % cache.cfg.page_size
                       for i in range(st.num_tokens)], dtype=torch.long, device=k.device)
    return k.reshape(-1, HKV, D)[at], v.reshape(-1, HKV, D)[at]


def accepted_rows(backend, dev, kern, dtype, poison):
    """The accepted nodes' rows lie behind the sequence's, in every layer; what rejected ones hold does not reach what
    follows."""
    rng, g = random.Random(7), torch.Generator().manual_seed(7)
    cache = make(backend, dev, kern, dtype=dtype)
    lens, ns = [7, 0, 20], [9, 4, 1]
    ids = ["a", "b", "c"]
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).to(dev)
    kept = {(s, i): ([], []) for s in ids for i in range(L)}
    for sid, n in zip(ids, lens):
        cache.allocate_sequence(sid)
        if n:
            ctx = cache.begin_forward([sid], [n])
            for i in range(L):
                k, v = r(1, n, HKV, D), r(1, n, HKV, D)
                ctx.attend(i, r(1, n, HQ, D), k, v, HQ, HKV)
                for pool, x in zip(kept[sid, i], (k, v)):
                    pool.append(x[0])
            cache.end_forward(ctx)
    paths = [[0, 2, 5, 8], [0], [0]]
    ctx = cache.begin_tree(ids, [[-1] + [rng.randrange(j) for j in range(1, n)] for n in ns])
    for i in range(L):
        k, v = r(3, 9, HKV, D), r(3, 9, HKV, D)
        for b, (sid, p) in enumerate(zip(ids, paths)):
            for pool, x in zip(kept[sid, i], (k, v)):
                pool.append(x[b, p].clone())
            if poison:
                bad = [j for j in range(ns[b]) if j not in p]
                k[b, bad], v[b, bad] = float("inf"), float("nan")
        ctx.attend(i, r(3, 9, HQ, D), k, v, HQ, HKV)
    path = torch.tensor([p + [-1] * (9 - len(p)) for p in paths], dtype=torch.int32, device=dev)
    assert cache.end_tree(ctx, path, torch.tensor([4, 1, 1], dtype=torch.int32, device=dev)) == [4, 1, 1]
    for (sid, i), pools in kept.items():
        for have, x in zip(rows(cache, sid, i), pools):
            assert torch.equal(have, torch.cat(x))
    # a decode step, and a chunk of three, over what is left
    for n in (1, 3):
        ctx = cache.begin_forward(ids, [n] * 3)
        for i in range(L):
            q, k, v = r(3, n, HQ, D), r(3, n, HKV, D), r(3, n, HKV, D)
            out = ctx.attend(i, q, k, v, HQ, HKV).view(3, n, HQ, D)
            for b, sid in enumerate(ids):
                for pool, x in zip(kept[sid, i], (k, v)):
                    pool.append(x[b])
                want, mag, _ = O.attention(q[b], *(torch.cat(x) for x in kept[sid, i]), torch.tril(torch.ones(n, n)).bool())
                # (a rounding of the output, of the probabilities and of the sums, as the kernels' own tests count them)
                u = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
                assert ((out[b].double() - want).abs() <= u * want.abs() + (4 * u + 2.0 ** -15) * mag + 2.0 ** -20).all(), (n, i, sid)
        cache.end_forward(ctx)


@pytest.mark.parametrize("backend", ["paged", "contiguous"])
@pytest.mark.parametrize("poison", [False, True])
def test_accepted_rows(backend, poison):
    accepted_rows(backend, "cpu", CPU, torch.float32, poison)


@pytest.mark.gpu
@pytest.mark.parametrize("backend", ["paged", "contiguous"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("poison", [False, True])
def test_accepted_rows_gpu(backend, dtype, poison):
    from nanoslg_amd import kernels
    accepted_rows(backend, "cuda:0", kernels, dtype, poison)


def test_shared_pages_are_copied_before_a_tree_writes_them():
    cache, model = make("paged", "cpu", CPU), Model("cpu")
    prompt = list(range(10))
    (a,), _ = prefill(cache, model, [prompt], "cpu")
    cache.release_sequence(a)
    for sid in ("x", "y"):  # both start on the cached pages, the partial one included
        done = cache.allocate_sequence(sid, token_ids=prompt + [11])
        cache.seqs[sid].num_tokens = done
        assert done == 10
    before = [rows(cache, "y", i)[0].clone() for i in range(L)]
    ctx = cache.begin_tree(["x", "y"], [[-1, 0, 0], [-1, 0, 1]])
    model(torch.tensor([[11, 3, 4], [12, 5, 6]]), ctx)
    assert int(cache.seqs["x"].bt[2]) != int(cache.seqs["y"].bt[2]) and int(cache.seqs["x"].bt[1]) == int(cache.seqs["y"].bt[1])
    assert cache.end_tree(ctx, torch.tensor([[0, 2, -1], [0, 1, 2]], dtype=torch.int32), torch.tensor([2, 3], dtype=torch.int32)) == [2, 3]
    assert [cache.seqs[s].num_tokens for s in "xy"] == [12, 13]
    assert all(torch.equal(rows(cache, "y", i)[0][:10], before[i]) for i in range(L))
    assert [int(cache.pool.tokens_used[cache.seqs[s].bt[p]]) for s in "xy" for p in (2, 3) if p < cache.seqs[s].n_pages] == [4, 0, 4, 1]


@pytest.mark.parametrize("backend", ["paged", "contiguous"])
def test_refusals(backend):
    cache, model = make(backend, "cpu", CPU), Model("cpu")
    ids, _ = prefill(cache, model, [[1, 2, 3], [4, 5]], "cpu")
    for seqs, parents in [(ids, [[-1, 0]]), (ids, [[-1], []]), (ids, [[-1, 1], [-1]]), (ids, [[-1, -1], [-1]]), (ids, [[0], [-1]]),
                          ([], []), ([ids[0], ids[0]], [[-1], [-1]]), (ids, [[-1, 0, 3], [-1]]),
                          (ids[:1], [list(range(-1, 1024))]), (ids, torch.full((2, 2), -1)), (ids, torch.full((3, 2), -1).int()),
                          (ids, torch.full((2, 0), -1).int())]:
        with pytest.raises(ValueError, match="begin_tree"):
            cache.begin_tree(seqs, parents)
    assert [cache._states[s].num_tokens for s in ids] == [3, 2]
    ctx = cache.begin_tree(ids, [[-1, 0, 0], [-1, 0]])
    tok, u, un, p = torch.zeros(2, 3).long(), torch.rand(2, 3), torch.rand(2), torch.full((2, 3, V), 1 / V)
    with pytest.raises(ValueError, match="accept_tree"):
        cache.end_forward(ctx)
    x = torch.zeros(2, 2, HQ, D)
    with pytest.raises(ValueError, match="columns"):
        ctx.attend(0, x, x[:, :, :HKV], x[:, :, :HKV], HQ, HKV)
    with pytest.raises(ValueError, match="columns"):
        ctx.attend_rope(0, x, x[:, :, :HKV], x[:, :, :HKV], model.cos, model.sin, HQ, HKV)
    y = torch.zeros(2, 3, HQ, D)
    with pytest.raises(IndexError):
        ctx.attend_rope(0, y, y[:, :, :HKV], y[:, :, :HKV], model.cos[:4], model.sin[:4], HQ, HKV)
    ctx.attend_rope(0, y, y[:, :, :HKV], y[:, :, :HKV], model.cos[:5], model.sin[:5], HQ, HKV)  # depths, not nodes
    for args in [(tok[:, :2], p, u, un), (tok, p[:, :2], u, un), (tok, p, u[:1], un), (tok, p[0], u, un), (tok, p, u, un, p[:, :, 1:])]:
        with pytest.raises(ValueError, match="accept_tree"):
            cache.accept_tree(ctx, *args)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)
    for path, count in [([[0, 1]], [2]), ([[0, 3, -1], [0, 1, -1]], [2, 2]), ([[0, 0, -1], [0, 1, -1]], [2, 2]),
                        ([[2, 1, -1], [0, 1, -1]], [2, 2]), ([[0, 1, 2], [0, 1, -1]], [3, 3]), ([[0], [0]], [2, 1]), ([[0], [0]], [-1, 1])]:
        with pytest.raises(ValueError, match="end_tree"):
            cache.end_tree(ctx, i32(path), i32(count))
    other = make(backend, "cpu", CPU)
    with pytest.raises(ValueError, match="open context"):
        other.end_tree(ctx, i32([[0], [0]]), i32([1, 1]))
    plain_ctx = cache.begin_forward(ids, [1, 1])
    with pytest.raises(ValueError, match="open context"):
        cache.end_tree(plain_ctx, i32([[0], [0]]), i32([1, 1]))
    cache.end_forward(plain_ctx)
    with pytest.raises(ValueError, match="has changed"):
        cache.end_tree(ctx, i32([[0], [0]]), i32([1, 1]))
    assert [cache._states[s].num_tokens for s in ids] == [4, 3]
    assert cache.end_tree(cache.begin_tree(ids, [[-1, 0], [-1]]), i32([[-1, -1]] * 2), i32([0, 0])) == [0, 0]


@pytest.mark.parametrize("backend", ["paged", "contiguous"])
def test_an_ended_context_attends_nothing(backend):
    cache, model = make(backend, "cpu", CPU), Model("cpu")
    ids, _ = prefill(cache, model, [[1, 2, 3]], "cpu")
    parents = torch.tensor([[-1, 0, 1]], dtype=torch.int32)
    ctx = cache.begin_tree(ids, parents)
    parents.fill_(-1)  # the context has its own
    probs = torch.zeros(1, 3, V).scatter_(2, torch.tensor([[[5], [6], [7]]]), 1.0)
    done = cache.accept_tree(ctx, torch.tensor([[4, 5, 6]]), probs, torch.zeros(1, 3), torch.zeros(1))
    assert done.counts == [3] and done.next_tokens.tolist() == [7]
    x = torch.zeros(1, 3, HQ, D)
    for call in (lambda: ctx.attend(0, x, x[:, :, :HKV], x[:, :, :HKV], HQ, HKV),
                 lambda: ctx.attend_rope(0, x, x[:, :, :HKV], x[:, :, :HKV], model.cos, model.sin, HQ, HKV)):
        with pytest.raises(ValueError, match="has ended"):
            call()


@pytest.mark.parametrize("backend", ["paged", "contiguous"])
def test_eight_bit_caches_are_refused(backend):
    cache = make(backend, "cpu", CPU, dtype=torch.float16, cache_dtype=torch.int8)
    cache.allocate_sequence("a")
    with pytest.raises(ValueError, match="cache_dtype"):
        cache.begin_tree(["a"], [[-1, 0]])
