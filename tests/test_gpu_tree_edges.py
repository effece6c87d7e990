"""Calls for trees of drafted tokens at the edges of what the wrappers take."""
import math
import random

import pytest
import torch

from test_gpu_tree import DEV, U, Setup, _i32, chain, random_tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("empty", [True, False])  # q_rows without entries, or with some that no node has
@pytest.mark.parametrize("max_q", [0, 5])
def test_grids_without_nodes_are_zeroed(empty, max_q):
    from nanoslg_amd import kernels
    B, S, W = 3, 7, (max_q + 31) // 32
    zeros = _i32([0] * (B + 1))
    q_rows = _i32([] if empty else [1, 2])
    none = _i32([])
    held = torch.full((B * S,), 7, dtype=torch.int32, device=DEV)  # (its memory is the positions' next)
    del held
    mask, pos = kernels.tree_plan(none, zeros, _i32([4, 0, 9]), 0, max_q, q_rows=q_rows, grid_width=S)
    assert mask.shape == (0, W) and pos.shape == (B * S,) and not pos.any()
    for dtype in (torch.float16, torch.float32):
        q = torch.randn(B * S, 8, 128, device=DEV).to(dtype)
        pool = torch.randn(4, 16, 2, 128, device=DEV).to(dtype)
        new = torch.randn(B * S, 2, 128, device=DEV).to(dtype)
        out = torch.full_like(q, 7)
        k, v = pool.clone(), pool.clone()
        for kw in ({}, {"k_new": new, "v_new": new}):
            out.fill_(7)
            kernels.paged_tree_attention(q, mask, zeros, 0, max_q, k, v, _i32([0, 1, 1, 2]), _i32([1, 2]), _i32([4, 0, 9]), 2, out=out,
                                         q_rows=q_rows, grid_width=S, **kw)
            assert not out.any() and torch.equal(k, pool) and torch.equal(v, pool)
    path, count, token = kernels.verify_tree(none, none, zeros, 0, max_q, torch.rand(B * S, 9, device=DEV), torch.zeros(0, device=DEV),
                                             torch.rand(B, device=DEV), q_rows=q_rows)
    assert path.shape == (B, max_q) and (path == -1).all() and not count.any() and (token == -1).all()


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("dtype,D,nodes,ps", [(torch.float16, 128, 20, 16), (torch.bfloat16, 128, 20, 16), (torch.bfloat16, 64, 60, 1),
                                              (torch.float16, 256, 9, 16), (torch.float32, 128, 20, 16), (torch.bfloat16, 128, 90, 16)])
def test_infinite_values_of_cached_tokens(dtype, D, nodes, ps, fused, workspace):
    """Every row sees the tokens before its tree: an infinite element of their values makes the output's element that
    infinity (both signs, or NaN: NaN), at a token of a weight of 1, of ordinary and of small weights, and the others stay exact."""
    from test_gpu_tree_exact import _whole
    trees = [random_tree(random.Random(1), nodes), chain(3), random_tree(random.Random(2), nodes)]
    s = Setup(5, [700, 0, 1301], trees, dtype, 8, 2, D, ps)
    # sequence 2's token 9 outweighs all others of KV head 0: its weight is 1 to the last bit
    at = s.slots(2)
    s.k.view(-1, 2, D)[at[9], 0] = 0
    s.k.view(-1, 2, D)[at[9], 0, 0] = 240
    s.q[s.n[0] + 3:, :4, 0] = 8
    k, v = s.written()
    want = _formula(s, k, v)
    inf = float("inf")
    marks = [(2, 9, 0, 5, inf), (2, 9, 1, 6, -inf), (2, 1290, 1, 7, inf), (0, 0, 0, 8, inf), (0, 699, 0, 8, inf), (0, 350, 1, 9, -inf),
             (0, 351, 1, 10, inf), (0, 13, 1, 10, -inf), (2, 640, 1, 11, float("nan"))]
    for b, t, h, d, x in marks:
        for pool in (s.v, v):
            pool.view(-1, 2, D)[s.slots(b)[t], h, d] = x
    if not fused:
        s.k, s.v = k.clone(), v.clone()
    if workspace:
        out = s.run(fused)
    else:
        s.k_new, s.v_new = (s.k_new, s.v_new) if fused else (None, None)
        out = _whole(s, D ** -0.5)
    hit = {(0, 0, 8): inf, (0, 1, 9): -inf, (0, 1, 10): None, (2, 0, 5): inf, (2, 1, 6): -inf, (2, 1, 7): inf, (2, 1, 11): None}
    o = out.clone()
    for (b, h, d), x in hit.items():
        rows = slice(s.qo[b], s.qo[b + 1])
        got = out[rows, 4 * h:4 * h + 4, d]
        assert (got == x).all() if x else got.isnan().all(), (b, h, d, got)
        o[rows, 4 * h:4 * h + 4, d] = want[rows, 4 * h:4 * h + 4, d].to(dtype)
    assert o.isfinite().all()
    s.n_rows = s.T
    s.check(o, *s.clean)


def _formula(s, k, v):
    """The outputs in 64 bits over pools k and v, which the setup keeps for check()."""
    from oracle import tree_oracle as O
    s.clean = (k.clone(), v.clone())
    return torch.cat([O.attention(s.q[s.qo[b]:s.qo[b + 1]], k.view(-1, s.Hkv, s.D)[s.slots(b)], v.view(-1, s.Hkv, s.D)[s.slots(b)], s.see[b])[0]
                      for b in range(s.B)])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bits", [0, 12, 24, 31, 40, 90])
@pytest.mark.parametrize("ctx", [40, 600])
def test_infinite_values_of_weak_keys(dtype, bits, ctx):
    """One cached key 2^bits times as heavy as all others, one of which has an infinite value: the result is infinite there and
    the heavy key's elsewhere, off by the others' N 2^-bits and what tests/test_gpu_tree_exact.py counts."""
    s = Setup(2, [ctx], [chain(3)], dtype, 4, 1, 128)
    s.k.zero_(), s.k_new.zero_(), s.v.zero_(), s.v_new.zero_(), s.q.zero_()
    at = s.slots(0)
    s.k.view(-1, 1, 128)[at[3], 0, 0], s.q[:, :, 0] = 1, 1
    s.v.view(-1, 1, 128)[at[3]] = 1
    s.v.view(-1, 1, 128)[at[33], 0, 17] = float("inf")
    out = s.run(sm_scale=max(bits, 1e-6) * math.log(2))
    assert (out[:, :, 17] == float("inf")).all()
    rest = torch.cat([out[:, :, :17], out[:, :, 18:]], 2).double()
    for t in range(3):
        want = 1 / (1 + (ctx + t) * 2.0 ** -bits)  # (node t sees ctx tokens and t + 1 nodes)
        tol = U[dtype] * want + 2.0 ** -15 * want + (ctx + 3) * 2.0 ** -24
        assert ((rest[t] - want).abs() <= tol).all()


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("ctx,ps", [(4000, 16), (4000, 5000), (4400, 5000)])
def test_keys_on_both_sides_of_what_the_caches_hold(ctx, ps, workspace):
    """16 sequences of 4000 tokens are 246 MiB of K and V, of 4400 271, on both sides of 256: the longer ones' are loaded past the caches, by their lengths
    and not by the pages that they have."""
    from test_gpu_tree_exact import _whole
    s = Setup(ctx, [ctx - 9 * b for b in range(16)], [random_tree(random.Random(b), 8) for b in range(16)], torch.float16, 8, 8, 128, ps)
    s.k, s.v = s.written()
    if not workspace:
        s.k_new = s.v_new = None
    out = s.run(False) if workspace else _whole(s, 128 ** -0.5)
    s.check(out, s.k, s.v)


@pytest.mark.parametrize("dtype,D,ps,ctx", [(torch.float16, 128, 1, 3000), (torch.bfloat16, 64, 1, 5200), (torch.float32, 128, 1, 2100),
                                            (torch.float16, 256, 2, 4500), (torch.bfloat16, 128, 3, 7001)])
@pytest.mark.parametrize("pages", [None, 1])  # no scratch: all keys by one workgroup; spans for a page: nearly so
def test_more_pages_than_a_window(dtype, D, ps, ctx, pages):
    """More than 1024 pages of a sequence in one workgroup's keys: their places are loaded anew on the way, in the plain blocks and
    in those of the tree."""
    from test_gpu_tree_exact import _whole
    s = Setup(ctx, [ctx, 1023 * ps, 1024 * ps + 5], [random_tree(random.Random(n), n) for n in (33, 4, 70)], dtype, 4, 1, D, ps)
    k, v = s.written()
    out = _whole(s, D ** -0.5) if pages is None else s.run(total_pages=pages)
    s.check(out, k, v)
    assert torch.equal(s.k, k) and torch.equal(s.v, v)


def test_counts_past_a_tree_or_a_path_move_nothing():
    """The first count entries of such a path are not rising nodes of the tree: the sequence is left as it is."""
    from nanoslg_amd import kernels
    s = Setup(7, [10, 20, 30, 5], [chain(3), chain(6), chain(6), chain(4)], torch.float16, 2, 2, 64, 16, layers=2)
    k, v = s.k.clone(), s.v.clone()
    path = _i32([[1, 2, -1, -1], [1, 3, 4, 5], [1, 3, 4, 5], [-1] * 4])
    kernels.move_accepted(s.k, s.v, path, _i32([4, 5, 3, -2]), s.qo, s.indptr, s.indices, s.last)
    at = s.slots(2)[30:].tolist()
    for pool in (k, v):
        flat = pool.view(2, -1, 2, 64)
        for i, node in enumerate((1, 3, 4)):
            flat[:, at[i]] = flat[:, at[node]].clone()
    assert torch.equal(s.k, k) and torch.equal(s.v, v)
