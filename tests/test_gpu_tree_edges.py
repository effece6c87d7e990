"""Calls for trees of drafted tokens at the edges of what the wrappers take."""
import random

import pytest
import torch

from test_gpu_tree import DEV, Setup, _i32, chain, random_tree

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
