"""Speculative decoding on the caches: a forward over trees of drafted tokens, ended with the accepted ones.

One step with any drafter is

    ctx = cache.begin_tree(seq_ids, parents)        # a tree for each sequence
    logits = model(tokens, ctx)                     # ctx.get_position_ids, and attend / attend_rope in every layer
    done = cache.accept_tree(ctx, tokens, probs, u_accept, u_next, draft_probs)

Node 0 of a tree, its root, is the sequence's last sampled token, whose K/V is not cached yet; the others are drafted.
parents[j] < j is node j's parent; a node's children are tried in the order of their indices. The forward writes the nodes' K/V
behind the sequence's tokens; each node sees those tokens, its ancestors and itself, and has the position of a token behind its
ancestors. accept_tree verifies the drafted tokens (``kernels.verify_tree``), moves the accepted nodes' K/V together in
every layer and advances the sequences by them; the token that follows them is the next step's root. end_tree ends a
forward with paths that the caller has found. A context that is dropped leaves its sequences as they were; it is dropped by
the next forward of any of its sequences (begin_forward, begin_tree, a DecodeGraph's step) and by a sequence's release, if not before.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Sequence, Union

import numpy as np
import torch

from .kv_cache import CacheContext, _current_stream, _upload_i32

Trees = Union[Sequence[Sequence[int]], torch.Tensor]


def _host_trees(parents: Sequence[Sequence[int]]):
    """(node counts, flat parents) of trees given as lists."""
    counts = [len(t) for t in parents]
    flat = np.fromiter((p for t in parents for p in t), np.int64, sum(counts))
    first = np.cumsum([0] + counts[:-1]) if counts else np.zeros(0, np.int64)
    node = np.arange(flat.size) - np.repeat(first, counts)
    if not np.where(node == 0, flat == -1, (flat >= 0) & (flat < node)).all():
        raise ValueError("begin_tree: node 0 is the root (parent -1) and every other node's parent lies before it")
    return counts, flat


def _raw_stream(device: torch.device) -> int:
    """The current stream's handle."""
    return torch._C._cuda_getCurrentRawStream(device.index) if device.type == "cuda" else 0


class TreeCacheContext(CacheContext):
    """The context of a forward over trees (a manager's begin_tree). Tensors are [B, S, ...] grids, S at least the largest
    tree's nodes, tree b's nodes the first columns of row b; outputs of the other columns are zero. A forward may run
    on any stream that waits for the one begin_tree ran on; the context may be dropped while it runs there."""

    is_tree = True

    def __init__(self, cache, seq_ids: Sequence[str], parents: Trees):
        kern, pools = cache.kernels, cache._kv_pools
        device = pools.k.device
        seq_ids = list(seq_ids)
        if pools.k_scale is not None:
            # (an accepted token's codes would be rounded once more where it moves to a block of another scale)
            raise ValueError("begin_tree: trees need a cache in the model's own dtype (no cache_dtype)")
        if not seq_ids or len(set(seq_ids)) != len(seq_ids):
            raise ValueError("begin_tree: one or more sequences, each once")
        if isinstance(parents, torch.Tensor):
            if parents.dim() != 2 or parents.dtype != torch.int32 or parents.device != device:
                raise ValueError(f"begin_tree: parents as a tensor must be int32 [B, nodes] on {device}")
            counts, self._host_parents = [parents.shape[1]] * parents.shape[0], None
        else:
            counts, self._host_parents = _host_trees(parents)
        if len(counts) != len(seq_ids) or min(counts) < 1 or max(counts) > kern.MAX_TREE_NODES:
            raise ValueError(f"begin_tree: a tree of 1 to {kern.MAX_TREE_NODES} nodes for each of {len(seq_ids)} sequences")

        ctx = cache._begin_nodes(seq_ids, counts)  # pages, copy-on-write, block table
        self.cache = cache
        self.seq_ids, self.new_token_counts, self.input_offsets = ctx.seq_ids, counts, [0] * len(counts)
        self.batch_size, self.seq_lens, self.start_positions = ctx.batch_size, ctx.seq_lens, ctx.start_positions
        self.max_kv_len = ctx.max_kv_len
        self._plan, self._max_q, self._total = ctx._plan, max(counts), sum(counts)
        self._uniform = min(counts) == self._max_q
        self._open, self._live = True, [True]  # not ended; not dropped (kv_cache._drop_trees)
        start = np.asarray(self.start_positions, np.int32)
        if self._host_parents is None:
            (self._start,) = _upload_i32([start], device)
            self._parents = parents.reshape(-1).clone()  # (the caller may write the next trees there)
        else:
            self._start, self._parents = _upload_i32([start, self._host_parents.astype(np.int32)], device)
        self._mask, pos = kern.tree_plan(self._parents, self._plan.qo_indptr, self._start, self._total, self._max_q,
                                         **self._rows(self._max_q))
        self._pos = {self._max_q: pos}  # by grid width
        self._device, self._stream, self._used_on = device, _raw_stream(device), set()
        cache._open_trees.update(dict.fromkeys(seq_ids, self._live))

    def _rows(self, S: int):
        """The kernels' row arguments for [B, S] grids."""
        if not self._open or not self._live[0]:
            raise ValueError("the context's forward has ended" if not self._open else "the context's sequences have changed since begin_tree")
        if S < self._max_q:
            raise ValueError(f"the input grid has {S} columns; this forward's trees need {self._max_q}")
        return {} if self._uniform and S == self._max_q else {"q_rows": self._plan.rows_for(S), "grid_width": S}

    def _pos_for(self, S: int) -> torch.Tensor:
        """int32 positions of the [B, S] grid (zeros on columns without a node)."""
        p = self._pos.get(S)
        if p is None:
            grid = self._pos[self._max_q].view(self.batch_size, self._max_q)
            p = torch.cat([grid, grid.new_zeros(self.batch_size, S - self._max_q)], 1) if S > self._max_q else grid[:, :S]
            p = self._pos[S] = p.reshape(-1)
        return p

    def get_position_ids(self, S: int) -> torch.Tensor:
        return self._pos_for(S).view(self.batch_size, S).long()

    def get_start_pos(self, idx: int = 0) -> int:
        return self.start_positions[idx]

    def _check_positions(self, limit: int) -> None:
        """Positions are inside rope tables of `limit` rows. A node's depth is below its index; only where that does not
        settle it, the depths are counted (parents on the device: the trees are taken as chains)."""
        last = max(s + n - 1 for s, n in zip(self.start_positions, self.new_token_counts))
        if last >= limit and self._host_parents is not None:
            first, last = 0, 0
            for s, n in zip(self.start_positions, self.new_token_counts):
                depth = [s] * n
                for j, p in enumerate(self._host_parents[first:first + n].tolist()):
                    if j:
                        depth[j] = depth[p] + 1
                first, last = first + n, max(last, max(depth))
        if last >= limit:
            raise IndexError(f"position {last} is outside the rope tables ({limit} rows)")

    def _hold(self, S: int) -> None:
        """The memory of what an attend of this width reads is given back behind the current stream's work too, where that is not
        the stream which it was made on."""
        raw = _raw_stream(self._device)
        if (raw == self._stream and not self._used_on) or (raw, S) in self._used_on:
            return
        self._used_on.add((raw, S))
        stream, plan = _current_stream(self._device.index), vars(self._plan)
        own = [self._mask, self._start, self._parents, *self._pos.values()]
        for x in (*plan.values(), *(t for d in plan.values() if isinstance(d, dict) for t in d.values())):
            if isinstance(x, torch.Tensor) and x.device == self._device:
                own.append(x)
        for t in own:
            t.record_stream(stream)

    def _attend(self, q, k_layer, v_layer, **new):
        plan = self._plan
        B, S, Hq, D = q.shape
        rows = self._rows(S)
        self._hold(S)
        # (scratch from the allocator: forwards of one cache may run on several streams)
        out = self.cache.kernels.paged_tree_attention(q.reshape(B * S, Hq, D), self._mask, plan.qo_indptr, self._total, self._max_q,
                                                      k_layer, v_layer, plan.indptr, plan.indices, plan.lpl, plan.total_pages,
                                                      **rows, **new)
        return out.view(B, S, Hq * D)

    def attend(self, layer_idx, q, k_new, v_new, n_heads, n_kv_heads):
        """Write the nodes' k_new / v_new [B, S, Hkv, D] behind their sequences' tokens and attend q [B, S, Hq, D] in one
        launch: [B, S, Hq * D]."""
        return self._attend(q, *self.cache._kv_layer(layer_idx), k_new=k_new, v_new=v_new)

    def attend_rope(self, layer_idx, q, k_new, v_new, cos, sin, n_heads, n_kv_heads):
        """attend() on q and k_new rotated at the nodes' positions, the rotation in the launch that writes the rows."""
        self._check_positions(cos.shape[0])
        S = q.shape[1]
        self._rows(S)  # (refuses a grid that is too narrow)
        k_layer, v_layer = self.cache._kv_layer(layer_idx)
        pos, slots = self._pos_for(S), self._plan.slots_for(S)
        self._hold(S)
        q = self.cache.kernels.rope_append(q, k_new, v_new, pos, slots, cos, sin, k_layer, v_layer)
        return self._attend(q, k_layer, v_layer)


@dataclass
class TreeResult:
    """What accept_tree found: the accepted nodes of each tree (path, int32 [B, nodes] on the device, the root first, -1
    behind them), their numbers (counts, on the host), and the token that follows each (next_tokens, int32 [B] on the device)."""
    path: torch.Tensor
    counts: List[int]
    next_tokens: torch.Tensor


def _check_open(cache, ctx, what: str) -> None:
    if not isinstance(ctx, TreeCacheContext) or ctx.cache is not cache or not ctx._open:
        raise ValueError(f"{what}: needs an open context of this cache's begin_tree")
    # (a forward begun since writes the same slots; a sequence released has given its pages away, whoever has its id)
    for sid, start in zip(ctx.seq_ids, ctx.start_positions):
        if not ctx._live[0] or cache._states[sid].num_tokens != start:
            raise ValueError(f"{what}: sequence {sid!r} has changed since begin_tree")


def _nodes(ctx: TreeCacheContext, t: torch.Tensor, name: str) -> torch.Tensor:
    """A [B, S] grid's entries of the nodes, ragged and one behind the other (a column of a wider tensor is neither)."""
    B = ctx.batch_size
    if t.dim() != 2 or t.shape[0] != B or t.shape[1] < ctx._max_q:
        raise ValueError(f"accept_tree: {name} must be [{B}, S], S at least {ctx._max_q}")
    rows = ctx._rows(t.shape[1])
    return t.reshape(-1)[rows["q_rows"][:ctx._total].long()] if rows else t.reshape(-1).contiguous()


def accept_tree(cache, ctx: TreeCacheContext, tokens: torch.Tensor, target_probs: torch.Tensor, u_accept: torch.Tensor,
                u_next: torch.Tensor, draft_probs: Optional[torch.Tensor] = None) -> TreeResult:
    """See KVCacheManager.accept_tree."""
    _check_open(cache, ctx, "accept_tree")
    B = ctx.batch_size
    if target_probs.dim() != 3 or target_probs.shape[0] != B or target_probs.shape[1] < ctx._max_q:
        raise ValueError(f"accept_tree: target_probs must be [{B}, S, vocabulary], S at least {ctx._max_q}")
    if draft_probs is not None and draft_probs.shape != target_probs.shape:
        raise ValueError("accept_tree: draft_probs must be shaped like target_probs")
    S, V = target_probs.shape[1:]
    path, count, token = cache.kernels.verify_tree(
        _nodes(ctx, tokens, "tokens").to(torch.int32), ctx._parents, ctx._plan.qo_indptr, ctx._total, ctx._max_q,
        target_probs.reshape(B * S, V), _nodes(ctx, u_accept, "u_accept"), u_next.reshape(-1).contiguous(),
        draft_probs=None if draft_probs is None else draft_probs.reshape(B * S, V), q_rows=ctx._rows(S).get("q_rows"),
        workspace=cache.workspace)
    _move(cache, ctx, path, count)
    counts = count.tolist()  # (waits for the launches)
    _advance(cache, ctx, counts)
    return TreeResult(path, counts, token)


def end_tree(cache, ctx: TreeCacheContext, path: torch.Tensor, count: torch.Tensor) -> List[int]:
    """See KVCacheManager.end_tree."""
    _check_open(cache, ctx, "end_tree")
    if path.dim() != 2 or path.shape[0] != ctx.batch_size or count.shape != path.shape[:1]:
        raise ValueError(f"end_tree: path must be [{ctx.batch_size}, nodes] and count [{ctx.batch_size}]")
    counts = count.tolist()
    for c, nodes, n in zip(counts, path.tolist(), ctx.new_token_counts):
        if not 0 <= c <= min(n, len(nodes)) or any(b <= a for a, b in zip([-1] + nodes[:c], nodes[:c] + [n])):
            raise ValueError(f"end_tree: nodes {nodes[:max(c, 0)]} of {n}: a path is rising nodes of its tree")
    _move(cache, ctx, path, count)
    _advance(cache, ctx, counts)
    return counts


def _move(cache, ctx: TreeCacheContext, path: torch.Tensor, count: torch.Tensor) -> None:
    if ctx._max_q > 1:  # (a root is in its place)
        plan, pools = ctx._plan, cache._kv_pools
        cache.kernels.move_accepted(pools.k, pools.v, path, count, plan.qo_indptr, plan.indptr, plan.indices, plan.lpl)


def _advance(cache, ctx: TreeCacheContext, counts: List[int]) -> None:
    for sid, c, n in zip(ctx.seq_ids, counts, ctx.new_token_counts):
        cache._end_tree(cache._states[sid], c, n)
        del cache._open_trees[sid]
    ctx._open = False
