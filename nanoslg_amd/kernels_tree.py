"""Tensor-level wrappers of the kernels for trees of drafted tokens (speculative decoding).

A tree has n nodes, each one token: node 0, its root, is the sequence's last sampled token, the others are
drafted. parents[j] < j is node j's parent (-1: a root); children of a node are in the order of their
indices. A batch's trees are ragged: the nodes of sequence b are rows qo_indptr[b] .. qo_indptr[b + 1] - 1 of
total_q, at most max_q (<= 1024) a tree. Rows of a model's tensors are those rows or, with q_rows (int32
[total_q]), rows of a padded grid of B * grid_width, a tree's contiguous in its block. While a tree is verified its nodes
are the last tokens that the block table covers, in the order of their indices.

As in ``kernels``, everything is checked on the host, runs on the current stream of the tensors' device, and nothing is
computed on the CPU.
"""
from __future__ import annotations

import math
from typing import Dict, Optional, Tuple

import torch

from . import _lib
from .kernels import _DTYPE_CODE, Workspace, _i32, _layer_geom, _pool_geom, _require_gpu, _stream
from .kernels_q8 import _call, _new_rows, _one_device, _table

MAX_TREE_NODES = 1024


def _ints(names: str, *ts: torch.Tensor) -> None:
    """Contiguous int32 tensors."""
    for t in ts:
        if t.dtype is not torch.int32 or not t.is_contiguous():
            break
    else:
        return
    for t, name in zip(ts, names.split()):
        _i32(t, name)  # raises its error


def _trees(what: str, qo_indptr: torch.Tensor, total_q: int, max_q: int, q_rows: Optional[torch.Tensor],
           grid_width: int = 1) -> Tuple[int, int, int]:
    """(batch, total_q, max_q) of a batch of trees."""
    B, total_q, max_q = qo_indptr.numel() - 1, int(total_q), int(max_q)
    if B < 0 or total_q < 0 or max_q < 0 or max_q * B < total_q:
        raise ValueError(f"{what}: {total_q} nodes in {B} trees of at most {max_q}")
    if max_q > MAX_TREE_NODES:
        raise ValueError(f"{what}: trees of up to {MAX_TREE_NODES} nodes (max_q = {max_q})")
    if q_rows is not None:
        _ints("q_rows", q_rows)
        if q_rows.numel() < total_q or grid_width < 1:
            raise ValueError(f"{what}: a grid of B x grid_width rows and one q_rows entry per node")
    return B, total_q, max_q


def _rows_ptr(q_rows: Optional[torch.Tensor], total_q: int, qo_indptr: torch.Tensor) -> Optional[int]:
    """q_rows as the entry points take it: null is no grid, so a grid without nodes, whose q_rows may be empty and is not read,
    goes by another address."""
    return None if q_rows is None else q_rows.data_ptr() if total_q else qo_indptr.data_ptr()


def tree_plan(parents: torch.Tensor, qo_indptr: torch.Tensor, start: torch.Tensor, total_q: int, max_q: int,
              q_rows: Optional[torch.Tensor] = None, grid_width: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Ancestor masks and positions of a batch of trees (nslg_tree_plan).

    parents int32 [total_q], start int32 [B] (tokens before each tree). Returns the masks, int32 [total_q,
    ceil(max_q / 32)] (bit j % 32 of word j / 32: the node sees node j of its tree), and the positions, start + depth,
    int32 [total_q] or, with q_rows, [B * grid_width] with 0 on rows without a node."""
    dev = _one_device(parents, qo_indptr, start) if q_rows is None else _one_device(parents, qo_indptr, start, q_rows)
    B, total_q, max_q = _trees("tree_plan", qo_indptr, total_q, max_q, q_rows, grid_width)
    _ints("qo_indptr parents start", qo_indptr, parents, start)
    if parents.numel() < total_q or start.numel() < B:
        raise ValueError("tree_plan: one parent per node and one start per tree")
    W = (max_q + 31) // 32
    n_pos = total_q if q_rows is None else B * int(grid_width)
    buf = torch.empty(total_q * W + n_pos, dtype=torch.int32, device=parents.device)
    at = buf.data_ptr()
    rc = _call(dev, _lib.fast_tree().tree_plan, parents.data_ptr(), qo_indptr.data_ptr(), start.data_ptr(),
               _rows_ptr(q_rows, total_q, qo_indptr), int(grid_width), total_q, max_q, B, at, W,
               at + 4 * total_q * W, _stream(parents))
    if rc:
        _lib.check(rc, "nslg_tree_plan")
    return buf.as_strided((total_q, W), (W, 1)), buf.as_strided((n_pos,), (1,), total_q * W)


_WS_BYTES: Dict[Tuple[int, ...], int] = {}  # nslg_paged_tree_workspace_size by call shape


def _workspace_bytes(*key: int) -> int:
    need = _WS_BYTES.get(key)
    if need is None:  # a pure function of the call shape
        need = int(_lib.load().nslg_paged_tree_workspace_size(*key))
        if len(_WS_BYTES) > 4096:
            _WS_BYTES.clear()
        _WS_BYTES[key] = need
    return need


def paged_tree_attention(q: torch.Tensor, mask: torch.Tensor, qo_indptr: torch.Tensor, total_q: int, max_q: int,
                         k_layer: torch.Tensor, v_layer: torch.Tensor, kv_indptr: torch.Tensor, kv_indices: torch.Tensor,
                         kv_last_page_len: torch.Tensor, total_pages: int, k_new: Optional[torch.Tensor] = None,
                         v_new: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None,
                         out: Optional[torch.Tensor] = None, workspace: Optional[Workspace] = None,
                         q_rows: Optional[torch.Tensor] = None, grid_width: int = 0) -> torch.Tensor:
    """Attention of a batch of trees over a cache layer (nslg_paged_tree_attention): q [rows, Hq, D], returned in its
    shape (grid rows without a node are zero).

    Each node sees the tokens before its tree and the nodes whose bits its row of `mask` has (tree_plan's masks, or
    int32 [total_q, words] masks of any other form); a row that sees nothing is zero, and what an unseen token holds does not
    matter. With k_new and v_new ([..., Hkv, D], q's rows) the nodes' K/V rows are written to their slots in the same
    launch; without, they are in the cache. `workspace`: scratch kept from call to call, one call at a time; without it
    a call's scratch is allocated on the current stream."""
    dev = _one_device(q, mask, qo_indptr, k_layer, v_layer, kv_indptr, kv_indices, kv_last_page_len)
    B, total_q, max_q = _trees("paged_tree_attention", qo_indptr, total_q, max_q, q_rows, grid_width)
    _ints("qo_indptr", qo_indptr)
    P, ps, Hkv, D = _layer_geom(k_layer, v_layer)
    dtype = q.dtype
    code = _DTYPE_CODE.get(dtype)
    if code is None or dtype is not k_layer.dtype:
        raise TypeError(f"paged_tree_attention: q ({dtype}) must be of the cache's type, float16, bfloat16 or float32")
    if q.dim() != 3 or q.shape[2] != D or q.stride(2) != 1 or q.stride(1) != D:
        raise ValueError(f"paged_tree_attention: q must be [rows, Hq, {D}] with a contiguous [Hq, D] block")
    if _table("paged_tree_attention", kv_indptr, kv_indices, kv_last_page_len) != B:
        raise ValueError("paged_tree_attention: qo_indptr and kv_indptr must have B+1 entries")
    rows, Hq, _ = q.shape
    if q_rows is not None:
        _require_gpu(q, q_rows)
        if rows != B * int(grid_width):
            raise ValueError(f"paged_tree_attention: {rows} rows of q for a grid of {B} x {grid_width}")
    elif rows < total_q:
        raise ValueError(f"paged_tree_attention: {rows} rows of q for {total_q} nodes")
    if mask.dtype != torch.int32 or not mask.is_contiguous() or mask.dim() != 2 or mask.shape[0] < total_q:
        raise ValueError("paged_tree_attention: mask must be contiguous int32 [total_q, words]")
    esize = k_layer.element_size()
    q_stride = q.stride(0) if rows > 1 else Hq * D
    if q.data_ptr() % 16 or q_stride * esize % 16 or q_stride < Hq * D:
        q, q_stride = q.contiguous() if q.data_ptr() % 16 == 0 else q.clone(memory_format=torch.contiguous_format), Hq * D
    new = (None, 0, None, 0)
    if k_new is not None or v_new is not None:
        if k_new is None or v_new is None:
            raise ValueError("paged_tree_attention: k_new and v_new go together")
        _one_device(q, k_new, v_new)
        if k_new.dtype is not dtype or v_new.dtype is not dtype:
            raise TypeError("paged_tree_attention: q, k_new and v_new must share one dtype")
        k_new, ks = _new_rows("paged_tree_attention", k_new, "k_new", rows, Hkv, D)
        v_new, vs = _new_rows("paged_tree_attention", v_new, "v_new", rows, Hkv, D)
        new = (k_new.data_ptr(), ks, v_new.data_ptr(), vs)
    if out is None:
        out = torch.empty((rows, Hq, D), dtype=dtype, device=q.device)
        out_stride = Hq * D
    else:
        _one_device(q, out)
        if out.shape != (rows, Hq, D) or out.dtype is not dtype or out.stride(2) != 1 or out.stride(1) != D:
            raise ValueError("paged_tree_attention: bad out tensor")
        out_stride = out.stride(0) if rows > 1 else Hq * D
    need = _workspace_bytes(B, Hq, Hkv, D, int(total_pages), ps, max_q, code)
    ws = None
    if need:
        ws = workspace.get_prefill(need) if workspace is not None else torch.empty(need, dtype=torch.uint8, device=q.device)
    rc = _call(dev, _lib.fast_tree().paged_tree_attention, q.data_ptr(), q_stride, mask.data_ptr(), mask.shape[1],
               qo_indptr.data_ptr(), _rows_ptr(q_rows, total_q, qo_indptr), int(grid_width), total_q, max_q, *new,
               k_layer.data_ptr(), v_layer.data_ptr(), P, ps, kv_indptr.data_ptr(), kv_indices.data_ptr(),
               kv_last_page_len.data_ptr(), int(total_pages), B, Hq, Hkv, D,
               1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale), code, out.data_ptr(), out_stride,
               None if ws is None else ws.data_ptr(), need, _stream(q))
    if rc:
        _lib.check(rc, "nslg_paged_tree_attention")
    return out


_VERIFY_BYTES: Dict[Tuple[int, int], int] = {}  # nslg_verify_tree_workspace_size by batch and vocabulary


def verify_tree(tokens: torch.Tensor, parents: torch.Tensor, qo_indptr: torch.Tensor, total_q: int, max_q: int,
                target_probs: torch.Tensor, u_accept: torch.Tensor, u_next: torch.Tensor,
                draft_probs: Optional[torch.Tensor] = None, q_rows: Optional[torch.Tensor] = None,
                workspace: Optional[Workspace] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Verify drafted tokens against the target's probabilities, from given uniform numbers in [0, 1) (nslg_verify_tree).

    tokens, parents int32 [total_q]; target_probs [rows, vocab] (float16, bfloat16 or float32), the row of node t being t,
    or q_rows[t]; u_accept float32 [total_q], u_next float32 [B]. draft_probs, like target_probs: a node's row is the
    distribution that its children were drawn from, independently; without it the drafted tokens are taken as given.
    Returns (path, count, next): int32 [B, max_q] accepted nodes, the root first, -1 behind them; their number
    [B]; the token that follows [B]. Accepted and next tokens have the target's distribution where rows sum to 1 (a row
    filtered by top-k or top-p is normalised again first; nothing here does it). Rows with the
    probability of one token 1 make this greedy verification. `workspace`: with it, kept from call to call and used by one call
    at a time, several workgroups take a sequence."""
    dev = _one_device(tokens, parents, qo_indptr, target_probs, u_accept, u_next)
    B, total_q, max_q = _trees("verify_tree", qo_indptr, total_q, max_q, q_rows)
    _ints("qo_indptr tokens parents", qo_indptr, tokens, parents)
    if tokens.numel() < total_q or parents.numel() < total_q or u_accept.numel() < total_q or u_next.numel() < B:
        raise ValueError("verify_tree: a token, a parent and a number u_accept per node, and u_next per tree")
    if not (u_accept.dtype is u_next.dtype is torch.float32 and u_accept.is_contiguous() and u_next.is_contiguous()):
        raise ValueError("verify_tree: u_accept and u_next must be contiguous float32")
    code = _DTYPE_CODE.get(target_probs.dtype)
    if code is None:
        raise TypeError(f"verify_tree: probabilities of float16, bfloat16 or float32 (got {target_probs.dtype})")
    if q_rows is not None:
        _require_gpu(tokens, q_rows)
    if target_probs.dim() != 2 or target_probs.stride(1) != 1 or (q_rows is None and target_probs.shape[0] < total_q):
        raise ValueError("verify_tree: target_probs must be [rows, vocab], a row per node, with contiguous rows")
    rows, vocab = target_probs.shape
    ts = target_probs.stride(0) if rows > 1 else vocab
    ds = 0
    if draft_probs is not None:
        _require_gpu(tokens, draft_probs)
        if draft_probs.dtype is not target_probs.dtype:
            raise TypeError("verify_tree: draft_probs must be of target_probs' type")
        if draft_probs.shape != target_probs.shape or draft_probs.stride(1) != 1:
            raise ValueError("verify_tree: draft_probs must be shaped like target_probs")
        ds = draft_probs.stride(0) if rows > 1 else vocab
    ws, need = None, 0
    if workspace is not None:
        key = (B, vocab)
        need = _VERIFY_BYTES.get(key)
        if need is None:  # a pure function of the call shape
            need = _VERIFY_BYTES[key] = int(_lib.load().nslg_verify_tree_workspace_size(B, vocab))
        if need:
            ws = workspace.get_verify(need)
    buf = torch.empty(B * (max_q + 2), dtype=torch.int32, device=tokens.device)
    at = buf.data_ptr()
    rc = _call(dev, _lib.fast_tree().verify_tree, tokens.data_ptr(), parents.data_ptr(), qo_indptr.data_ptr(),
               None if q_rows is None else q_rows.data_ptr(), total_q, max_q, B, target_probs.data_ptr(), ts,
               None if draft_probs is None else draft_probs.data_ptr(), ds, rows, vocab, code, u_accept.data_ptr(),
               u_next.data_ptr(), at, at + 4 * B * max_q, at + 4 * B * (max_q + 1), None if ws is None else ws.data_ptr(), need,
               _stream(tokens))
    if rc:
        _lib.check(rc, "nslg_verify_tree")
    n = B * max_q
    return buf.as_strided((B, max_q), (max_q, 1)), buf.as_strided((B,), (1,), n), buf.as_strided((B,), (1,), n + B)


def move_accepted(k_pool: torch.Tensor, v_pool: torch.Tensor, path: torch.Tensor, count: torch.Tensor, qo_indptr: torch.Tensor,
                  kv_indptr: torch.Tensor, kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor) -> None:
    """Move the accepted nodes' K/V rows to the slots behind their sequence's tokens (nslg_move_accepted), in every layer of
    the [L, P, page_size, Hkv, D] pools: the row of node path[b, i] to position start_b + i for i < count[b]. path
    int32 [B, width] and count int32 [B] as verify_tree gives them; qo_indptr and the block table are those that the
    trees' attention ran with. A sequence whose path is not rising nodes of its tree is left as it is."""
    dev = _one_device(k_pool, v_pool, path, count, qo_indptr, kv_indptr, kv_indices, kv_last_page_len)
    L, P, ps, Hkv, D = _pool_geom(k_pool, v_pool)
    code = _DTYPE_CODE.get(k_pool.dtype)
    if code is None:
        raise TypeError(f"move_accepted: float16, bfloat16 or float32 pools (got {k_pool.dtype})")
    B = _table("move_accepted", kv_indptr, kv_indices, kv_last_page_len)
    _ints("path count qo_indptr", path, count, qo_indptr)
    if path.dim() != 2 or path.shape[0] != B or count.numel() != B or qo_indptr.numel() != B + 1:
        raise ValueError("move_accepted: path must be [B, width], count [B] and qo_indptr [B+1]")
    rc = _call(dev, _lib.fast_tree().move_accepted, k_pool.data_ptr(), v_pool.data_ptr(), L, P, ps, Hkv, D, code,
               path.data_ptr(), path.shape[1], count.data_ptr(), qo_indptr.data_ptr(), kv_indptr.data_ptr(),
               kv_indices.data_ptr(), kv_last_page_len.data_ptr(), B, _stream(k_pool))
    if rc:
        _lib.check(rc, "nslg_move_accepted")
