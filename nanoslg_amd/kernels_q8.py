"""Tensor-level wrappers of the 8-bit KV cache kernels (nslg_q8_* of the C ABI).

One layer of an 8-bit cache is four tensors: codes k_layer and v_layer [P, page_size, Hkv, D]
(torch.float8_e4m3fn or torch.int8) and scales k_scale and v_scale [P, nb, Hkv] (float32, nb =
ceil(page_size / 16)): one scale for each block of 16 slots of a page and KV head. A stored value is
code * scale; scales are powers of two or 0, as append_kv_q8 writes them. Rows, queries and
outputs are float16 or bfloat16. As in ``kernels``, everything is checked on the host, runs on the
current stream of the tensors' device, and nothing is computed on the CPU.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib
from .kernels import (_DTYPE_CODE, _LAYOUT_TAGS, DecodeGroups, DecodeLaunch, Workspace, _i32, _prefill_workspace,
                      _require_gpu, _rope_tables, _rows, _stream, rope_append)

BLOCK_TOKENS = 16  # slots of a page that share a scale
CODE_DTYPES = {torch.float8_e4m3fn: _lib.NSLG_E4M3, torch.int8: _lib.NSLG_INT8}
HEAD_DIMS_Q8 = (64, 128, 256)


_CURRENT_DEVICE = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _one_device(*ts: torch.Tensor) -> int:
    """The index of the one GPU that all tensors are on."""
    d = ts[0].get_device()
    if d >= 0:
        for t in ts:
            if t.get_device() != d:
                break
        else:
            return d
    _require_gpu(*ts)  # raises its error
    return d


def _call(device: int, fn, *args) -> int:
    """An entry point with the tensors' device as the current one (the library launches on the current device)."""
    if _CURRENT_DEVICE() == device:
        return fn(*args)
    with torch.cuda.device(device):
        return fn(*args)


def _layer(what: str, k_layer, v_layer, k_scale, v_scale):
    """(P, page_size, Hkv, D, code) of a cache layer."""
    shape, dtype = k_layer.shape, k_layer.dtype
    if len(shape) != 4 or shape != v_layer.shape or dtype != v_layer.dtype:
        raise ValueError(f"{what}: codes must be [P, page_size, Hkv, D] for both K and V")
    code = CODE_DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"{what}: codes must be float8_e4m3fn or int8 (got {dtype})")
    P, ps, Hkv, D = shape
    scales = (P, -(-ps // BLOCK_TOKENS), Hkv)
    if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
        raise TypeError(f"{what}: scales must be float32")
    if k_scale.shape != scales or v_scale.shape != scales:
        raise ValueError(f"{what}: scales must be {list(scales)}, one for each block of {BLOCK_TOKENS} slots and head")
    if not (k_layer.is_contiguous() and v_layer.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
        raise ValueError(f"{what}: the cache layer must be contiguous")
    return P, ps, Hkv, D, code


def _table(what: str, kv_indptr, kv_indices, kv_last_page_len) -> int:
    """The batch size of a block table."""
    i32 = torch.int32
    if not (kv_indptr.dtype is i32 and kv_indices.dtype is i32 and kv_last_page_len.dtype is i32 and kv_indptr.is_contiguous()
            and kv_indices.is_contiguous() and kv_last_page_len.is_contiguous()):
        for t, n in ((kv_indptr, "kv_indptr"), (kv_indices, "kv_indices"), (kv_last_page_len, "kv_last_page_len")):
            _i32(t, n)
    B = kv_indptr.numel() - 1
    if B < 0 or kv_last_page_len.numel() < B:
        raise ValueError(f"{what}: kv_indptr must have B+1 entries and kv_last_page_len B")
    return B


_ROW_TYPES = {torch.float16: _lib.NSLG_F16, torch.bfloat16: _lib.NSLG_BF16}


def _row_type(what: str, q, k_new=None, v_new=None) -> int:
    dtype = q.dtype
    code = _ROW_TYPES.get(dtype)
    if code is None:
        raise TypeError(f"{what}: float16 or bfloat16 rows (got {dtype})")
    if (k_new is not None and k_new.dtype is not dtype) or (v_new is not None and v_new.dtype is not dtype):
        raise TypeError(f"{what}: q, k_new and v_new must share one dtype")
    return code


def _new_rows(what: str, t: torch.Tensor, name: str, n: int, Hkv: int, D: int) -> Tuple[torch.Tensor, int]:
    """The rows of k_new / v_new at one 16-byte stride (others are copied) and the stride."""
    shape = t.shape
    if len(shape) < 2 or shape[-1] != D or shape[-2] != Hkv:
        raise ValueError(f"{what}: {name} must hold rows of [{Hkv}, {D}]")
    if t.is_contiguous():  # a model's own rows
        stride = Hkv * D
        rows = t.numel() // stride
    else:
        rows, stride, _ = _rows(t, name)
    if rows != n:
        raise ValueError(f"{what}: {rows} rows of {name} for {n}")
    if t.data_ptr() % 16 or stride % 8 or stride < Hkv * D:
        t, stride = t.reshape(rows, Hkv, D).clone(memory_format=torch.contiguous_format), Hkv * D
    return t, stride


def append_kv_q8(k_new: torch.Tensor, v_new: torch.Tensor, qo_indptr: torch.Tensor, total_q: int, k_layer: torch.Tensor,
                 v_layer: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, kv_indptr: torch.Tensor,
                 kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor, q_rows: Optional[torch.Tensor] = None,
                 grid_width: int = 0) -> None:
    """Write a forward's new K/V rows into an 8-bit cache layer (nslg_q8_append_kv).

    The block table covers the new tokens: sequence b's are its last qo_indptr[b+1] -
    qo_indptr[b] positions, rows qo_indptr[b] .. of k_new / v_new ([..., Hkv, D], total_q rows), or,
    with q_rows (int32 [total_q]), rows q_rows[qo_indptr[b]] .. of a padded grid of B * grid_width.
    Each block of 16 slots and head has one power-of-two scale: what the block's new rows need, or,
    if the block holds earlier tokens, the larger of that and its own, to which their codes are then
    rounded. Codes are rounded to nearest even. A token's value that is not finite, in K or in V, makes
    its K NaN (float8_e4m3fn: some of the row's codes; int8, which has no such code: the scale of the
    block's K until the block is written from its start), so that the queries that see the token (int8:
    a token of the block) answer NaN and no others; V holds 0 in its place."""
    dev = _one_device(k_layer, v_layer, k_scale, v_scale, k_new, v_new, qo_indptr, kv_indptr, kv_indices, kv_last_page_len)
    P, ps, Hkv, D, code = _layer("append_kv_q8", k_layer, v_layer, k_scale, v_scale)
    B = _table("append_kv_q8", kv_indptr, kv_indices, kv_last_page_len)
    _i32(qo_indptr, "qo_indptr")
    dt = _row_type("append_kv_q8", k_new, v_new)
    if qo_indptr.numel() != B + 1:
        raise ValueError("append_kv_q8: qo_indptr must have B+1 entries")
    n = total_q = int(total_q)
    if q_rows is not None:
        _require_gpu(k_new, q_rows)
        _i32(q_rows, "q_rows")
        if q_rows.numel() < total_q or grid_width < 1:
            raise ValueError("append_kv_q8: a grid of B x grid_width rows and one q_rows entry per token")
        n = B * int(grid_width)
    k_new, ks = _new_rows("append_kv_q8", k_new, "k_new", n, Hkv, D)
    v_new, vs = _new_rows("append_kv_q8", v_new, "v_new", n, Hkv, D)
    rc = _call(dev, _lib.fast_q8().append_kv, k_new.data_ptr(), ks, v_new.data_ptr(), vs, qo_indptr.data_ptr(),
               None if q_rows is None else q_rows.data_ptr(), int(grid_width), total_q, k_layer.data_ptr(),
               v_layer.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), P, ps, kv_indptr.data_ptr(),
               kv_indices.data_ptr(), kv_last_page_len.data_ptr(), B, Hkv, D, dt, code, _stream(k_layer))
    _lib.check(rc, "nslg_q8_append_kv")


def gather_kv_q8(k_layer: torch.Tensor, v_layer: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                 kv_indptr: torch.Tensor, kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor, max_len: int,
                 dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cached tokens' values (code * scale, rounded once) as contiguous [B, max_len, Hkv, D] K
    and V of `dtype` (float16, bfloat16 or float32), zeros past each length."""
    dev = _one_device(k_layer, v_layer, k_scale, v_scale, kv_indptr, kv_indices, kv_last_page_len)
    P, ps, Hkv, D, code = _layer("gather_kv_q8", k_layer, v_layer, k_scale, v_scale)
    B = _table("gather_kv_q8", kv_indptr, kv_indices, kv_last_page_len)
    if dtype not in _DTYPE_CODE:
        raise TypeError(f"gather_kv_q8: unsupported dtype {dtype}")
    k_out, v_out = torch.empty((2, B, int(max_len), Hkv, D), dtype=dtype, device=k_layer.device).unbind(0)
    rc = _call(dev, _lib.fast_q8().gather_kv, k_layer.data_ptr(), v_layer.data_ptr(), k_scale.data_ptr(),
               v_scale.data_ptr(), P, ps, kv_indptr.data_ptr(), kv_indices.data_ptr(), kv_last_page_len.data_ptr(), B,
               int(max_len), Hkv, D, code, _DTYPE_CODE[dtype], k_out.data_ptr(), v_out.data_ptr(), _stream(k_layer))
    _lib.check(rc, "nslg_q8_gather_kv")
    return k_out, v_out


def paged_decode_q8(q: torch.Tensor, k_layer: torch.Tensor, v_layer: torch.Tensor, k_scale: torch.Tensor,
                    v_scale: torch.Tensor, kv_indptr: torch.Tensor, kv_indices: torch.Tensor,
                    kv_last_page_len: torch.Tensor, total_pages: int, sm_scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, workspace: Optional[Workspace] = None,
                    groups: Optional[DecodeGroups] = None, layout: int = 0) -> torch.Tensor:
    """Decode attention over an 8-bit cache layer: ``kernels.paged_decode`` with its arguments
    (q [B, Hq, D], rows may be strided; returns [B, Hq, D])."""
    return _decode8("paged_decode_q8", q, None, None, None, k_layer, v_layer, k_scale, v_scale, kv_indptr, kv_indices,
                    kv_last_page_len, total_pages, sm_scale, out, workspace, groups, layout)


def paged_decode_append_q8(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, k_layer: torch.Tensor,
                           v_layer: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, kv_indptr: torch.Tensor,
                           kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor, total_pages: int,
                           sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                           workspace: Optional[Workspace] = None, groups: Optional[DecodeGroups] = None,
                           layout: int = 0) -> torch.Tensor:
    """One decode step of a layer: row b of k_new / v_new ([B, ..., Hkv, D], rows may be strided)
    written as sequence b's last token, then decode attention. Same result as append_kv_q8 of
    one row a sequence followed by paged_decode_q8; in the decode launch itself where 16
    divides the page size (a block then lies in one wave's work), with a launch of
    its own ahead otherwise."""
    return _decode8("paged_decode_append_q8", q, k_new, v_new, None, k_layer, v_layer, k_scale, v_scale, kv_indptr,
                    kv_indices, kv_last_page_len, total_pages, sm_scale, out, workspace, groups, layout)


def paged_decode_rope_append_q8(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, positions: torch.Tensor,
                                cos: torch.Tensor, sin: torch.Tensor, k_layer: torch.Tensor, v_layer: torch.Tensor,
                                k_scale: torch.Tensor, v_scale: torch.Tensor, kv_indptr: torch.Tensor,
                                kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor, total_pages: int,
                                sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                                workspace: Optional[Workspace] = None, groups: Optional[DecodeGroups] = None,
                                layout: int = 0) -> torch.Tensor:
    """paged_decode_append_q8 of q and k_new rotated at each sequence's `positions` entry (int32 [B]) with
    the model's [max_positions, >= D] cos / sin tables, as in ``kernels.paged_decode_rope_append``."""
    _require_gpu(q, positions, cos, sin)
    _i32(positions, "positions")
    if positions.numel() != q.shape[0]:
        raise ValueError("paged_decode_rope_append_q8: one position per sequence")
    return _decode8("paged_decode_rope_append_q8", q, k_new, v_new, (positions, *_rope_tables(cos, sin, q.shape[-1])),
                    k_layer, v_layer, k_scale, v_scale, kv_indptr, kv_indices, kv_last_page_len, total_pages, sm_scale, out,
                    workspace, groups, layout)


def rotate_rows(q, k_new, v_new, positions, cos, sin):
    """q and k_new ([..., H, D] rows, `positions` int32 one a row) rotated, as new contiguous rows
    (``kernels.rope_append`` into rows of its own)."""
    Hkv, D = k_new.shape[-2], k_new.shape[-1]
    n = positions.numel()
    k_rot = torch.empty((n, 1, Hkv, D), dtype=k_new.dtype, device=k_new.device)
    slots = torch.arange(n, dtype=torch.int32, device=k_new.device)
    q_rot = _call(q.get_device(), rope_append, q, k_new, v_new, positions, slots, cos, sin, k_rot, torch.empty_like(k_rot))
    return q_rot, k_rot.view(n, Hkv, D)


def _decode8(what, q, k_new, v_new, rope, k_layer, v_layer, k_scale, v_scale, kv_indptr, kv_indices, kv_last_page_len,
             total_pages, sm_scale, out, workspace, groups, layout):
    dev = _one_device(q, k_layer, v_layer, k_scale, v_scale, kv_indptr, kv_indices, kv_last_page_len)
    P, ps, Hkv, D, code = _layer(what, k_layer, v_layer, k_scale, v_scale)
    B = _table(what, kv_indptr, kv_indices, kv_last_page_len)
    qs, qst = q.shape, q.stride()
    if len(qs) != 3 or qs[0] != B or qs[2] != D or qst[2] != 1 or qst[1] != D:
        raise ValueError(f"{what}: q must be [{B}, Hq, {D}] with a contiguous [Hq, D] block")
    Hq = qs[1]
    if Hq % Hkv:
        raise ValueError(f"{what}: Hq={Hq} is not a multiple of Hkv={Hkv}")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif (out.shape != (B, Hq, D) or out.stride(2) != 1 or out.stride(1) != D or out.dtype != q.dtype
          or out.get_device() != q.get_device()):
        raise ValueError(f"{what}: bad out tensor")
    rows = (None, 0, None, 0)
    tables = (None, None, None, 0, 0)
    if k_new is None:
        dt = _row_type(what, q)
    else:
        _one_device(q, k_new, v_new)
        dt = _row_type(what, q, k_new, v_new)
        if ps % BLOCK_TOKENS:
            # a block may lie in two waves' work: the rows go in ahead
            if rope is not None:
                q, k_new = rotate_rows(q, k_new, v_new, *rope)
                rope = None
            append_kv_q8(k_new, v_new, torch.arange(B + 1, dtype=torch.int32, device=q.device), B, k_layer, v_layer,
                         k_scale, v_scale, kv_indptr, kv_indices, kv_last_page_len)
        else:
            k_new, ks = _new_rows(what, k_new, "k_new", B, Hkv, D)
            v_new, vs = _new_rows(what, v_new, "v_new", B, Hkv, D)
            rows = (k_new.data_ptr(), ks, v_new.data_ptr(), vs)
            if rope is not None:
                pos, cos, sin = rope
                if cos.data_ptr() % 16 or sin.data_ptr() % 16 or cos.stride(0) % 4:
                    cos, sin = (t[:, :D].clone(memory_format=torch.contiguous_format) for t in (cos, sin))
                tables = (pos.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.stride(0), cos.shape[0])
    grp = (None, 0, None, None)
    if groups is not None:
        _require_gpu(q, groups.seq_group_slot)
        _i32(groups.seq_group_slot, "seq_group_slot")
        if groups.seq_group_slot.numel() != B:
            raise ValueError(f"{what}: one group slot per sequence")
        grp = (groups.seq_group_slot.data_ptr(), groups.num_groups, groups.prefix_pages_np.ctypes.data,
               groups.members_np.ctypes.data)
    scale = (1.0 / math.sqrt(D)) if sm_scale is None else float(sm_scale)
    total_pages = int(total_pages)
    args = (q.data_ptr(), q.stride(0), *rows, *tables, k_layer.data_ptr(), v_layer.data_ptr(), k_scale.data_ptr(),
            v_scale.data_ptr(), P, ps, kv_indptr.data_ptr(), kv_indices.data_ptr(), kv_last_page_len.data_ptr(),
            total_pages, B, Hq, Hkv, D, scale, dt, code, *grp, out.data_ptr(), out.stride(0))
    stream = _stream(q)
    fn = (_lib._fast_q8 or _lib.fast_q8()).paged_decode
    rc = _lib.NSLG_EWORKSPACE
    if workspace is not None:  # a kept workspace mostly suffices: the call itself says if it does not
        ws = workspace.buf
        rc = _call(dev, fn, *args, ws.data_ptr(), ws.numel(), layout, stream)
    if rc == _lib.NSLG_EWORKSPACE:
        need = int(_call(dev, _lib.load().nslg_q8_paged_decode_workspace_size, B, Hq, Hkv, D, total_pages, ps, dt, code,
                         grp[1]))
        ws = (workspace or Workspace(q.device)).get(need)
        rc = _call(dev, fn, *args, ws.data_ptr(), ws.numel(), layout, stream)
    _lib.check(rc, "nslg_q8_paged_decode")
    return out


def paged_prefill_q8(q: torch.Tensor, qo_indptr: torch.Tensor, total_q: int, max_q: int, k_layer: torch.Tensor,
                     v_layer: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, kv_indptr: torch.Tensor,
                     kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor, sm_scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None, workspace: Optional[Workspace] = None,
                     q_rows: Optional[torch.Tensor] = None, grid_width: int = 0,
                     max_kv: Optional[int] = None) -> torch.Tensor:
    """Causal (bottom-right) prefill attention over an 8-bit cache layer that holds the new tokens too
    (append_kv_q8 first): ``kernels.paged_prefill`` with its arguments. max_kv: the longest
    sequence's keys, where the caller knows it (it decides whether keys are cut into runs)."""
    dev = _one_device(q, qo_indptr, k_layer, v_layer, k_scale, v_scale, kv_indptr, kv_indices, kv_last_page_len)
    P, ps, Hkv, D, code = _layer("paged_prefill_q8", k_layer, v_layer, k_scale, v_scale)
    B = _table("paged_prefill_q8", kv_indptr, kv_indices, kv_last_page_len)
    _i32(qo_indptr, "qo_indptr")
    dt = _row_type("paged_prefill_q8", q)
    total_q = int(total_q)
    if q.dim() != 3 or q.shape[2] != D or q.stride(2) != 1 or q.stride(1) != D:
        raise ValueError(f"paged_prefill_q8: q must be [T, Hq, {D}] with a contiguous [Hq, D] block")
    T, Hq, _ = q.shape
    if Hq % Hkv:
        raise ValueError(f"paged_prefill_q8: Hq={Hq} is not a multiple of Hkv={Hkv}")
    if qo_indptr.numel() != B + 1 or T < total_q:
        raise ValueError("paged_prefill_q8: qo_indptr must have B+1 entries and q at least total_q rows")
    if q_rows is not None:
        _require_gpu(q, q_rows)
        _i32(q_rows, "q_rows")
        if q_rows.numel() < total_q or grid_width < 1 or T != B * grid_width:
            raise ValueError("paged_prefill_q8: a grid of B x grid_width rows of q and one q_rows entry per token")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif (out.shape != (T, Hq, D) or out.stride(2) != 1 or out.stride(1) != D or out.dtype != q.dtype
          or out.get_device() != q.get_device()):
        raise ValueError("paged_prefill_q8: out must be shaped like q")
    if max_kv is None:  # the average sequence's table stands for the longest one (its length is on the device)
        max_kv = kv_indices.numel() * ps // max(B, 1)
    scale = (1.0 / math.sqrt(D)) if sm_scale is None else float(sm_scale)
    ws, ws_ptr, ws_bytes = _prefill_workspace(q, B, Hq, D, total_q, int(max_q), max_kv, workspace)
    rc = _call(dev, _lib.fast_q8().paged_prefill, q.data_ptr(), q.stride(0), qo_indptr.data_ptr(),
               None if q_rows is None else q_rows.data_ptr(), int(grid_width), total_q, int(max_q), k_layer.data_ptr(),
               v_layer.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), P, ps, kv_indptr.data_ptr(),
               kv_indices.data_ptr(), kv_last_page_len.data_ptr(), B, Hq, Hkv, D, scale, dt, code, out.data_ptr(),
               out.stride(0), ws_ptr, ws_bytes, _stream(q))
    _lib.check(rc, "nslg_q8_paged_prefill")
    return out


class DecodeLaunchQ8(DecodeLaunch):
    """Append + decode for every layer of one decode forward over an 8-bit cache: what
    ``kernels.DecodeLaunch`` does over 16-bit pools, with its interface. The step's rows go in
    in the decode launch (nslg_q8_paged_decode with new rows; on pages that 16 does not divide
    nslg_q8_append_kv goes ahead), with RoPE rotated there too. The forward's first call
    of a row type records its chunk layout for the other layers'."""

    def __init__(self, k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                 slot_mapping: torch.Tensor, kv_indptr: torch.Tensor, kv_indices: torch.Tensor,
                 kv_last_page_len: torch.Tensor, total_pages: int, num_qo_heads: int,
                 workspace: Optional[Workspace] = None, sm_scale: Optional[float] = None,
                 groups: Optional[DecodeGroups] = None):
        _require_gpu(k_pool, v_pool, k_scale, v_scale)
        if k_pool.dim() != 5 or k_scale.dim() != 4:
            raise ValueError("DecodeLaunchQ8: pools must be [L, P, page_size, Hkv, D] and scales [L, P, nb, Hkv]")
        self.L = k_pool.shape[0]
        if not (v_pool.dim() == 5 and v_scale.dim() == 4 and v_pool.shape[0] == k_scale.shape[0] == v_scale.shape[0] == self.L):
            raise ValueError("DecodeLaunchQ8: pools and scales of as many layers")
        self.P, self.ps, self.Hkv, self.D, self.q8 = _layer("DecodeLaunchQ8", k_pool[0], v_pool[0], k_scale[0], v_scale[0])
        if not all(t.is_contiguous() for t in (k_pool, v_pool, k_scale, v_scale)):
            raise ValueError("DecodeLaunchQ8: pools and scales must be contiguous")
        if num_qo_heads % self.Hkv:
            raise ValueError(f"DecodeLaunchQ8: Hq={num_qo_heads} is not a multiple of Hkv={self.Hkv}")
        self.lib = _lib.load()
        self._f_decode8 = _lib.fast_q8().paged_decode
        self.device, self.dev_index, self.dtype = k_pool.device, k_pool.get_device(), k_pool.dtype
        self.Hq = num_qo_heads
        self.kp0, self.vp0, self.ksp0, self.vsp0 = (t.data_ptr() for t in (k_pool, v_pool, k_scale, v_scale))
        self.layer_bytes = k_pool[0].numel()
        self.scale_bytes = 4 * k_scale[0].numel()
        self.pools = (k_pool, v_pool, k_scale, v_scale)
        self.workspace = workspace or Workspace(self.device)
        self.scale = (1.0 / math.sqrt(self.D)) if sm_scale is None else float(sm_scale)
        self.B = kv_indptr.numel() - 1
        self.groups, self._ws_pages = None, -1
        self.rebind(slot_mapping, kv_indptr, kv_indices, kv_last_page_len, total_pages, groups, check=True)

    def rebind(self, slot_mapping: torch.Tensor, kv_indptr: torch.Tensor, kv_indices: torch.Tensor,
               kv_last_page_len: torch.Tensor, total_pages: int, groups: Optional[DecodeGroups] = None,
               check: bool = True) -> "DecodeLaunchQ8":
        """Point the launcher at another forward's plan of the same batch size (slot_mapping is not used: the
        slots come from the block table)."""
        B = self.B
        self._layouts = [0, 0]  # by row type, whose kernels may cut the plan into other chunks
        if check:
            _require_gpu(self.pools[0], kv_indptr, kv_indices, kv_last_page_len)
            if _table("DecodeLaunchQ8", kv_indptr, kv_indices, kv_last_page_len) != B:
                raise ValueError(f"DecodeLaunchQ8: a plan of {B} sequences")
            if groups is not None:
                _require_gpu(self.pools[0], groups.seq_group_slot)
                _i32(groups.seq_group_slot, "seq_group_slot")
                if groups.seq_group_slot.numel() != B:
                    raise ValueError("DecodeLaunchQ8: one group slot per sequence")
        self.table = (kv_indptr, kv_indices, kv_last_page_len)
        self.table_ptrs = (kv_indptr.data_ptr(), kv_indices.data_ptr(), kv_last_page_len.data_ptr())
        self.total_pages = int(total_pages)
        if groups is self.groups and self.total_pages <= self._ws_pages:
            return self
        self.groups = groups
        self.grp = (None, 0, None, None)
        if groups is not None:
            self.grp = (groups.seq_group_slot.data_ptr(), groups.num_groups, groups.prefix_pages_np.ctypes.data,
                        groups.members_np.ctypes.data)
        # sized for some headroom, as in DecodeLaunch; f16 and bf16 calls may both come
        bound = self.total_pages + max(self.total_pages // 4, 1024)
        need = max(int(_call(self.dev_index, self.lib.nslg_q8_paged_decode_workspace_size, B, self.Hq, self.Hkv, self.D, bound,
                             self.ps, dt, self.q8, self.grp[1])) for dt in (_lib.NSLG_F16, _lib.NSLG_BF16))
        if groups is not None and need == 0:
            raise ValueError("DecodeLaunchQ8: unsupported grouped decode shape")
        self.ws = self.workspace.get(need)
        self.ws_args = (self.ws.data_ptr(), self.ws.numel())
        self._ws_pages = bound
        return self

    def __call__(self, layer: int, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                 rope: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]] = None) -> torch.Tensor:
        """As DecodeLaunch: q [B, Hq, D] or [B, 1, Hq, D], k_new / v_new [B, ..., Hkv, D] rows of one token each,
        float16 or bfloat16; rope = (cos, sin, positions int32 [B])."""
        if not 0 <= layer < self.L:
            raise IndexError(f"layer {layer} out of range [0, {self.L})")
        B, Hq, Hkv, D, di = self.B, self.Hq, self.Hkv, self.D, self.dev_index
        if q.get_device() != di or k_new.get_device() != di or v_new.get_device() != di:
            raise ValueError(f"DecodeLaunchQ8: tensors must be on {self.device}")
        dt = _row_type("DecodeLaunchQ8", q, k_new, v_new)
        qs, qst, out_shape = q.shape, q.stride(), (B, Hq, D)
        if len(qs) == 4 and qs[1] == 1:
            out_shape, ok = (B, 1, Hq * D), qs == (B, 1, Hq, D)
        else:
            ok = qs == out_shape
        if not ok or qst[-1] != 1 or qst[-2] != D:
            raise ValueError(f"DecodeLaunchQ8: q must be [{B}, {Hq}, {D}] with a contiguous [Hq, D] block")
        if q.data_ptr() % 16 or qst[0] % 8 or qst[0] < Hq * D:
            q = q.clone(memory_format=torch.contiguous_format)
        tables = (None, None, None, 0, 0)
        if rope is not None:
            cos, sin, pos = rope
            _require_gpu(self.pools[0], cos, sin, pos)
            _i32(pos, "positions")
            if pos.numel() != B:
                raise ValueError("DecodeLaunchQ8: one position per sequence")
            cos, sin = _rope_tables(cos, sin, D)
        rows = (None, 0, None, 0)
        if self.ps % BLOCK_TOKENS:
            if rope is not None:
                q, k_new = rotate_rows(q.reshape(B, Hq, D), k_new, v_new, pos, cos, sin)
            append_kv_q8(k_new, v_new, torch.arange(B + 1, dtype=torch.int32, device=self.device), B,
                         *(t[layer] for t in self.pools), *self.table)
        else:
            k_new, ks = _new_rows("DecodeLaunchQ8", k_new, "k_new", B, Hkv, D)
            v_new, vs = _new_rows("DecodeLaunchQ8", v_new, "v_new", B, Hkv, D)
            rows = (k_new.data_ptr(), ks, v_new.data_ptr(), vs)
            if rope is not None:
                if cos.data_ptr() % 16 or sin.data_ptr() % 16 or cos.stride(0) % 4:
                    cos, sin = (t[:, :D].clone(memory_format=torch.contiguous_format) for t in (cos, sin))
                tables = (pos.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.stride(0), cos.shape[0])
        out = q.new_empty(out_shape)
        lay = self._layouts[dt]  # < 0: read the layout recorded under tag -lay
        if lay == 0:  # the first call of this type on this plan records its chunk layout
            lay = next(_LAYOUT_TAGS)
            self._layouts[dt] = -lay
        off, soff = layer * self.layer_bytes, layer * self.scale_bytes
        rc = _call(di, self._f_decode8, q.data_ptr(), q.stride(0), *rows, *tables, self.kp0 + off, self.vp0 + off,
                   self.ksp0 + soff, self.vsp0 + soff, self.P, self.ps, *self.table_ptrs, self.total_pages, B, Hq, Hkv, D,
                   self.scale, dt, self.q8, *self.grp, out.data_ptr(), Hq * D, *self.ws_args, lay, _stream(q))
        _lib.check(rc, "nslg_q8_paged_decode")
        return out
