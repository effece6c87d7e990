"""Caches whose pool tensors were replaced (moved to other memory): zeroing, copies, writes and reads all go to the tensors
that the cache holds then."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
L, HQ, HKV, D = 2, 8, 2, 64


def make(backend, cache_dtype):
    from nanoslg_amd import kv_cache as KC
    cfg = KC.KVCacheConfig(num_layers=L, num_kv_heads=HKV, num_qo_heads=HQ, head_dim=D, page_size=16, max_pages=40, max_batch_size=3,
                           max_seq_len=64, dtype=torch.float16, device=DEV, backend=backend, cache_dtype=cache_dtype)
    return (KC.PagedKVCache if backend == "paged" else KC.ContiguousKVCache)(cfg)


def forward(ms, new, g):
    ids = ["a", "b"]
    ctxs = [m.begin_forward(ids, new) for m in ms]
    for layer in range(L):
        q, k, v = (torch.randn(2, max(new), h, D, generator=g).half().to(DEV) for h in (HQ, HKV, HKV))
        x, y = (c.attend(layer, q, k, v, HQ, HKV) for c in ctxs)
        assert torch.equal(x, y)
    for m, c in zip(ms, ctxs):
        m.end_forward(c)


@pytest.mark.parametrize("cache_dtype", [None, "int8"])
def test_contiguous_pools_moved_between_forwards(cache_dtype):
    g = torch.Generator().manual_seed(1)
    ms = [make("contiguous", cache_dtype) for _ in range(2)]
    for m in ms:
        for s in ("a", "b"):
            m.allocate_sequence(s)
    forward(ms, [9, 4], g)
    forward(ms, [1, 1], g)
    m = ms[1]
    for move in range(2):
        old = [m.k, m.v]
        m.k, m.v = m.k.clone(), m.v.clone()
        if cache_dtype:
            old += [m.pools.k_scale, m.pools.v_scale]
            m.pools.k_scale, m.pools.v_scale = m.pools.k_scale.clone(), m.pools.v_scale.clone()
        for t in old:
            t.zero_()
        forward(ms, [1, 1], g)
        forward(ms, [1, 1], g)
        forward(ms, [5, 2], g)
        assert not any(t.any() for t in old)
    assert torch.equal(ms[0].k.view(torch.int8), m.k.view(torch.int8))
    m.allocate_sequence("c")  # its slot is zeroed where the pool is now
    assert not m.k[:, 2].any()


@pytest.mark.parametrize("cache_dtype", [None, "int8"])
def test_paged_pools_replaced_before_use(cache_dtype):
    """A pool in memory that the caller brought, not zeros: pages are zeroed when they are taken, and copied on write, there."""
    m = make("paged", cache_dtype)
    pool = m.pool
    pool.k, pool.v = (torch.full_like(t, 3) for t in (pool.k, pool.v))
    m.allocate_sequence("a", num_tokens=20)
    pages = m.seqs["a"].block_table
    assert not pool.k[:, pages].any() and not pool.v[:, pages].any()
    pool.k[:, pages[1]] = 5
    copy = pool.cow(pages[1])
    assert (pool.k[:, copy] == 5).all() and not pool.v[:, copy].any()
