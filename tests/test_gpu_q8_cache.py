"""8-bit caches through the managers: prefill, decode, rotary embedding, shared prefixes and copy-on-write, the
contiguous backend and replayed steps, against a plain 64-bit cache that is given the same rows."""
import numpy as np
import pytest
import torch

from oracle import q8_oracle as Q

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
L, HQ, HKV, D = 2, 8, 2, 128
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def make(code, dtype="fp16", ps=16, pages=64, backend="paged", smax=128, prefix=True):
    from nanoslg_amd import kv_cache as KC
    cfg = KC.KVCacheConfig(num_layers=L, num_kv_heads=HKV, num_qo_heads=HQ, head_dim=D, page_size=ps, max_pages=pages,
                           max_batch_size=4, max_seq_len=smax, dtype=DT[dtype], device=DEV, enable_prefix_caching=prefix,
                           backend=backend, cache_dtype=CODE[code])
    return (KC.PagedKVCache if backend == "paged" else KC.ContiguousKVCache)(cfg)


class Twin:
    """One sequence's tokens in 64 bits: a page table of its own (page i is page i), every layer's K and V."""

    def __init__(self, code, ps, pages=24):
        nb = -(-ps // 16)
        self.ps, self.code, self.len = ps, code, 0
        self.table = list(range(pages))
        self.side = [[Q.Layer(np.zeros((pages, ps, HKV, D)), np.zeros((pages, nb, HKV)), code) for _ in "kv"] for _ in range(L)]

    def prefix(self, n):
        """A sequence that shares this one's first n tokens (n inside a block: the block's scale comes along)."""
        t = Twin(self.code, self.ps, len(self.table))
        for mine, its in zip(self.side, t.side):
            for a, b in zip(mine, its):
                b.values[:], b.scale[:] = a.values, a.scale
        t.len = n
        return t


def forward(mgr, twins, ids, new, g, dtype, offs=None, rope=None, spread=1.0, check=True):
    """One forward through the manager and the twins; outputs within the bounds. Returns the outputs."""
    offs = offs or [0] * len(ids)
    S, B = max(o + n for o, n in zip(offs, new)), len(ids)
    ctx = mgr.begin_forward(ids, new, offs)
    outs = []
    for layer in range(L):
        q = torch.randn(B, S, HQ, D, generator=g).to(DT[dtype])
        k = (torch.randn(B, S, HKV, D, generator=g) * spread).to(DT[dtype])
        v = (torch.randn(B, S, HKV, D, generator=g) * spread).to(DT[dtype])
        o = ctx.attend(layer, q.to(DEV), k.to(DEV), v.to(DEV), HQ, HKV)
        outs.append(o)
        assert o.shape == (B, S, HQ * D) and o.dtype == DT[dtype]
        o = o.view(B, S, HQ, D).cpu().double().numpy()
        for b, sid in enumerate(ids):
            t, r = twins[sid], slice(offs[b], offs[b] + new[b])
            Q.write_kv(*t.side[layer], t.table, t.len, k[b, r].double().numpy(), v[b, r].double().numpy())
            pad = np.ones(S, bool)
            pad[r] = False
            assert not o[b, pad].any()
            if new[b] and check:
                n = t.len + new[b]
                by = "bf16half" if S > 1 and dtype == "bf16" else dtype  # a prefill's weights
                want, mag, big, low = Q.attend(q[b, r].double().numpy(), t.side[layer][0].read(t.table, n),
                                               t.side[layer][1].read(t.table, n), None, by)
                bound = Q.attention_bound(want, mag, big, low, n, by)
                off = np.abs(o[b, r] - want)
                assert (off <= bound).all(), (layer, sid, float((off / bound).max()))
    mgr.end_forward(ctx)
    for b, sid in enumerate(ids):
        twins[sid].len += new[b]
    return outs


def stored(mgr, twins):
    """Every sequence's stored codes and scales are the twin's, read through its block table."""
    for sid, t in twins.items():
        st = mgr.seqs[sid]
        bt = st.block_table
        for layer in range(L):
            for lay, codes, scale in zip(t.side[layer], (mgr.pool.k, mgr.pool.v), (mgr.pool.k_scale, mgr.pool.v_scale)):
                got = codes[layer, bt].float().double().cpu().numpy().reshape(-1, HKV, D)[:t.len]
                sc = scale[layer, bt].double().cpu().numpy()
                np.testing.assert_array_equal(got, lay.values.reshape(-1, HKV, D)[:t.len], err_msg=f"{sid} layer {layer}")
                for tok in range(t.len):
                    np.testing.assert_array_equal(sc[tok // t.ps, tok % t.ps // 16],
                                                  lay.scale[tok // t.ps, tok % t.ps // 16], err_msg=f"{sid} token {tok}")


@pytest.mark.parametrize("ps", [16, 20, 32])
@pytest.mark.parametrize("code,dtype", [("e4m3", "fp16"), ("int8", "bf16")])
def test_paged_prefill_decode(code, dtype, ps):
    g = torch.Generator().manual_seed(1)
    m = make(code, dtype, ps)
    ids, lens = ["a", "b", "c"], [37, 5, 16]
    twins = {s: Twin(code, ps) for s in ids}
    for s, n in zip(ids, lens):
        m.allocate_sequence(s, num_tokens=n)
    forward(m, twins, ids, lens, g, dtype, offs=[0, 32, 21])  # left-padded
    stored(m, twins)
    for i in range(6):  # eager steps, planned on the device from the second on; scales grow
        forward(m, twins, ids, [1, 1, 1], g, dtype, spread=1.0 + i)
    forward(m, twins, ids[:2], [30, 1], g, dtype)  # a chunk and a token in one forward
    forward(m, twins, ["c", "a"], [1, 1], g, dtype)
    stored(m, twins)
    m.release_sequence("b")
    m.allocate_sequence("d", num_tokens=50)  # pages that held other tokens
    twins.pop("b")
    twins["d"] = Twin(code, ps)
    forward(m, twins, ["d"], [50], g, dtype)
    forward(m, twins, ["a", "c", "d"], [1, 1, 1], g, dtype)
    stored(m, twins)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_shared_prefix_and_copy_on_write(code):
    """Sequences on a cached prompt that ends inside a page: the page is copied with its scales at the first
    write, the others read theirs unchanged, and the decode reads the shared pages once for the group."""
    g = torch.Generator().manual_seed(2)
    m = make(code)
    prompt = list(range(1000, 1000 + 16 * 6 + 9))
    twins = {"first": Twin(code, 16)}
    m.allocate_sequence("first", token_ids=prompt)
    forward(m, twins, ["first"], [len(prompt)], g, "fp16")
    first = twins.pop("first")
    m.release_sequence("first")
    ids = ["x", "y", "z"]
    for s in ids:
        assert m.allocate_sequence(s, token_ids=prompt + [7]) == len(prompt)
        twins[s] = first.prefix(len(prompt))
    ctx_new = [3, 1, 2]
    forward(m, twins, ids, ctx_new, g, "fp16", spread=9.0)  # copies; the scale of the partial block grows in the copies
    stored(m, twins)
    for _ in range(3):
        forward(m, twins, ids, [1, 1, 1], g, "fp16", spread=2.0)
    assert m._dev_plan[1].groups is not None
    stored(m, twins)
    # the cached pages still read as the first sequence left them
    assert m.allocate_sequence("again", token_ids=prompt) == len(prompt)
    twins["again"] = first.prefix(len(prompt))
    stored(m, {"again": twins["again"]})


@pytest.mark.parametrize("smax", [128, 100])  # a slot is a page of smax tokens; 100 ends inside a block
@pytest.mark.parametrize("code,dtype", [("e4m3", "bf16"), ("int8", "fp16")])
def test_contiguous(code, dtype, smax):
    g = torch.Generator().manual_seed(3)
    m = make(code, dtype, backend="contiguous", smax=smax)
    ids = ["a", "b", "c"]
    twins = {s: Twin(code, smax, 1) for s in ids}
    for s in ids:
        m.allocate_sequence(s)
    forward(m, twins, ids, [60, 3, 33], g, dtype, offs=[0, 57, 27])
    for i in range(4):
        forward(m, twins, ids, [1, 1, 1], g, dtype, spread=1.0 + 2 * i)
    forward(m, twins, ids, [1, 1, 1], g, dtype, offs=[1, 0, 1])  # a padded step
    forward(m, twins, ids, [smax - 65, 20, 1], g, dtype)  # sequence a to the end of its slot
    for layer in range(L):
        for b, s in enumerate(ids):
            lay, t = twins[s].side[layer][0], twins[s]
            np.testing.assert_array_equal(m.k[layer, b, :t.len].float().double().cpu().numpy(), lay.values[0, :t.len])


@pytest.mark.parametrize("backend,ps", [("paged", 16), ("paged", 20), ("contiguous", 16)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_rope_forward_is_the_eager_rotation(backend, ps, dtype):
    """attend_rope against attend of rows that torch rotated: the same bits out and in the pool."""
    from nanoslg_amd import attention_forward
    g = torch.Generator().manual_seed(4)
    a = torch.outer(torch.arange(200, dtype=torch.float64), 1e4 ** (-torch.arange(0, D, 2) / D))
    a = torch.cat([a, a], 1)
    cos, sin = a.cos().float().to(DEV), a.sin().float().to(DEV)

    def rotate(x, pos):
        c, s = cos[pos][:, :, None].to(x.dtype), sin[pos][:, :, None].to(x.dtype)
        h = D // 2
        return x * c + torch.cat([-x[..., h:], x[..., :h]], -1) * s

    ms = [make("e4m3", dtype, ps, backend=backend) for _ in range(2)]
    ids = ["a", "b"]
    for m in ms:
        for s, n in zip(ids, (40, 23)):
            m.allocate_sequence(s, num_tokens=n)
    for new, offs in (([40, 23], [0, 17]), ([1, 1], None), ([1, 1], None), ([5, 9], [4, 0])):
        S = max(n + o for n, o in zip(new, offs or [0, 0]))
        c0, c1 = (m.begin_forward(ids, new, offs) for m in ms)
        pos = c0.get_position_ids(S)
        for layer in range(L):
            q, k, v = (torch.randn(2, S, h, D, generator=g).to(DT[dtype]).to(DEV) for h in (HQ, HKV, HKV))
            x = attention_forward(q, k, v, layer, HQ, HKV, cos, sin, c0)
            y = c1.attend(layer, rotate(q, pos), rotate(k, pos), v, HQ, HKV)
            assert torch.equal(x, y)
        for m, c in zip(ms, (c0, c1)):
            m.end_forward(c)
    pools = [m.pool if backend == "paged" else m.pools for m in ms]
    for name in ("k", "v", "k_scale", "v_scale"):
        x, y = (getattr(p, name) for p in pools)
        assert torch.equal(x.view(torch.int8) if x.element_size() == 1 else x, y.view(torch.int8) if y.element_size() == 1 else y)


@pytest.mark.parametrize("longest", [1070, 70])
@pytest.mark.parametrize("ps", [16, 20])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_graph_steps_match_eager_ones(code, ps, longest):
    """Steps replayed from the captured graphs, between eager work of another cache: the same bits. Few tokens: eager
    steps go out in one launch where 16 divides the page, so their sums are in another order."""
    from nanoslg_amd import kv_cache as KC
    g = torch.Generator().manual_seed(5)
    ms = [make(code, "fp16", ps, pages=120, prefix=False) for _ in range(2)]
    ids, lens = ["a", "b", "c"], [15, 16, longest]
    q0, k0 = (torch.randn(3, longest, h, D, generator=g).half().to(DEV) for h in (HQ, HKV))
    for m in ms:
        for s, n in zip(ids, lens):
            m.allocate_sequence(s, num_tokens=n)
        c = m.begin_forward(ids, lens)
        for layer in range(L):
            c.attend(layer, q0, k0, k0, HQ, HKV)
        m.end_forward(c)
    qs, ks, vs = (torch.zeros(3, 1, h, D, dtype=torch.float16, device=DEV) for h in (HQ, HKV, HKV))
    graph = KC.DecodeGraph(ms[0], ids, lambda ctx: [ctx.attend(layer, qs, ks, vs, HQ, HKV) for layer in range(L)])
    for _ in range(20):
        for t in (qs, ks, vs):
            t.copy_(torch.randn(t.shape, generator=g).half())
        outs = graph.step()
        c = ms[1].begin_forward(ids, [1] * 3)
        ref = [c.attend(layer, qs, ks, vs, HQ, HKV) for layer in range(L)]
        ms[1].end_forward(c)
        torch.cuda.synchronize()
        for x, y in zip(outs, ref):
            if longest < 1000 and ps == 16:
                # each is within 2^-11 |out| + (1 + 2^-11) (2 * 2^-11 + 2^-14) sum p |v| of the exact output (half weights,
                # rounded for P.V and for their sum; the scores' part for |q k| / sqrt(D) < 100; half's subnormals far
                # less), and sum p |v| <= max |v| < 6 here
                torch.testing.assert_close(x, y.reshape(x.shape), rtol=2 ** -10, atol=2 * 6 * (2 ** -10 + 2 ** -13))
            else:
                assert torch.equal(x, y.reshape(x.shape))
    for s in ids:
        a, b = (m.seqs[s].block_table for m in ms)
        assert torch.equal(ms[0].pool.k.view(torch.int8)[:, a], ms[1].pool.k.view(torch.int8)[:, b])


def test_factory_and_size():
    """nanoslg's factory with kv_cache_dtype; a pool sized from memory holds nearly twice the pages."""
    from types import SimpleNamespace as NS
    from nanoslg_amd import KVCacheConfig, create_cache_manager
    hf = NS(num_hidden_layers=L, num_key_value_heads=HKV, num_attention_heads=HQ, hidden_size=HQ * D)
    m = create_cache_manager(hf, None, DEV, torch.bfloat16, NS(max_kv_pages=32, kv_cache_dtype="fp8"))
    assert m.pool.k.dtype == torch.float8_e4m3fn and m.pool.k_scale.shape == (L, 32, 1, HKV)
    m.allocate_sequence("s", num_tokens=20)
    c = m.begin_forward(["s"], [20])
    x = torch.randn(1, 20, HQ, D, device=DEV).bfloat16()
    assert torch.isfinite(c.attend(0, x, x[:, :, :HKV], x[:, :, :HKV], HQ, HKV)).all()
    sizes = []
    for t in (None, torch.int8):
        cfg = KVCacheConfig(num_layers=32, num_kv_heads=8, num_qo_heads=32, head_dim=128, device=DEV, max_pages_cap=1 << 30,
                            cache_dtype=t)
        sizes.append(cfg.max_pages)
    assert 1.9 < sizes[1] / sizes[0] < 2.0


def test_refusals():
    from nanoslg_amd import kernels as K
    x = torch.zeros(4, 16, HKV, D, dtype=torch.int8, device=DEV)
    s = torch.zeros(4, 1, HKV, device=DEV)
    i = torch.zeros(2, dtype=torch.int32, device=DEV)
    r = torch.zeros(1, HKV, D, dtype=torch.float16, device=DEV)
    q = torch.zeros(1, HQ, D, dtype=torch.float16, device=DEV)
    ok = dict(k_new=r, v_new=r, qo_indptr=i, total_q=1, k_layer=x, v_layer=x, k_scale=s, v_scale=s, kv_indptr=i, kv_indices=i,
              kv_last_page_len=i)
    for bad, err in ((dict(k_layer=x.half(), v_layer=x.half()), TypeError), (dict(k_scale=s.half()), TypeError),
                     (dict(k_scale=s[:, :, :1]), ValueError), (dict(v_layer=x[:2]), ValueError), (dict(k_new=r.float()), TypeError),
                     (dict(v_new=r.bfloat16()), TypeError), (dict(k_new=r[:, :1]), ValueError), (dict(total_q=2), ValueError),
                     (dict(qo_indptr=i.long()), ValueError), (dict(qo_indptr=i[:1]), ValueError),
                     (dict(q_rows=i[:0], grid_width=1), ValueError), (dict(q_rows=i, grid_width=0), ValueError),
                     (dict(k_new=r.cpu()), ValueError), (dict(k_layer=x.transpose(0, 1), v_layer=x.transpose(0, 1)), ValueError)):
        with pytest.raises(err):
            K.append_kv_q8(**{**ok, **bad})
    dec = dict(q=q, k_layer=x, v_layer=x, k_scale=s, v_scale=s, kv_indptr=i, kv_indices=i, kv_last_page_len=i, total_pages=1)
    for bad, err in ((dict(q=q.float()), TypeError), (dict(q=q[:, :3]), ValueError), (dict(q=q[:, :, :64]), ValueError),
                     (dict(out=q.bfloat16()), ValueError), (dict(out=q.cpu()), ValueError), (dict(q=q[:0]), ValueError),
                     (dict(sm_scale=0.0), RuntimeError)):
        with pytest.raises(err):
            K.paged_decode_q8(**{**dec, **bad})
    with pytest.raises(ValueError):
        K.paged_decode_append_q8(k_new=torch.cat([r, r]), v_new=r, **dec)
    pre = dict(q=q, qo_indptr=i, total_q=1, max_q=1, **{k: v for k, v in dec.items() if k not in ("q", "total_pages")})
    for bad, err in ((dict(total_q=2), ValueError), (dict(q_rows=i, grid_width=2), ValueError), (dict(out=q[:, :4]), ValueError),
                     (dict(q=q[:, :3]), ValueError)):
        with pytest.raises(err):
            K.paged_prefill_q8(**{**pre, **bad})
    with pytest.raises(TypeError):
        K.gather_kv_q8(x, x, s, s, i, i, i, 16, torch.float64)


def test_decode_launch_refusals():
    from nanoslg_amd import kernels as K
    x = torch.zeros(L, 4, 16, HKV, D, dtype=torch.int8, device=DEV)
    s = torch.zeros(L, 4, 1, HKV, device=DEV)
    indptr, one = torch.tensor([0, 1], dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    ok = (x, x.clone(), s, s.clone(), one, indptr, one, one, 1, HQ)
    for at, bad, err in ((0, x[0], ValueError), (1, x[:1], ValueError), (2, s[:, :, :, :1], ValueError), (3, s.half(), TypeError),
                         (0, x.half(), ValueError), (0, x.cpu(), ValueError), (5, indptr.long(), ValueError), (9, HQ + 1, ValueError)):
        with pytest.raises(err):
            K.DecodeLaunchQ8(*ok[:at], bad, *ok[at + 1:])
    launch = K.DecodeLaunchQ8(*ok)
    q, r = torch.zeros(1, HQ, D, dtype=torch.float16, device=DEV), torch.zeros(1, HKV, D, dtype=torch.float16, device=DEV)
    rope = torch.zeros(64, D, device=DEV)
    for args, kw, err in (((L, q, r, r), {}, IndexError), ((-1, q, r, r), {}, IndexError), ((0, q.float(), r, r), {}, TypeError),
                          ((0, q, r.bfloat16(), r), {}, TypeError), ((0, q[:, :3], r, r), {}, ValueError),
                          ((0, q, r[:, :1], r), {}, ValueError), ((0, q, r, torch.cat([r, r])), {}, ValueError),
                          ((0, q.cpu(), r, r), {}, ValueError), ((0, q, r, r), dict(rope=(rope, rope, one.long())), ValueError),
                          ((0, q, r, r), dict(rope=(rope, rope, indptr)), ValueError)):
        with pytest.raises(err):
            launch(*args, **kw)
    assert not x.any() and launch(0, q, r, r).shape == (1, HQ, D)
    with pytest.raises(ValueError):
        launch.rebind(one, torch.zeros(3, dtype=torch.int32, device=DEV), one, one, 1)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("bad", [float("inf"), 6e4])
def test_a_request_does_not_change_the_prompt_that_others_share(code, bad):
    """A sequence writes a prompt and then a token that is not finite, or far larger than the prompt's, and is released
    with the prompt's ids alone. The next request on that prompt reads it as it was written."""
    g = torch.Generator().manual_seed(6)
    prompt = list(range(500, 521))
    m = make(code)
    twins = {"a": Twin(code, 16)}
    m.allocate_sequence("a", token_ids=prompt)
    forward(m, twins, ["a"], [21], g, "fp16")
    c = m.begin_forward(["a"], [1])
    for layer in range(L):
        x = torch.ones(1, 1, HQ, D, dtype=torch.float16, device=DEV)
        c.attend(layer, x, x[:, :, :HKV] * bad, x[:, :, :HKV] * bad, HQ, HKV)
    m.end_forward(c)
    m.release_sequence("a")
    got = m.allocate_sequence("b", token_ids=prompt + [9])
    twins = {"b": twins["a"].prefix(got)}
    o = forward(m, twins, ["b"], [22 - got], g, "fp16")
    assert all(torch.isfinite(x).all() for x in o)
    stored(m, twins)
