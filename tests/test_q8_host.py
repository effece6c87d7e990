"""8-bit cache: the C entry points' checks of arguments (no device work), the wrappers' refusal of CPU
tensors, and the oracle's format against torch's own float8 conversion."""
import numpy as np
import pytest
import torch

from oracle import q8_oracle as Q

A = 4096  # an aligned stand-in for a device address: every call below ends in a host check


def _lib():
    from nanoslg_amd import _lib
    return _lib


def append_args(**kw):
    a = dict(k=A, ks=1024, v=A, vs=1024, qo=A, rows=None, width=0, T=4, kp=A, vp=A, ksc=A, vsc=A, P=100, ps=16, ip=A, ix=A,
             ll=A, B=2, hkv=8, d=128, dt=0, code=0, stream=None)
    a.update(kw)
    return list(a.values())


def gather_args(**kw):
    a = dict(kp=A, vp=A, ksc=A, vsc=A, P=100, ps=16, ip=A, ix=A, ll=A, B=2, n=64, hkv=8, d=128, code=0, dt=0, ko=A, vo=A,
             stream=None)
    a.update(kw)
    return list(a.values())


def decode_args(**kw):
    a = dict(q=A, qs=4096, k=None, ks=0, v=None, vs=0, pos=None, cos=None, sin=None, ts=0, tr=0, kp=A, vp=A, ksc=A, vsc=A,
             P=100, ps=16, ip=A, ix=A, ll=A, tp=10, B=2, hq=32, hkv=8, d=128, scale=0.1, dt=0, code=0, slot=None, ng=0,
             pre=None, mem=None, out=A, os=4096, ws=None, wsn=0, layout=0, stream=None)
    a.update(kw)
    return list(a.values())


def prefill_args(**kw):
    a = dict(q=A, qs=4096, qo=A, rows=None, width=0, T=4, mq=4, kp=A, vp=A, ksc=A, vsc=A, P=100, ps=16, ip=A, ix=A, ll=A, B=2,
             hq=32, hkv=8, d=128, scale=0.1, dt=0, code=0, out=A, os=4096, ws=None, wsn=0, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("bad,status", [
    (dict(code=2), -1), (dict(code=-1), -1), (dict(d=96), -2), (dict(d=0), -1), (dict(dt=2), -2), (dict(dt=7), -2),
    (dict(ps=0), -1), (dict(P=0), -1), (dict(P=1 << 28, ps=16), -2), (dict(B=-1), -1), (dict(T=-1), -1), (dict(k=None), -1),
    (dict(qo=None), -1), (dict(ksc=None), -1), (dict(vsc=A + 2), -1), (dict(kp=A + 8), -1), (dict(k=A + 2), -1),
    (dict(ks=1028), -1), (dict(ks=512), -1), (dict(vs=0), -1), (dict(rows=A, width=0), -1), (dict(rows=A, width=1, T=3), -1),
    (dict(hkv=70000, ks=70000 * 128, vs=70000 * 128), -2), (dict(T=1 << 33), -1),
])
def test_append_refusals(bad, status):
    L = _lib()
    assert L.load().nslg_q8_append_kv(*append_args(**bad)) == status
    assert L.last_error()


@pytest.mark.parametrize("bad,status", [
    (dict(code=5), -1), (dict(d=80), -2), (dict(dt=9), -1), (dict(n=-1), -1), (dict(B=70000), -1), (dict(ko=None), -1),
    (dict(vo=A + 4), -1), (dict(ix=None), -1),
])
def test_gather_refusals(bad, status):
    assert _lib().load().nslg_q8_gather_kv(*gather_args(**bad)) == status


@pytest.mark.parametrize("bad,status", [
    (dict(code=2), -1), (dict(dt=2), -2), (dict(dt=3), -2), (dict(d=96), -2), (dict(hq=30), -1), (dict(hq=136), -2),
    (dict(scale=0.0), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(ksc=None), -1),
    (dict(ksc=A + 1), -1), (dict(kp=A + 8), -1), (dict(qs=4095), -1), (dict(qs=4097), -1), (dict(k=A, v=None, ks=1024), -1),
    (dict(k=A, v=A, ks=1024, vs=1024, ps=20), -2),  # a block may lie in two waves' work
    (dict(k=A, v=A, ks=1024, vs=1023), -1), (dict(k=A + 2, v=A, ks=1024, vs=1024), -1),
    (dict(cos=A, sin=A, pos=A, ts=128, tr=10), -1),  # tables without rows to rotate
    (dict(ng=33, slot=A, pre=A, mem=A), -2), (dict(ng=1, slot=None, pre=A, mem=A), -1), (dict(ng=-1), -2), (dict(tp=-1), -1),
    (dict(tp=1 << 28), -2), (dict(), -4),  # no workspace
])
def test_decode_refusals(bad, status):
    assert _lib().load().nslg_q8_paged_decode(*decode_args(**bad)) == status


@pytest.mark.parametrize("bad,status", [
    (dict(code=2), -1), (dict(dt=2), -2), (dict(d=96), -2), (dict(hq=30), -1), (dict(hq=136), -2), (dict(scale=-1.0), -1),
    (dict(vsc=None), -1), (dict(vsc=A + 2), -1), (dict(qs=64), -1), (dict(rows=A, width=0), -1), (dict(T=-1), -1),
])
def test_prefill_refusals(bad, status):
    assert _lib().load().nslg_q8_paged_prefill(*prefill_args(**bad)) == status


def test_empty_calls_do_nothing():
    lib = _lib().load()
    assert lib.nslg_q8_append_kv(*append_args(B=0, T=0)) == 0
    assert lib.nslg_q8_append_kv(*append_args(T=0, k=None, v=None)) == 0
    assert lib.nslg_q8_gather_kv(*gather_args(B=0)) == 0
    assert lib.nslg_q8_gather_kv(*gather_args(n=0, ko=None, vo=None)) == 0
    assert lib.nslg_q8_paged_decode(*decode_args(B=0)) == 0
    assert lib.nslg_q8_paged_prefill(*prefill_args(B=0)) == 0
    assert lib.nslg_q8_paged_prefill(*prefill_args(T=0)) == 0


def test_workspace_size():
    f = _lib().load().nslg_q8_paged_decode_workspace_size
    one = f(4, 32, 8, 128, 1000, 16, 0, 0, 0)
    assert one > 0 and f(4, 32, 8, 128, 1000, 16, 1, 1, 0) > 0
    assert f(4, 32, 8, 128, 1000, 16, 0, 0, 2) > one  # groups hold their members' partials
    for bad in ((4, 32, 8, 96, 1000, 16, 0, 0, 0), (4, 32, 8, 128, 1000, 16, 2, 0, 0), (4, 32, 8, 128, 1000, 16, 0, 2, 0),
                (4, 32, 8, 128, 1000, 16, 0, 0, 33), (4, 136, 8, 128, 1000, 16, 0, 0, 0), (0, 32, 8, 128, 10, 16, 0, 0, 0)):
        assert f(*bad) == 0


def test_wrappers_refuse_cpu_tensors():
    from nanoslg_amd import kernels as K
    x, s = torch.zeros(2, 16, 1, 64, dtype=torch.int8), torch.zeros(2, 1, 1)
    i = torch.zeros(2, dtype=torch.int32)
    rows = torch.zeros(1, 1, 64, dtype=torch.float16)
    for call in (lambda: K.append_kv_q8(rows, rows, i, 1, x, x, s, s, i, i, i), lambda: K.gather_kv_q8(x, x, s, s, i, i, i, 16),
                 lambda: K.paged_decode_q8(rows, x, x, s, s, i, i, i, 1),
                 lambda: K.paged_decode_append_q8(rows, rows, rows, x, x, s, s, i, i, i, 1),
                 lambda: K.paged_prefill_q8(rows, i, 1, 1, x, x, s, s, i, i, i)):
        with pytest.raises(ValueError, match="device tensors"):
            call()
    with pytest.raises(AttributeError):
        K.no_such_call


def test_oracle_rounds_e4m3_as_torch_does():
    x = np.concatenate([np.linspace(-448, 448, 20011), np.ldexp(np.linspace(-1, 1, 4001), -5)]).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(Q.round_code(x, "e4m3"), want)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_oracle_scale(code):
    M = Q.MOST[code]
    for e in (-126, -20, 0, 3, 100):
        assert Q.need_scale(M * 2.0 ** e, code) == 2.0 ** e
        assert Q.need_scale(M * 2.0 ** e * (1 + 2 ** -30), code) == 2.0 ** (e + 1)
    assert Q.need_scale(1e-45, code) == 2.0 ** -126 and Q.need_scale(0.0, code) == 0.0


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_oracle_error_of_written_rows(code):
    """A value read back is within half a step of the row written with the block's last scale, and within
    one step where the scale grew after it."""
    g = np.random.default_rng(0)
    lay = Q.Layer(np.zeros((2, 16, 1, 64)), np.zeros((2, 1, 1)), code)
    x = g.standard_normal((16, 1, 64)) * np.exp(2 * g.standard_normal((16, 1, 1)))
    for t in range(16):
        lay.write([1], t, x[t:t + 1])
    s = lay.scale[1, 0, 0]
    step = np.full_like(x, s) if code == "int8" else np.maximum(np.ldexp(1.0, np.frexp(np.abs(x))[1] - 4), s * 2.0 ** -9)
    off = np.abs(lay.read([1], 16) - x)
    assert (off <= step).all()
    assert (off[-1] <= step[-1] / 2 * (1 + 1e-12)).all()


def test_config_of_the_cache_type():
    from nanoslg_amd import KVCacheConfig
    base = dict(num_layers=2, num_kv_heads=2, num_qo_heads=4, head_dim=64, max_pages=8)
    for name, t in (("fp8", torch.float8_e4m3fn), ("fp8_e4m3", torch.float8_e4m3fn), ("int8", torch.int8), ("auto", None),
                    (None, None), (torch.int8, torch.int8), (torch.bfloat16, None)):
        assert KVCacheConfig(**base, cache_dtype=name).cache_dtype == t
    for bad in ("fp4", torch.float16, torch.float8_e5m2, torch.uint8):
        with pytest.raises(ValueError):
            KVCacheConfig(**base, cache_dtype=bad)
    with pytest.raises(ValueError, match="float16 and bfloat16"):
        KVCacheConfig(**base, dtype=torch.float32, cache_dtype="fp8")
    with pytest.raises(ValueError, match="head_dim"):
        KVCacheConfig(**{**base, "head_dim": 80}, cache_dtype="int8")


def test_pool_of_an_8_bit_cache():
    """Codes, their 16-bit words and the scales of the paged and the contiguous pool (host memory: no kernels)."""
    import fake_kernels
    from nanoslg_amd import ContiguousKVCache, KVCacheConfig, PagePool
    cfg = KVCacheConfig(num_layers=3, num_kv_heads=2, num_qo_heads=4, head_dim=64, page_size=20, max_pages=8, cache_dtype="int8")
    p = PagePool(cfg, kernels=fake_kernels)
    assert p.k.dtype == torch.int8 and p.k.shape == (3, 8, 20, 2, 64) and p.k_scale.shape == (3, 8, 2, 2)
    assert p.k_words.shape == (3, 8, 20, 2, 32) and p.k_words.data_ptr() == p.k.data_ptr()
    assert [t.data_ptr() for t in p.layer8(1)] == [t[1].data_ptr() for t in (p.k, p.v, p.k_scale, p.v_scale)]
    p.k.random_(-127, 128), p.v.random_(-127, 128), p.k_scale.uniform_(), p.v_scale.uniform_()
    src, dst = p.alloc(1, zero=False)[0], p.cow(1)
    for t in (p.k, p.v, p.k_scale, p.v_scale):  # copy-on-write takes the scales along
        assert torch.equal(t[:, src], t[:, dst])
    p.zero([src])
    assert not p.k[:, src].any() and not p.v[:, src].any() and p.k[:, dst].any()
    c = ContiguousKVCache(KVCacheConfig(num_layers=1, num_kv_heads=2, num_qo_heads=4, head_dim=64, max_batch_size=2, max_seq_len=100,
                                        backend="contiguous", cache_dtype="fp8"), kernels=fake_kernels)
    assert c.k.dtype == torch.float8_e4m3fn and c.pools.v_scale.shape == (1, 2, 7, 2)


def test_fast_binding_of_the_8_bit_entry_points():
    """_nslg_fast_q8 calls the same C functions as ctypes, with the types of their declarations."""
    import re
    from ctypes import c_float, c_int32, c_int64, c_size_t, c_void_p
    from pathlib import Path
    L = _lib()
    lib, fast = L.load(), L.fast_q8()
    assert fast.append_kv(*append_args(code=2)) == lib.nslg_q8_append_kv(*append_args(code=2)) == -1
    assert fast.gather_kv(*gather_args(d=80)) == -2 and fast.paged_prefill(*prefill_args(dt=2)) == -2
    assert fast.paged_decode(*decode_args()) == L.NSLG_EWORKSPACE
    with pytest.raises(TypeError):
        fast.append_kv(*append_args()[:-1])
    code = {c_void_p: "p", c_int64: "q", c_int32: "i", c_size_t: "z", c_float: "f"}
    src = (Path(__file__).resolve().parent.parent / "nanoslg_amd" / "csrc" / "fastcall_q8.c").read_text()
    found = re.findall(r'parse\("(\w+)", "(\w+)"', src)
    assert len(found) == 4
    for fn, sig in found:
        assert sig == "".join(code[t] for t in L.SIGNATURES["nslg_" + fn][1]), fn


@pytest.mark.parametrize("groups", [0, 3])
@pytest.mark.parametrize("batch,hq,hkv,d,page", [(192, 64, 8, 128, 16), (288, 48, 8, 128, 128), (300, 32, 8, 64, 20), (400, 16, 2, 256, 32),
                                                 (1500, 8, 1, 128, 16), (5, 32, 8, 128, 16)])
def test_workspace_size_serves_every_smaller_call(batch, hq, hkv, d, page, groups):
    """A workspace sized for a number of pages is enough for a call of fewer (as DecodeLaunch and DecodeLaunchQ8 rely on):
    the size asked for does not fall as pages come, though a call's own chunks may become fewer."""
    from nanoslg_amd import _lib as L
    lib = L.load()
    pages = sorted({batch, *range(batch, batch + 40), *(batch + round(1.03 ** i) for i in range(330))})
    for dt in (L.NSLG_F16, L.NSLG_BF16, L.NSLG_F32):
        sizes = []
        if dt != L.NSLG_F32:
            sizes = [[lib.nslg_q8_paged_decode_workspace_size(batch, hq, hkv, d, p, page, dt, code, groups) for p in pages]
                     for code in (L.NSLG_E4M3, L.NSLG_INT8)]
        if not groups:
            sizes.append([lib.nslg_paged_decode_workspace_size(batch, hq, hkv, d, p, page, dt) for p in pages])
        elif dt != L.NSLG_F32:
            sizes.append([lib.nslg_paged_decode_grouped_workspace_size(batch, hq, hkv, d, p, page, dt, groups) for p in pages])
        for s in sizes:
            assert min(s) > 0 and s == sorted(s)


@pytest.mark.parametrize("code", [None, "int8", "fp8"])
@pytest.mark.parametrize("page,prompt,later,want", [
    (16, 21, 2, 16),  # the tail block (tokens 16 .. 20) holds tokens 21 and 22 too
    (16, 21, 0, 21), (16, 32, 3, 32), (16, 9, 1, 0), (16, 9, 0, 9),
    (64, 16 * 6 + 5, 1, 16 * 6), (64, 16 * 6 + 5, 0, 16 * 6 + 5), (64, 16 * 6, 9, 16 * 6), (64, 70, 59, 64),
    (20, 39, 1, 36), (20, 20, 7, 20), (20, 33, 2, 20), (20, 37, 2, 36),
])
def test_a_cached_tail_holds_no_later_tokens(code, page, prompt, later, want):
    """A released sequence's last page is cached for the ids that were given. Where it holds later tokens (generated, ids
    never given), their values are in an 8-bit block's scale: what is shared ends with the last block without them."""
    import fake_kernels
    from nanoslg_amd import KVCacheConfig, PagedKVCache
    m = PagedKVCache(KVCacheConfig(num_layers=1, num_kv_heads=2, num_qo_heads=4, head_dim=64, page_size=page, max_pages=40,
                                   cache_dtype=code), kernels=fake_kernels)
    ids = list(range(100, 100 + prompt))
    assert m.allocate_sequence("a", token_ids=ids) == 0
    for n in [prompt] + [1] * later:
        m.end_forward(m.begin_forward(["a"], [n]))
    m.release_sequence("a")
    want = prompt if code is None else want
    assert m.allocate_sequence("b", token_ids=ids + [7, 8]) == want
    m.end_forward(m.begin_forward(["b"], [prompt + 2 - want]))  # (its ids are all given: its whole tail is cached)
    m.release_sequence("b")
    assert m.allocate_sequence("c", token_ids=ids + [7, 8, 9]) == prompt + 2


def test_a_failed_forward_leaves_no_tail_to_share():
    """Rows of a forward that did not end are in the tail block's scale too."""
    import fake_kernels
    from nanoslg_amd import KVCacheConfig, PagedKVCache
    m = PagedKVCache(KVCacheConfig(num_layers=1, num_kv_heads=2, num_qo_heads=4, head_dim=64, page_size=16, max_pages=40,
                                   cache_dtype="int8"), kernels=fake_kernels)
    ids = list(range(100, 121))
    m.allocate_sequence("a", token_ids=ids)
    m.end_forward(m.begin_forward(["a"], [21]))
    m.begin_forward(["a"], [1])  # written, perhaps, and given up
    m.release_sequence("a")
    assert m.allocate_sequence("b", token_ids=ids) == 16


@pytest.mark.parametrize("call", ["paged_decode_rope_append", "paged_decode_rope_append_q8"])
def test_rope_tables_on_another_device_are_refused(call):
    """Positions and tables that agree with each other, but are not where q is (stand-ins: only what the check looks at)."""
    from types import SimpleNamespace
    from nanoslg_amd import kernels as K

    def on(device, *shape, dtype=torch.float32):
        n = int(np.prod(shape))
        return SimpleNamespace(is_cuda=True, device=torch.device(device), get_device=lambda: int(device[-1]), dtype=dtype, shape=shape,
                               numel=lambda: n, is_contiguous=lambda: True, dim=lambda: len(shape), stride=lambda i: (shape[-1], 1)[i])

    q = on("cuda:0", 2, 4, 64, dtype=torch.float16)
    for other in range(3):
        pos, cos, sin = (on("cuda:1" if other != i else "cuda:0", *s, dtype=t) for i, (s, t) in
                         enumerate((((2,), torch.int32), ((9, 64), torch.float32), ((9, 64), torch.float32))))
        rest = [q] * (8 if call.endswith("q8") else 6)
        with pytest.raises(ValueError, match="different devices"):
            getattr(K, call)(q, q, q, pos, cos, sin, *rest[:-1], 1)
    pos, cos, sin = on("cuda:1", 2, dtype=torch.int32), on("cuda:1", 9, 64), on("cuda:1", 9, 64)
    with pytest.raises(ValueError, match="different devices"):
        getattr(K, call)(q, q, q, pos, cos, sin, *rest[:-1], 1)
