"""8-bit cache kernels against plain 64-bit arithmetic: the write (codes and scales, exactly), the
read-back (exactly) and attention (within bounds derived in the oracle from the roundings)."""
import math

import numpy as np
import pytest
import torch

from oracle import q8_oracle as Q

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
DEV = "cuda:0"


def K():
    from nanoslg_amd import kernels
    return kernels


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


class Cache:
    """A layer on the GPU and its oracle twin, with sequences in scattered pages. Every slot starts as written."""

    def __init__(self, seed, code, page, hkv, d, lens, dtype="fp16", extra_pages=3, spread=1.5, stale_nan=False):
        self.g = g = np.random.default_rng(seed)
        self.code, self.page, self.hkv, self.d, self.lens, self.dtype = code, page, hkv, d, list(lens), dtype
        npg = [-(-n // page) for n in lens]
        P = self.P = sum(npg) + extra_pages + 1
        nb = -(-page // 16)
        order = g.permutation(np.arange(1, P))
        at = np.concatenate([[0], np.cumsum(npg)])
        self.tables = [order[a:b].tolist() for a, b in zip(at[:-1], at[1:])]
        self.side = {}
        for name in "kv":
            s = np.ldexp(1.0, g.integers(-6, 3, (P, nb, hkv)))
            lim = Q.MOST[code]
            v = Q.round_code(np.clip(g.standard_normal((P, page, hkv, d)) * lim / 4 * spread, -lim, lim), code)
            v *= g.random((P, page, hkv, 1)) < 0.97  # some rows of zeros
            if stale_nan and code == "e4m3":  # slots past every sequence hold NaN
                for tab, n in zip(self.tables, lens):
                    if n % page:
                        v[tab[-1], n % page:] = np.nan
                v[order[at[-1]:]] = np.nan
            if stale_nan:  # and so do the scales of blocks without a token
                for tab, n in zip(self.tables, lens):
                    if n % page:
                        s[tab[-1], -(-(n % page) // 16):] = np.nan
                s[order[at[-1]:]] = np.nan
            lay = Q.Layer(v, s, code)
            t = torch.from_numpy(v).float()
            t = t.to(CODE[code]) if code == "e4m3" else t.to(torch.int8)
            self.side[name] = (lay, t.to(DEV).contiguous(), torch.from_numpy(s).float().to(DEV).contiguous())
        self.indptr, self.indices = i32(at), i32(np.concatenate([*self.tables, [0]]).astype(np.int64)[:max(1, at[-1])])
        self.last = i32([n - (p - 1) * page if p else 0 for n, p in zip(lens, npg)])
        self.total_pages = int(at[-1])

    @property
    def layer(self):
        return (self.side["k"][1], self.side["v"][1], self.side["k"][2], self.side["v"][2])

    @property
    def table(self):
        return (self.indptr, self.indices, self.last)

    def rows(self, n, scale=1.0):
        x = self.g.standard_normal((n, self.hkv, self.d)) * scale * np.exp(self.g.standard_normal((n, 1, 1)))
        return torch.from_numpy(x).to(DT[self.dtype])

    def values(self, name, b):
        return self.side[name][0].read(self.tables[b], self.lens[b])

    def same(self):
        for name in "kv":
            lay, codes, scale = self.side[name]
            np.testing.assert_array_equal(scale.cpu().double().numpy(), lay.scale, err_msg=name + " scales")
            np.testing.assert_array_equal(codes.cpu().float().double().numpy(), lay.values, err_msg=name + " codes")


def append(c, new, kn, vn, grid=0, offs=None):
    """The forward's rows through the kernel and the oracle: new[b] last tokens of each sequence."""
    qo = np.concatenate([[0], np.cumsum(new)])
    kw = {}
    rows = [list(range(qo[b], qo[b + 1])) for b in range(len(new))]
    if grid:
        rows = [[b * grid + offs[b] + t for t in range(n)] for b, n in enumerate(new)]
        kw = dict(q_rows=i32(sum(rows, []) or [0]), grid_width=grid)
    K().append_kv_q8(kn, vn, i32(qo), int(qo[-1]), *c.layer, *c.table, **kw)
    k, v = (x.reshape(-1, c.hkv, c.d).cpu().double().numpy() for x in (kn, vn))
    for b, n in enumerate(new):
        Q.write_kv(c.side["k"][0], c.side["v"][0], c.tables[b], c.lens[b] - n, k[rows[b]], v[rows[b]])


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("page,d,hkv,dtype,lens,new", [
    (16, 128, 8, "fp16", [1, 16, 17, 40, 100, 3], [1, 16, 1, 24, 37, 0]),
    (16, 128, 8, "bf16", [33, 64], [1, 1]),
    (32, 64, 3, "bf16", [31, 97, 5], [14, 66, 5]),
    (64, 256, 2, "fp16", [130, 64], [67, 1]),
    (20, 128, 4, "fp16", [45, 20, 19, 81], [30, 4, 1, 81]),
    (5, 64, 8, "bf16", [23, 4], [9, 2]),
    (1, 128, 2, "fp16", [7, 2], [7, 1]),
    (48, 128, 1, "fp16", [500], [411]),
])
def test_append_codes_and_scales(code, page, d, hkv, dtype, lens, new):
    c = Cache(1, code, page, hkv, d, lens, dtype)
    T = sum(new)
    append(c, new, c.rows(T).to(DEV), c.rows(T, 30.0).to(DEV))
    c.same()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_append_padded_grid_and_strided_rows(code):
    c = Cache(2, code, 16, 4, 128, [50, 7, 20], "bf16")
    new, W = [9, 7, 1], 12
    offs = [W - n for n in new]
    kv = torch.randn(3, W, 2, 4, 128, device=DEV).bfloat16()  # K and V as halves of one projection output
    append(c, new, kv[:, :, 0], kv[:, :, 1], grid=W, offs=offs)
    c.same()


@pytest.mark.parametrize("shift", [1, 4])
def test_append_rows_off_16_byte_alignment(shift):
    c = Cache(3, "e4m3", 16, 2, 64, [20, 18])
    flat = torch.randn(2 * 3 * 128 + 8, device=DEV).half()
    kn = flat[shift:shift + 3 * 128].view(3, 2, 64)
    append(c, [2, 1], kn, kn.clone())
    c.same()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_append_extremes(code, dtype):
    """The largest and smallest values, values at and just past MOST * 2^k, zero rows, a scale that grows by far."""
    lim = Q.MOST[code]
    big = 65504.0 if dtype == "fp16" else 3.3e38
    tiny = 2.0 ** -24 if dtype == "fp16" else 2.0 ** -133
    amax = [lim, lim * 2.0 ** -5, lim + (0.5 if code == "int8" else 1.0), big, tiny, 0.0, 1e-30, lim * 2 - 1]
    c = Cache(4, code, 16, 1, 64, [16 + i % 5 + 1 for i in range(len(amax))], dtype)
    rows = []
    for i, a in enumerate(amax):
        n = i % 5 + 1
        x = c.rows(n)
        x = x / x.abs().max().float().clamp(min=1) * 0.7 if a == 0 else (x.float() / x.float().abs().max() * a).to(DT[dtype])
        if a == 0:
            x = torch.zeros_like(x)
        elif math.isfinite(a):
            x[n // 2, 0, 5] = a
        rows.append(x)
    x = torch.cat(rows).to(DEV)
    append(c, [i % 5 + 1 for i in range(len(amax))], x, -x)
    c.same()
    # one more token each: blocks that hold tokens, scales growing and not
    c2 = Cache(5, code, 16, 1, 64, [18] * 6, dtype)
    y = c2.rows(6).float() * torch.tensor([1e-3, 1.0, 1e2, 1e4, 0.0, 6e4]).view(6, 1, 1)
    y = y.clamp(-big, big).to(DT[dtype]).to(DEV)
    append(c2, [1] * 6, y, y.flip(0))
    c2.same()
    append(c2, [1] * 6, y.flip(0), y)  # the same slots once more
    c2.same()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_append_values_that_are_not_finite(code, bad):
    c = Cache(6, code, 16, 2, 64, [20, 33, 20], "bf16")
    x, y = c.rows(9), c.rows(9)
    x[1, 0, 3] = bad   # sequence 0: K of token 17, head 0
    y[3, 1, 40] = bad  # V of token 19, head 1
    x[8, 1, 63] = bad  # sequence 2: its only new token, head 1
    append(c, [4, 4, 1], x.to(DEV), y.to(DEV))
    c.same()
    k, v = K().gather_kv_q8(*c.layer, *c.table, 33, torch.float32)
    want = [c.values("k", b) for b in range(3)]
    for b in range(3):
        np.testing.assert_array_equal(k[b, :c.lens[b]].cpu().double().numpy(), want[b])
    assert np.isnan(want[0][17, 0]).any() and np.isnan(want[0][19, 1]).any() and not np.isnan(want[1]).any()
    assert not torch.isnan(v).any()
    # the block written from its first slot again is whole again
    append(c, [20, 33, 20], c.rows(73).to(DEV), c.rows(73).to(DEV))
    c.same()
    assert not torch.isnan(K().gather_kv_q8(*c.layer, *c.table, 33, torch.float32)[0]).any()


@pytest.mark.parametrize("in_v", [False, True])
@pytest.mark.parametrize("page", [16, 20])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_only_queries_that_see_it_get_what_is_not_finite(dtype, code, page, in_v):
    """A token that is not finite, in K or V: NaN for its own and later queries of that KV head, nothing for those before it
    (int8: before its block)."""
    n, at = 70, 50
    c = Cache(18, code, page, 2, 128, [n, 40], dtype)
    kn, vn = c.rows(n), c.rows(n)
    (vn if in_v else kn)[at, 1, 77] = math.inf
    append(c, [n, 0], kn.to(DEV), vn.to(DEV))
    c.same()
    q = torch.randn(n, 8, 128, device=DEV).to(DT[dtype])
    out = K().paged_prefill_q8(q, i32([0, n, n]), n, n, *c.layer, *c.table)
    first = at if code == "e4m3" else at - at % page % 16
    assert torch.isnan(out[at:, 4:]).all()
    assert torch.isfinite(out[:first, 4:]).all() and torch.isfinite(out[:, :4]).all()
    c.side["k"][0].values[np.isnan(c.side["k"][0].values)] = 0
    c.side["k"][0].scale[np.isnan(c.side["k"][0].scale)] = 0
    by = "bf16half" if dtype == "bf16" else dtype
    want = Q.attend(q.cpu().double().numpy(), c.values("k", 0), c.values("v", 0), None, by)
    bound = Q.attention_bound(*want, n, by)
    off = np.abs(out.cpu().double().numpy() - want[0])
    assert (off <= bound)[:first].all() and (off <= bound)[:, :4].all()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_append_skips_bad_pages_and_writes_nothing_else(code):
    c = Cache(7, code, 16, 2, 64, [40, 20, 5])
    before = [t.clone() for t in c.layer]
    idx = c.indices.clone()
    idx[1], idx[3] = -1, c.P  # sequence 0's second page, sequence 1's first
    c.indices = idx
    T = 40 + 20
    kn = c.rows(T)
    qo = i32([0, 40, 60, 60])
    K().append_kv_q8(kn.to(DEV), kn.to(DEV), qo, T, *c.layer, *c.table)
    x = kn.double().numpy()
    for b, (a, n) in enumerate(((0, 40), (40, 20))):
        for p in range(-(-n // 16)):
            pid = int(idx[(0, 3)[b] + p])
            if 0 <= pid < c.P:
                r = x[a + 16 * p:a + min(n, 16 * p + 16)]
                Q.write_kv(c.side["k"][0], c.side["v"][0], {p: pid}, 16 * p, r, r)
    c.same()
    assert len(before) == 4


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("out", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page,d", [(16, 128), (20, 64), (64, 256), (3, 64)])
def test_gather(code, out, page, d):
    c = Cache(8, code, page, 3, d, [37, 0, 1, 64], stale_nan=True)
    k, v = K().gather_kv_q8(*c.layer, *c.table, 66, out)
    for name, got in (("k", k), ("v", v)):
        for b, n in enumerate(c.lens):
            want = torch.from_numpy(c.values(name, b)).float().to(out)
            assert torch.equal(got[b, :n].cpu(), want), (name, b)
            assert not got[b, n:].any()


def check(c, out, q, b, new=1, scale=None, prefill=False):
    """Sequence b's output rows against the oracle's."""
    dtype = "bf16half" if prefill and c.dtype == "bf16" else c.dtype
    want, mag, big, low = Q.attend(q.cpu().double().numpy(), c.values("k", b), c.values("v", b), scale, dtype)
    bound = Q.attention_bound(want, mag, big, low, c.lens[b], dtype)
    off = np.abs(out.cpu().double().numpy() - want)
    assert (off <= bound).all(), (b, float((off / bound).max()))


DECODE = [  # page, d, hkv, group, lens
    (16, 128, 8, 4, [1, 16, 17, 100, 0, 700]),
    (16, 128, 1, 16, [33, 2500]),
    (16, 64, 2, 1, [15, 31, 300]),
    (32, 256, 4, 4, [1, 64, 65, 900]),
    (64, 128, 3, 7, [129, 5000]),
    (48, 64, 5, 8, [47, 48, 49, 1]),
    (20, 128, 4, 4, [1, 39, 40, 41, 777]),
    (8, 256, 2, 2, [9, 250]),
    (1, 64, 2, 3, [1, 50]),
    (16, 128, 8, 4, [1, 16, 0, 1700]),  # (past what one launch takes; of the above the first, third and sixth are not)
    (32, 256, 4, 4, [1, 33, 300]),
    (16, 128, 1, 16, [300, 5]),
    (64, 128, 3, 7, [129, 500]),
    (16, 64, 16, 2, [1, 15, 16, 17, 31, 32, 33, 0, 64, 255, 257]),
    (16, 128, 64, 1, [20, 100, 3, 4, 5]),
]


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("page,d,hkv,group,lens", DECODE)
def test_decode(code, dtype, page, d, hkv, group, lens):
    c = Cache(9, code, page, hkv, d, lens, dtype, stale_nan=True)
    wide = torch.randn(len(lens), hkv * group + 2, d, device=DEV).to(DT[dtype])
    q = wide[:, 1:-1]  # strided rows
    out = K().paged_decode_q8(q, *c.layer, *c.table, c.total_pages)
    for b, n in enumerate(lens):
        if n:
            check(c, out[b:b + 1], q[b:b + 1], b)
        else:
            assert not out[b].any()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("page,d,hkv,group,lens", [x for x in DECODE if 0 not in x[4]])
def test_decode_append(code, dtype, page, d, hkv, group, lens):
    """The step's rows written (codes and scales, exactly) and attended, in one call; a second step behind it."""
    c = Cache(10, code, page, hkv, d, lens, dtype)
    B = len(lens)
    q = torch.randn(B, hkv * group, d, device=DEV).to(DT[dtype])
    for scale in (1.0, 40.0):
        kn, vn = c.rows(B, scale), c.rows(B, scale)
        out = K().paged_decode_append_q8(q, kn.to(DEV)[:, None], vn.to(DEV)[:, None], *c.layer, *c.table, c.total_pages)
        for b in range(B):
            Q.write_kv(c.side["k"][0], c.side["v"][0], c.tables[b], lens[b] - 1, kn[b:b + 1].double().numpy(), vn[b:b + 1].double().numpy())
        c.same()
        for b in range(B):
            check(c, out[b:b + 1], q[b:b + 1], b)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 32), (256, 16), (128, 20)])
@pytest.mark.parametrize("longest", [257, 1800])
def test_decode_rope_append(dtype, d, page, longest):
    """Bit for bit rope_append into rows of its own, then the decode of the rotated rows."""
    lens, hkv, G = [5, 40, longest], 2, 4
    c = Cache(11, "e4m3", page, hkv, d, lens, dtype)
    twin = [t.clone() for t in c.layer]
    B = len(lens)
    q = torch.randn(B, hkv * G, d, device=DEV).to(DT[dtype])
    kn, vn = c.rows(B, 5).to(DEV), c.rows(B, 5).to(DEV)
    a = torch.outer(torch.arange(2000, dtype=torch.float64), 1e4 ** (-torch.arange(0, d, 2) / d))
    a = torch.cat([a, a], 1)
    cos, sin = a.cos().float().to(DEV), a.sin().float().to(DEV)
    pos = i32([n - 1 for n in lens])
    out = K().paged_decode_rope_append_q8(q, kn, vn, pos, cos, sin, *c.layer, *c.table, c.total_pages)
    kr, vr = torch.empty(B, 1, hkv, d, device=DEV, dtype=DT[dtype]), torch.empty(B, 1, hkv, d, device=DEV, dtype=DT[dtype])
    qr = K().rope_append(q, kn, vn, pos, i32(range(B)), cos, sin, kr, vr)
    K().append_kv_q8(kr[:, 0], vn, i32(range(B + 1)), B, *twin, *c.table)
    for x, y in zip(c.layer, twin):
        assert torch.equal(x.view(torch.int8) if x.element_size() == 1 else x, y.view(torch.int8) if y.element_size() == 1 else y)
    assert torch.equal(out, K().paged_decode_q8(qr, *twin, *c.table, c.total_pages))


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_decode_groups(code):
    """Sequences on one prefix of pages, read once for the group: the same result within the bounds."""
    c = Cache(12, code, 16, 2, 128, [200, 161, 170, 33], "fp16")
    for b in (1, 2):  # their first 8 pages are sequence 0's
        c.tables[b][:8] = c.tables[0][:8]
    c.indices = i32(sum(c.tables, []))
    grp = K().DecodeGroups(4, [[0, 1, 2]], [8], torch.device(DEV))
    q = torch.randn(4, 8, 128, device=DEV).half()
    kn, vn = c.rows(4, 20), c.rows(4, 20)
    out = K().paged_decode_append_q8(q, kn.to(DEV), vn.to(DEV), *c.layer, *c.table, c.total_pages, groups=grp)
    for b in range(4):
        Q.write_kv(c.side["k"][0], c.side["v"][0], c.tables[b], c.lens[b] - 1, kn[b:b + 1].double().numpy(), vn[b:b + 1].double().numpy())
    c.same()
    for b in range(4):
        check(c, out[b:b + 1], q[b:b + 1], b)


@pytest.mark.parametrize("n", [40, 1000])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_decode_of_a_block_that_is_not_finite(code, n):
    """What reads such a block is NaN; other heads and sequences are not touched."""
    c = Cache(13, code, 16, 2, 64, [n, n], "fp16")
    x = c.rows(2)
    x[0, 0, 7] = math.nan
    q = torch.randn(2, 4, 64, device=DEV).half()
    out = K().paged_decode_append_q8(q, x.to(DEV), c.rows(2).to(DEV), *c.layer, *c.table, c.total_pages)
    assert torch.isnan(out[0, :2]).all()
    assert torch.isfinite(out[0, 2:]).all() and torch.isfinite(out[1]).all()


PREFILL = [  # page, d, hkv, group, lens, new
    (16, 128, 8, 4, [1, 40, 300, 17], [1, 40, 60, 0]),
    (16, 128, 1, 16, [900], [70]),
    (64, 64, 2, 3, [129, 64, 500], [129, 1, 200]),
    (32, 256, 2, 4, [70, 400], [33, 150]),
    (20, 128, 4, 1, [41, 39, 300], [41, 3, 120]),
    (5, 64, 2, 4, [23], [23]),
    (16, 128, 2, 4, [2300], [16]),
]


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("page,d,hkv,group,lens,new", PREFILL)
def test_prefill(code, dtype, page, d, hkv, group, lens, new):
    c = Cache(14, code, page, hkv, d, lens, dtype, stale_nan=True)
    qo = np.concatenate([[0], np.cumsum(new)])
    T, hq = int(qo[-1]), hkv * group
    q = torch.randn(T, hq + 1, d, device=DEV).to(DT[dtype])[:, :hq]
    ws = K().Workspace(torch.device(DEV))
    out = K().paged_prefill_q8(q, i32(qo), T, max(new), *c.layer, *c.table, workspace=ws)
    whole = K().paged_prefill_q8(q, i32(qo), T, max(new), *c.layer, *c.table, max_kv=0)  # keys in one run
    W = max(new) + 3
    offs = [W - n for n in new]
    rows = [b * W + offs[b] + t for b, n in enumerate(new) for t in range(n)]
    grid = torch.zeros(len(lens) * W, hq, d, device=DEV, dtype=DT[dtype])
    grid[rows] = q
    padded = K().paged_prefill_q8(grid, i32(qo), T, max(new), *c.layer, *c.table, workspace=ws, q_rows=i32(rows), grid_width=W)
    pad = torch.ones(len(lens) * W, dtype=torch.bool)
    pad[rows] = False
    assert not padded[pad.to(DEV)].any()
    assert torch.equal(padded[rows], out)
    for b in range(len(lens)):
        if new[b]:
            check(c, out[qo[b]:qo[b + 1]], q[qo[b]:qo[b + 1]], b, prefill=True)
            check(c, whole[qo[b]:qo[b + 1]], q[qo[b]:qo[b + 1]], b, prefill=True)


def test_write_then_attend_as_a_forward_does():
    """A prompt in two chunks and three decode steps, each call on what the calls before left."""
    c = Cache(15, "e4m3", 16, 2, 128, [90, 57], "bf16")
    full = c.lens
    kn, vn = [c.rows(95, 3) for _ in full], [c.rows(95, 3) for _ in full]
    ws = K().Workspace(torch.device(DEV))
    done = [0, 0]
    c.tables[0].append(0 + c.P - 1)
    for step in ([50, 17], [39, 39], [1, 1], [1, 1], [1, 1]):
        now = [a + n for a, n in zip(done, step)]
        c.lens = now
        npg = [-(-n // 16) for n in now]
        c.indptr, c.indices = i32([0, npg[0], sum(npg)]), i32(c.tables[0][:npg[0]] + c.tables[1][:npg[1]])
        c.last = i32([n - 16 * (p - 1) for n, p in zip(now, npg)])
        ks = torch.cat([x[a:n] for x, a, n in zip(kn, done, now)]).to(DEV)
        vs = torch.cat([x[a:n] for x, a, n in zip(vn, done, now)]).to(DEV)
        qo = np.concatenate([[0], np.cumsum(step)])
        q = torch.randn(int(qo[-1]), 8, 128, device=DEV).bfloat16()
        if step == [1, 1]:
            out = K().paged_decode_append_q8(q, ks, vs, *c.layer, *c.table, sum(npg), workspace=ws)
        else:
            K().append_kv_q8(ks, vs, i32(qo), int(qo[-1]), *c.layer, *c.table)
            out = K().paged_prefill_q8(q, i32(qo), int(qo[-1]), max(step), *c.layer, *c.table, workspace=ws)
        for b in range(2):
            Q.write_kv(c.side["k"][0], c.side["v"][0], c.tables[b], done[b], kn[b][done[b]:now[b]].double().numpy(), vn[b][done[b]:now[b]].double().numpy())
        c.same()
        for b in range(2):
            check(c, out[qo[b]:qo[b + 1]], q[qo[b]:qo[b + 1]], b, prefill=step != [1, 1])
        done = now


@pytest.mark.parametrize("lens", [[300, 77, 1000], [300, 77, 100]])
def test_side_stream_and_graph_replays(lens):
    """The step captured into a graph and replayed between eager work: every replay gives the eager bits."""
    c = Cache(16, "e4m3", 16, 4, 128, lens, "fp16")
    q = torch.randn(3, 16, 128, device=DEV).half()
    kn, vn = c.rows(3).to(DEV), c.rows(3).to(DEV)
    ws, ws2 = K().Workspace(torch.device(DEV)), K().Workspace(torch.device(DEV))
    want = K().paged_decode_append_q8(q, kn, vn, *c.layer, *c.table, c.total_pages, workspace=ws)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = K().paged_decode_append_q8(q, kn, vn, *c.layer, *c.table, c.total_pages, workspace=ws2)
    side.synchronize()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        static = K().paged_decode_append_q8(q, kn, vn, *c.layer, *c.table, c.total_pages, workspace=ws2)
    for i in range(4):
        static.zero_()
        g.replay()
        assert torch.equal(static, want)
        assert torch.equal(K().paged_decode_q8(q, *c.layer, *c.table, c.total_pages, workspace=ws), want)
        torch.cuda.synchronize()


@pytest.mark.parametrize("longest", [200, 1500])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("page", [16, 20])
def test_attention_at_the_ends_of_the_scales(code, dtype, page, longest):
    """Blocks with scales from under half's range to its largest values (a code may stand for 65536), next to each
    other; and bf16's."""
    c = Cache(17, code, page, 2, 128, [70, 33, longest], dtype)
    top = 65504.0 if dtype == "fp16" else 1e30
    for name in "kv":
        lay, codes, scale = c.side[name]
        # K small enough for finite scores; V anything
        exps = np.array([-40, -33, -26, -24, -20, -10, 0, 5] if name == "v" else [-40, -30, -24, -9])
        s = np.ldexp(1.0, c.g.choice(exps, lay.scale.shape))
        if name == "v":
            big = c.g.random(s.shape) < 0.25
            s = np.where(big, Q.need_scale(top, code), s)
        lay.scale[:] = s
        scale.copy_(torch.from_numpy(s).float())
    if dtype == "fp16":  # the largest half rounds up to 65536 in e4m3 and int8
        for lay, codes, _ in (c.side["v"],):
            x = np.minimum(np.abs(lay.values * lay.scale.repeat(16, 1)[:, :page, :, None]), 65536) / lay.scale.repeat(
                16, 1)[:, :page, :, None] * np.sign(lay.values)
            lay.values[:] = Q.round_code(x, code)
            codes.copy_(torch.from_numpy(lay.values).float().to(CODE[code]))
    B = len(c.lens)
    q = torch.randn(B, 8, 128, device=DEV).to(DT[dtype])
    out = K().paged_decode_q8(q, *c.layer, *c.table, c.total_pages)
    pre = K().paged_prefill_q8(q, i32(range(B + 1)), B, 1, *c.layer, *c.table)
    for b in range(B):
        for o in (out, pre):
            check(c, o[b:b + 1], q[b:b + 1], b, prefill=o is pre)


def test_offsets_past_32_bits():
    """Pages behind the first 2^32 bytes of a pool: what a small pool with the same pages gives, bit for bit."""
    page, hkv, d, lens, new = 16, 8, 128, [50, 7, 200], [20, 1, 3]
    far = 2 ** 32 // (page * hkv * d) + 40
    g = torch.Generator().manual_seed(31)
    npg = [-(-n // page) for n in lens]
    n_pages = sum(npg)
    near = torch.randperm(n_pages, generator=g)
    indptr, last = i32(np.concatenate([[0], np.cumsum(npg)])), i32([n - page * (p - 1) for n, p in zip(lens, npg)])
    codes = torch.randint(-127, 128, (2, n_pages, page, hkv, d), generator=g).to(torch.int8)
    scales = torch.ldexp(torch.ones(2, n_pages, 1, hkv), torch.randint(-8, -3, (2, n_pages, 1, hkv), generator=g))
    total = sum(new)
    x = torch.randn(2, total, hkv, d, generator=g).half().to(DEV)
    q = torch.randn(total, 2 * hkv, d, generator=g).half().to(DEV)
    qo = i32(np.concatenate([[0], np.cumsum(new)]))
    got = []
    for base, size in ((0, n_pages), (far - n_pages, far)):
        ids = near + base
        layer = [torch.zeros(size, page, hkv, d, dtype=torch.int8, device=DEV) for _ in "kv"]
        layer += [torch.zeros(size, 1, hkv, device=DEV) for _ in "kv"]
        for i in range(2):
            layer[i][base:] = codes[i].to(DEV)
            layer[2 + i][base:] = scales[i].to(DEV)
        table = (indptr, i32(ids), last)
        K().append_kv_q8(x[0], x[1], qo, total, *layer, *table)
        outs = [K().paged_prefill_q8(q, qo, total, max(new), *layer, *table),
                K().paged_decode_append_q8(q[:3], x[0, :3], x[1, :3], *layer, *table, n_pages),
                K().paged_decode_q8(q[:3], *layer, *table, n_pages),
                *K().gather_kv_q8(*layer, *table, 210), *(t[base:].clone() for t in layer)]
        if base:
            assert not any(t[:base].any() for t in layer)
        got.append(outs)
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("out", [torch.float16, torch.float32])
def test_gather_of_a_large_output(out):
    """An output past 128 MiB (stored past the caches): the values of the small calls that make it up."""
    c = Cache(32, "e4m3", 16, 8, 128, [700, 16, 0, 33])
    rows = 2 ** 27 // (2 * 4 * 8 * 128 * 2) + 1  # a little more at 2 bytes an element
    k, v = K().gather_kv_q8(*c.layer, *c.table, rows, out)
    small = K().gather_kv_q8(*c.layer, *c.table, 710, out)
    for x, y in zip((k, v), small):
        assert torch.equal(x[:, :710], y) and not x[:, 710:].any()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("grouped", [False, True])
def test_decode_by_a_recorded_layout(code, grouped):
    """A call that records its chunk layout and the calls of other layers that read it: the bits of calls without."""
    c = Cache(33, code, 16, 2, 128, [400, 161, 170, 33], "bf16")
    grp = None
    if grouped:
        for b in (1, 2):
            c.tables[b][:8] = c.tables[0][:8]
        c.indices = i32(sum(c.tables, []))
        grp = K().DecodeGroups(4, [[0, 1, 2]], [8], torch.device(DEV))
    ws = K().Workspace(torch.device(DEV))
    qs = [torch.randn(4, 8, 128, device=DEV).bfloat16() for _ in range(3)]
    want = [K().paged_decode_q8(q, *c.layer, *c.table, c.total_pages, groups=grp) for q in qs]
    K().paged_decode_q8(qs[0], *c.layer, *c.table, c.total_pages, workspace=ws, groups=grp)  # (sizes the workspace)
    for q, w, layout in zip(qs, want, (4242, -4242, -4242)):
        out = K().paged_decode_q8(q, *c.layer, *c.table, c.total_pages, workspace=ws, groups=grp, layout=layout)
        assert torch.equal(out, w)


@pytest.mark.parametrize("grid", [False, True])
def test_prefill_rows_of_no_token(grid):
    """Rows of the output that no token has keep what they held; the padding of a grid becomes 0, as over 16-bit pools."""
    lens, new = [60, 5, 33], [20, 0, 33]
    c = Cache(34, "int8", 16, 2, 64, lens, "fp16")
    T, kw = 64, {}
    rows = [list(range(20)), [], list(range(20, 53))]
    if grid:
        T, rows = 3 * 40, [list(range(3, 23)), [], list(range(80, 113))]
        kw = dict(q_rows=i32(sum(rows, [])), grid_width=40)
    q = torch.randn(T, 8, 64, device=DEV).half()
    out = torch.full_like(q, 7.0)
    K().paged_prefill_q8(q, i32([0, 20, 20, 53]), 53, 33, *c.layer, *c.table, out=out, **kw)
    for b in (0, 2):
        check(c, out[rows[b]], q[rows[b]], b)
    assert (out[sorted(set(range(T)) - set(sum(rows, [])))] == (0 if grid else 7)).all()


@pytest.mark.parametrize("d,page", [(64, 16), (128, 20), (128, 16), (256, 16)])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("at,apart", [(0, 0), (-118, 0), (100, 0), (0, 17), (0, 18), (0, 21), (-30, 60), (40, 100)])
def test_bf16_prefill_over_scales(code, d, page, at, apart):
    """V's scales anywhere in bf16's range, near each other (P.V in half) or with blocks far below the others (in bf16);
    keys in one run and in several, whose ranges differ."""
    lens, new = [700, 33], [70, 33]
    c = Cache(35, code, page, 2, d, lens, "bf16", stale_nan=True)
    lay, codes, scale = c.side["v"]
    rng = np.random.default_rng(36)
    lay.scale *= np.where(rng.random(lay.scale.shape) < 0.3, 2.0 ** (at - apart), 2.0 ** at)
    keep = np.ones(lay.scale.shape, bool)
    keep[c.tables[1]] = rng.random(lay.scale[c.tables[1]].shape) < 0.7  # some blocks of zeros, as written: codes too
    lay.scale[~keep] = 0
    slots = np.repeat(keep, 16, 1)[:, :page, :, None]
    lay.values = np.where(slots, lay.values, 0)
    scale.copy_(torch.from_numpy(lay.scale).float())
    codes.copy_(torch.where(torch.from_numpy(slots).to(DEV), codes.float(), 0).to(codes.dtype))
    qo = [0, 70, 103]
    q = torch.randn(103, 8, d, device=DEV).bfloat16()
    for max_kv in (None, 0, 20000):
        out = K().paged_prefill_q8(q, i32(qo), 103, 70, *c.layer, *c.table, max_kv=max_kv)
        for b in range(2):
            check(c, out[qo[b]:qo[b + 1]], q[qo[b]:qo[b + 1]], b, prefill=True)
