"""8-bit paths that only large calls take: decodes whose K/V stream past the caches, in chunks of more tokens than one window
of page ids and scales; writes of more sequences than a wave has lanes; prefills over runs of keys without a finite score."""
import math

import numpy as np
import pytest
import torch

from oracle import q8_oracle as Q
from test_gpu_q8 import Cache, append

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("code,dtype", [("e4m3", "fp16"), ("int8", "bf16"), ("int8", "fp16"), ("e4m3", "bf16")])
@pytest.mark.parametrize("page,d,hkv,lens", [(16, 64, 256, [17000, 40]), (32, 128, 200, [40, 13001]), (20, 64, 256, [17000, 40]),
                                             (64, 256, 100, [13000])])
def test_decode_in_long_streamed_chunks(code, dtype, page, d, hkv, lens):
    """Many KV heads leave few workgroups for a sequence: chunks of over 1024 tokens, 0.5 to 0.7 GB of K and V. A new row in
    the same call where the page allows it."""
    from nanoslg_amd import kernels as K
    g = torch.Generator(device=DEV).manual_seed(1)
    npg = [-(-n // page) for n in lens]
    P, nb = sum(npg) + 2, -(-page // 16)
    t = torch.int8 if code == "int8" else torch.float8_e4m3fn
    layer = [torch.randint(-60, 61, (P, page, hkv, d), generator=g, device=DEV, dtype=torch.int8) for _ in "kv"]
    if code == "e4m3":
        layer = [torch.cat([a.float().to(t) for a in x.split(128)]) for x in layer]
    layer += [torch.ldexp(torch.ones(P, nb, hkv, device=DEV), torch.randint(-9, -4, (P, nb, hkv), generator=g, device=DEV)) for _ in "kv"]
    ids = torch.randperm(P - 1, generator=torch.Generator().manual_seed(2))[:sum(npg)].numpy() + 1
    at = np.concatenate([[0], np.cumsum(npg)])
    table = i32(at), i32(ids), i32([n - page * (p - 1) for n, p in zip(lens, npg)])
    assert 2 * sum(lens) * hkv * d > 128 << 20
    q = torch.randn(len(lens), 2 * hkv, d, generator=g, device=DEV).to(DT[dtype])
    kn, vn = (torch.randn(len(lens), hkv, d, generator=g, device=DEV).to(DT[dtype]) for _ in "kv")
    out = K.paged_decode_append_q8(q, kn, vn, *layer, *table, sum(npg))
    assert torch.equal(out, K.paged_decode_q8(q, *layer, *table, sum(npg)))
    heads = [0, 1, hkv // 2, hkv - 1]
    for b, n in enumerate(lens):
        tok = np.arange(n)
        pid, slot = torch.from_numpy(ids[at[b] + tok // page]).to(DEV), torch.from_numpy(tok % page).to(DEV)
        k, v = (x[pid, slot][:, heads].double() * s[pid, slot // 16][:, heads, None].double() for x, s in
                ((layer[0].view(torch.int8).view(t), layer[2]), (layer[1].view(torch.int8).view(t), layer[3])))
        cols = [2 * h + i for h in heads for i in range(2)]
        want = Q.attend(q[b:b + 1, cols].double().cpu().numpy(), k.cpu().numpy(), v.cpu().numpy(), None, dtype)
        off = np.abs(out[b:b + 1, cols].double().cpu().numpy() - want[0])
        bound = Q.attention_bound(*want, n, dtype)
        assert (off <= bound).all(), (b, float((off / bound).max()))
        # the new row itself: within the step of its block's last scale
        for x, s, new in ((k, layer[2], kn), (v, layer[3], vn)):
            step = s[pid[-1], slot[-1] // 16][heads].double() * (1 if code == "int8" else 32)
            assert ((x[-1] - new[b, heads].double()).abs() <= step[:, None] / 2).all()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("page,batch", [(16, 65), (16, 130), (20, 65), (5, 130), (48, 200)])
def test_append_of_many_sequences(code, page, batch):
    """More sequences than lanes, some without a new token, some with a block and more of them."""
    g = np.random.default_rng(3)
    lens = [int(n) for n in g.integers(1, 60, batch)]
    new = [int(g.integers(0, min(n, 40) + 1)) * int(g.random() < 0.7) for n in lens]
    new[-1] = lens[-1]
    c = Cache(37, code, page, 2, 64, lens)
    append(c, new, c.rows(sum(new)).to(DEV), c.rows(sum(new), 20).to(DEV))
    c.same()


@pytest.mark.parametrize("max_kv", [0, 20000])  # keys in one run, and in several
@pytest.mark.parametrize("dtype,d", [("fp16", 64), ("bf16", 64), ("bf16", 128), ("fp16", 256)])
@pytest.mark.parametrize("code", ["e4m3", "int8", None])
def test_prefill_over_runs_that_are_not_finite(code, dtype, d, max_kv):
    """Runs of blocks of K that are NaN, whole runs of keys among them, over 8-bit and 16-bit pools: every row sees them."""
    from nanoslg_amd import kernels as K
    hkv, blocks, rows = 2, 100, 16
    n = 16 * blocks
    g = torch.Generator(device=DEV).manual_seed(4)
    k, v = (torch.randint(-60, 61, (blocks + 1, 16, hkv, d), generator=g, device=DEV) for _ in "kv")
    table = i32([0, blocks]), i32(range(1, blocks + 1)), i32([16])
    q = torch.randn(rows, 4 * hkv, d, generator=g, device=DEV).to(DT[dtype])
    if code is None:
        k, v = (k / 64).to(DT[dtype]), (v / 64).to(DT[dtype])
        call = lambda kk, ss: K.paged_prefill(q, i32([0, rows]), rows, rows, kk, v, *table, workspace=K.Workspace(torch.device(DEV)) if max_kv else None)  # noqa: E731
    else:
        t = torch.int8 if code == "int8" else torch.float8_e4m3fn
        k, v = k.float().to(t), v.float().to(t)
        call = lambda kk, ss: K.paged_prefill_q8(q, i32([0, rows]), rows, rows, kk, v, ss, s, *table, max_kv=max_kv)  # noqa: E731
    s = torch.full((blocks + 1, 1, hkv), 2.0 ** -6, device=DEV)
    want = call(k, s)
    assert torch.isfinite(want).all()
    for a, b in [(0, m) for m in range(1, blocks, 9)] + [(m, blocks - 1) for m in range(1, blocks - 1, 9)] + [(24, 48), (40, 41)]:
        kk, ss = k.clone(), s.clone()
        if code == "int8":
            ss[1 + a:1 + b, :, 0] = math.nan
        elif code == "e4m3":
            kk.view(torch.int8)[1 + a:1 + b, :, 0] = 0x7f
        else:
            kk[1 + a:1 + b, :, 0] = math.nan
        out = call(kk, ss)
        assert torch.isnan(out[:, :4]).all(), (a, b)
        assert torch.equal(out[:, 4:], want[:, 4:]), (a, b)
