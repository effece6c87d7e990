"""DecodeLaunchQ8 over the layers of one forward, fp16 and bf16 calls of one plan."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("d,hkv,group", [(64, 8, 4), (128, 8, 4), (128, 2, 8), (256, 4, 4)])
@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
def test_a_chunk_layout_is_read_by_calls_of_its_own_row_type(code, d, hkv, group):
    """A call of one row type cuts its chunks for the workgroups that its kernel keeps resident, and records them so. Layers
    of the other type have a record of their own; each layer gives the bits of a call alone."""
    from nanoslg_amd import kernels as K
    page, lens, layers = 16, [4000, 33, 9000, 1600, 12000], 6
    g = torch.Generator(device=DEV).manual_seed(1)
    npg = [-(-n // page) for n in lens]
    P = sum(npg) + 1
    codes = [torch.randint(-60, 61, (layers, P, page, hkv, d), generator=g, device=DEV).to(torch.int8) for _ in "kv"]
    if code is not torch.int8:
        codes = [x.float().to(code) for x in codes]
    scales = [torch.full((layers, P, 1, hkv), 2.0 ** -6, device=DEV) for _ in "kv"]
    indptr, ids = i32(np.concatenate([[0], np.cumsum(npg)])), i32(range(1, P))
    last = i32([n - page * (p - 1) for n, p in zip(lens, npg)])
    slots = i32([page * (1 + sum(npg[:b + 1]) - 1) + (n - 1) % page for b, n in enumerate(lens)])
    launch = K.DecodeLaunchQ8(*codes, *scales, slots, indptr, ids, last, P - 1, hkv * group)
    twin = [[t.clone() for t in (codes[0][i], codes[1][i], scales[0][i], scales[1][i])] for i in range(layers)]
    seen, call = [], launch._f_decode8
    launch._f_decode8 = lambda *a: (seen.append(a[-2]), call(*a))[1]
    types = [torch.float16, torch.bfloat16, torch.bfloat16, torch.float16, torch.float16, torch.bfloat16]
    for i, t in enumerate(types):
        q = torch.randn(len(lens), hkv * group, d, generator=g, device=DEV).to(t)
        kn, vn = (torch.randn(len(lens), hkv, d, generator=g, device=DEV).to(t) for _ in "kv")
        out = launch(i, q, kn, vn)
        want = K.paged_decode_append_q8(q, kn, vn, *twin[i], indptr, ids, last, P - 1)
        assert torch.equal(out, want), i
    tag = {}
    for t, layout in zip(types, seen):
        assert layout > 0 and layout not in tag.values() if t not in tag else layout == -tag[t], seen
        tag.setdefault(t, layout)


@pytest.mark.parametrize("code,d,hkv,group,tokens,one", [
    # (e4m3, up to 8 query heads a KV head: the whole bound)
    ("e4m3", 128, 1, 8, 1024, True), ("e4m3", 128, 1, 8, 1040, False), ("e4m3", 64, 2, 4, 1536, True), ("e4m3", 256, 1, 8, 512, True),
    ("e4m3", 256, 1, 8, 528, False),
    # few KV heads: int8, and more query heads, are slower in one launch from three quarters of it on
    ("int8", 128, 1, 8, 768, True), ("int8", 128, 1, 8, 784, False), ("int8", 128, 4, 4, 896, False), ("int8", 64, 1, 4, 1168, False),
    ("int8", 256, 1, 8, 512, True), ("e4m3", 128, 1, 16, 768, True), ("e4m3", 128, 1, 16, 896, False), ("e4m3", 256, 2, 16, 448, False),
    ("int8", 128, 1, 16, 576, True), ("int8", 128, 2, 16, 640, False), ("int8", 256, 1, 16, 384, True), ("int8", 256, 1, 16, 400, False),
    # more KV heads, whose chunks take two workgroups in the other form
    ("int8", 128, 8, 4, 1024, True), ("e4m3", 128, 8, 16, 1024, True), ("int8", 128, 8, 16, 768, True), ("int8", 128, 8, 16, 896, False),
    ("int8", 256, 8, 16, 512, True),
])
def test_which_calls_take_one_launch(code, d, hkv, group, tokens, one):
    """A call in chunks puts its layout's tag into the workspace, one launch leaves it; both give the longer form's values."""
    from nanoslg_amd import kernels as K
    page = 16
    g = torch.Generator(device=DEV).manual_seed(2)
    P = tokens // page + 1
    t = torch.int8 if code == "int8" else torch.float8_e4m3fn
    k, v = (torch.randint(-9, 10, (P, page, hkv, d), generator=g, device=DEV).float().to(t) for _ in "kv")
    s = torch.full((P, 1, hkv), 2.0 ** -3, device=DEV)
    q = torch.randn(1, hkv * group, d, generator=g, device=DEV).half()
    table = i32([0, P - 1]), i32(range(1, P)), i32([page])
    out = {}
    for pages in (P - 1, 4096):  # (a bound past every sequence: in chunks)
        ws = K.Workspace(torch.device(DEV), 64 << 20)
        out[pages] = K.paged_decode_q8(q, k, v, s, s, *table, pages, workspace=ws, layout=77)
        assert int(ws.buf[:8].view(torch.int64)) == (0 if one and pages == P - 1 else 77)
    # each is within 2^-11 |out| + 2^-10 max |v| of the exact output (as derived for the replayed steps), max |v| = 9 / 8
    torch.testing.assert_close(*out.values(), rtol=2.0 ** -10, atol=2 * 1.125 * (2 ** -10 + 2 ** -13))
