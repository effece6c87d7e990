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
