"""Tree attention where the probabilities' type could show: fp16 and bf16 rows take them in two terms, so that what is left
is the output's rounding and the fp32 sums.

Tolerances as tests/test_gpu_tree.py derives them, with the probabilities' own part smaller. fp16's are taken times 2^7, the
first term cut to 11 bits (less than 2^-10 of the probability is left) and the rest rounded to 11 bits: off by 2^-21 of it;
neither term is below fp16's smallest number, 2^-24, which over 2^7 is 2^-31 each: 2^-30 of the row's largest weight. bf16's
first term is cut to 8 bits, its rest rounded to 8: 2^-16, and 2^-23 more. The normaliser takes them as they are."""
import math
import random

import pytest
import torch

from oracle import tree_oracle as O
from test_gpu_tree import DEV, U, Setup, random_tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,ctx,nodes", [(128, 9, 16), (128, 40, 5), (64, 3, 30), (256, 21, 9)])
def test_probabilities_keep_more_bits_than_the_output(dtype, D, ctx, nodes):
    """Few keys, whose fp32 sums are nearly exact: one rounding of the probabilities to the rows' type would be seen."""
    s = Setup(D + ctx, [ctx, ctx + 1], [random_tree(random.Random(ctx), nodes)] * 2, dtype, 16, 4, D)
    k, v = s.written()
    out = s.run()
    row = 0
    for b in range(2):
        at = s.slots(b)
        src = slice(row, row + s.n[b])
        o, mag, big = O.attention(s.q[src], k.view(-1, 4, D)[at], v.view(-1, 4, D)[at], s.see[b])
        e = (D + 8) * 2.0 ** -24 * big + 2.0 ** -21
        up = 2.0 ** -21 if dtype == torch.float16 else 2.0 ** -16 + 2.0 ** -23
        least = s.lens[b] * 2.0 ** -30 * v.view(-1, 4, D)[at].abs().max().double() if dtype == torch.float16 else 0.0
        tol = U[dtype] * o.abs() + (up + 2 * e + (s.lens[b] + 16) * 2.0 ** -24) * mag + least
        worst = ((out[src].double() - o).abs() / tol).max().item()
        assert worst <= 1
        row += s.n[b]


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N", [20000, 131072])
def test_many_weak_keys_keep_their_weight(dtype, N, workspace):
    """One key of weight 1 and N of the largest weight that fp16 rounds to 0, values 1 throughout: the result is 1. Off by the
    output's rounding, by N 2^-30 and by the sums' roundings, 2^-24 each: N / 32 products of 32 keys, two a product and 64 within
    the products; fp32's products take 4 keys, N roundings in all."""
    s = Setup(1, [N], [[-1]], dtype, 4, 1, 64)
    s.k.zero_(), s.k_new.zero_(), s.v.fill_(1), s.v_new.fill_(1), s.q.zero_()
    s.k.view(-1, 1, 64)[s.slots(0)[7], 0, 0] = 1
    s.q[:, :, 0] = 1
    weak = math.log(2) * (25 + 2.0 ** -6)  # the score's distance
    out = s.run(sm_scale=weak) if workspace else _whole(s, weak)
    tol = U[dtype] + ((N if dtype == torch.float32 else N / 16) + 64) * 2.0 ** -24 + N * 2.0 ** -30
    off = (out.double() - 1).abs().max().item()
    assert off <= tol


def _whole(s, scale):
    """The call without scratch: a workgroup takes all keys of its rows."""
    from nanoslg_amd import _lib, kernels
    out = torch.empty_like(s.q)
    Hq, D = s.q.shape[1:]
    new = [None if x is None else x.data_ptr() for x in (s.k_new, s.v_new)]
    rc = _lib.load().nslg_paged_tree_attention(
        s.q.data_ptr(), Hq * D, s.mask.data_ptr(), s.mask.shape[1], s.qo.data_ptr(), None, 0, s.T, s.max_q, new[0],
        s.Hkv * D, new[1], s.Hkv * D, s.k.data_ptr(), s.v.data_ptr(), s.P, s.ps, s.indptr.data_ptr(),
        s.indices.data_ptr(), s.last.data_ptr(), s.total_pages, s.B, Hq, s.Hkv, D, scale, kernels.dtype_code(s.dtype),
        out.data_ptr(), Hq * D, None, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    return out
