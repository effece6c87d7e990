"""Prefill of bf16 rows over an 8-bit cache where the keys that matter have small weights: a first token that draws nearly
all of the weight and has no V (an attention sink), and values of very different size."""
import math

import numpy as np
import pytest
import torch

from oracle import q8_oracle as Q

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HKV, G, PAGE = 2, 2, 16


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def layer(code, d, n, v_rows, v_scale):
    """Key 0 is (1, 0, 0, ..), the others 0: a query (x, 0, ..) scores x ln 2 on key 0 and 0 elsewhere. V: v_rows * v_scale."""
    pages = -(-n // PAGE)
    kv = [np.zeros((pages + 1, PAGE, HKV, d)) for _ in "kv"]
    scale = [np.ones((pages + 1, 1, HKV)) for _ in "kv"]
    kv[0][1, 0, :, 0] = 1
    v = np.zeros((pages * PAGE, HKV, d))
    v[:n] = v_rows
    kv[1][1:] = v.reshape(pages, PAGE, HKV, d)
    scale[1][1:, 0] = np.asarray(v_scale)[:, None]
    twins = [Q.Layer(a, s, code) for a, s in zip(kv, scale)]
    t = torch.float8_e4m3fn if code == "e4m3" else torch.int8
    codes = [torch.from_numpy(a).float().to(DEV).to(t) for a in kv]
    return twins, (*codes, *(torch.from_numpy(s).float().to(DEV) for s in scale))


def prefill(twins, pools, n, rows, xs, max_kv, by):
    """The last `rows` tokens' queries, x dealt out over rows and heads; against the oracle by the bound `by`."""
    from nanoslg_amd import kernels as K
    d, pages = pools[0].shape[3], -(-n // PAGE)
    q = np.zeros((rows, HKV * G, d))
    q[:, :, 0] = np.resize(xs, rows * HKV * G).reshape(rows, HKV * G)
    qt = torch.from_numpy(q).to(DEV).bfloat16()
    assert (qt.double().cpu().numpy() == q).all()
    out = K.paged_prefill_q8(qt, i32([0, rows]), rows, rows, *pools, i32([0, pages]), i32(range(1, pages + 1)),
                             i32([n - PAGE * (pages - 1)]), sm_scale=math.log(2.0), max_kv=max_kv)
    k, v = (t.read(range(1, pages + 1), n) for t in twins)
    want = Q.attend(q, k, v, math.log(2.0), by)
    bound = Q.attention_bound(*want, n, by)
    off = np.abs(out.double().cpu().numpy() - want[0])
    assert (off <= bound).all(), (float((off / bound).max()), np.argwhere(off > bound)[:5])
    return want[0]


@pytest.mark.parametrize("max_kv", [0, 20000])  # keys in one run, and in several
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_small_weights_beside_a_sink(code, d, max_kv):
    """Weights of 2^-2.5 to 2^-40.5 of the row's largest, equal over the keys (so that their roundings add up)."""
    n, rows = 1500, 40
    g = np.random.default_rng(1)
    v = g.integers(1, 8, (1, HKV, d)) * 8.0 + np.zeros((n, 1, 1))
    v[0] = 0
    twins, pools = layer(code, d, n, v, np.full(-(-n // PAGE), 0.125))
    want = prefill(twins, pools, n, rows, np.arange(2, 41) + 0.5, max_kv, "bf16up")
    assert (np.abs(want) > 0).all()


@pytest.mark.parametrize("apart", [6, 8, 9, 13, 18, 20])
@pytest.mark.parametrize("max_kv", [0, 20000])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_small_weights_on_large_values(code, d, max_kv, apart):
    """The sink has a V of ordinary size; the keys of small weight have one 2^apart times as large. Past 2^8 what they
    give counts to the last bit of a bf16 pair."""
    n, rows = 1500, 40
    g = np.random.default_rng(2)
    v = g.integers(1, 8, (1, HKV, d)) * 8.0 + np.zeros((n, 1, 1))
    scale = np.full(-(-n // PAGE), 2.0 ** apart)
    scale[0] = 1.0
    twins, pools = layer(code, d, n, v, scale)
    # (in several runs, those behind the sink's have one scale and equal weights)
    by = "bf16up" if apart <= 8 else "bf16runs" if max_kv else "bf16"
    prefill(twins, pools, n, rows, np.arange(2, 41) + 0.5, max_kv, by)


@pytest.mark.parametrize("max_kv", [0, 20000])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_equal_weights_on_values_near_bf16s_end(code, max_kv):
    """1500 keys of V up to 2^110.8: their sum, 2^121.4, is in fp32's range with room for the maximum's lag only."""
    n, rows = 1500, 40
    g = np.random.default_rng(3)
    v = g.integers(1, 8, (1, HKV, 128)) * 8.0 + np.zeros((n, 1, 1))
    twins, pools = layer(code, 128, n, v, np.full(-(-n // PAGE), 2.0 ** 105))
    prefill(twins, pools, n, rows, np.zeros(1), max_kv, "bf16up")
