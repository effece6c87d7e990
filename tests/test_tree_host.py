"""Trees of drafted tokens without a GPU: the oracle against small cases worked by hand and against each other's forms, the C
entry points' refusals, their bindings."""
import random
import re
from pathlib import Path

import pytest
import torch

from oracle import tree_oracle as O

ROOT = Path(__file__).resolve().parent.parent


def test_ancestors_and_masks():
    t = [-1, 0, 0, 1, 3, 2]
    assert O.ancestors(t) == [{0}, {0, 1}, {0, 2}, {0, 1, 3}, {0, 1, 3, 4}, {0, 2, 5}]
    assert O.depths(t) == [0, 1, 1, 2, 3, 2]
    assert O.mask_words([t], 6)[:, 0].tolist() == [1, 3, 5, 11, 27, 37]
    assert O.depths([-1, 0, 7, 2, 3]) == [0, 1, 0, 1, 2]  # a parent behind its child is none
    words = O.mask_words([list(range(-1, 39))], 40)
    assert words.shape == (40, 2) and words[31].tolist() == [-1, 0] and words[39].tolist() == [-1, 255]


def test_attention_is_the_softmax_over_what_is_seen():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, h, 8, generator=g) for n, h in ((3, 4), (10, 2), (10, 2)))
    see = torch.tensor([[1, 0, 0], [1, 1, 0], [1, 0, 1]]).bool()
    v[8] = float("nan")  # node 1: seen by itself only
    out, _, _ = O.attention(q, k, v, see)
    assert out[1].isnan().all() and out[[0, 2]].isfinite().all()
    x = (q[2, 3].double() @ k[[0, 1, 2, 3, 4, 5, 6, 7, 9], 1].double().T) / 8 ** 0.5
    assert torch.allclose(out[2, 3], torch.softmax(x, -1) @ v[[0, 1, 2, 3, 4, 5, 6, 7, 9], 1].double())


def test_verification_by_hand():
    p = torch.tensor([[0.5, 0.3, 0.2], [0.1, 0.1, 0.8], [0.2, 0.2, 0.6]], dtype=torch.float64)
    tree, tokens = [-1, 0, 0], [0, 1, 0]
    # token 1 accepted
    assert O.verify(tree, tokens, p, [0, 0.29, 0], 0.15, None) == ([0, 1], 1)
    # rejected, then token 0 with 0.5 / 0.7
    assert O.verify(tree, tokens, p, [0, 0.31, 0.71], 0.9, None) == ([0, 2], 2)
    # both rejected: token 2 is left
    assert O.verify(tree, tokens, p, [0, 0.31, 0.72], 0.0, None) == ([0], 2)
    # drawn from q: accepted with p / q, else from max(p - q, 0)
    q = torch.tensor([[0.2, 0.6, 0.2]] * 3, dtype=torch.float64)
    assert O.verify([-1, 0], [0, 1], p, [0, 0.49], 0.5, q) == ([0, 1], 2)
    assert O.verify([-1, 0], [0, 1], p, [0, 0.51], 0.99, q) == ([0], 0)


@pytest.mark.parametrize("drawn", [True, False])
def test_verification_leaves_the_targets_distribution(drawn):
    """The probability of every first token, summed over the drafts and integrated over the numbers, is p's."""
    p = torch.tensor([0.5, 0.2, 0.3], dtype=torch.float64)
    q = torch.tensor([0.2, 0.5, 0.3], dtype=torch.float64)
    rng = random.Random(0)
    hits, n = [0] * 3, 20000
    rows = p.expand(4, 3)
    for _ in range(n):
        tokens = [0] + (rng.choices(range(3), q.tolist(), k=3) if drawn else [1, 0, 1])
        path, nxt = O.verify([-1, 0, 0, 0], tokens, rows, [rng.random() for _ in range(4)], rng.random(), q.expand(4, 3) if drawn else None)
        hits[tokens[path[1]] if len(path) > 1 else nxt] += 1
    for h, x in zip(hits, p.tolist()):
        assert abs(h / n - x) < 5 * (x * (1 - x) / n) ** 0.5


A = 4096  # an address that no check follows


def test_plan_refusals():
    from nanoslg_amd import _lib
    lib, fast = _lib.load(), _lib.fast_tree()

    def plan(parents=A, qo=A, start=A, rows=None, width=0, total=10, max_q=6, batch=2, mask=A, words=1, pos=A):
        args = (parents, qo, start, rows, width, total, max_q, batch, mask, words, pos, None)
        rc = lib.nslg_tree_plan(*args)
        assert fast.tree_plan(*args) == rc
        return rc

    assert plan(batch=0, total=0) == 0 and plan(total=0) == 0
    for kw in ({"total": -1}, {"batch": -1}, {"max_q": 4}, {"parents": None}, {"start": None}, {"mask": None}, {"pos": None},
               {"words": 0}, {"max_q": 40}, {"rows": A}, {"rows": A, "width": 4}, {"rows": A, "width": 1 << 30}):
        assert plan(**kw) == -1, kw
        assert "tree_plan" in _lib.last_error()
    assert plan(max_q=1025, words=99) == -2


def test_attention_refusals():
    from nanoslg_amd import _lib
    lib, fast = _lib.load(), _lib.fast_tree()
    ok = dict(q=A, qs=4096, mask=A, words=1, qo=A, rows=None, width=0, total=10, max_q=6, kn=None, kns=0, vn=None, vns=0, k=A, v=A, P=100,
              ps=16, ip=A, ix=A, last=A, pages=9, batch=2, hq=32, hkv=8, d=128, scale=0.1, dtype=0, out=A, os=4096, ws=None, wsb=0)

    def call(**kw):
        args = (*{**ok, **kw}.values(), None)
        rc = lib.nslg_paged_tree_attention(*args)
        assert fast.paged_tree_attention(*args) == rc
        if rc:
            assert "paged_tree_attention" in _lib.last_error()
        return rc

    assert call(batch=0, total=0) == 0 and call(total=0, max_q=0) == 0
    new = dict(kn=A, kns=1024, vn=A, vns=1024)
    for kw in ({"dtype": 7}, {"batch": -1}, {"hq": 30}, {"hkv": 0}, {"ps": 0}, {"P": 0}, {"total": -1}, {"max_q": 4}, {"max_q": 0},
               {"words": 0}, {"max_q": 33}, {"scale": 0.0}, {"scale": float("inf")}, {"scale": float("nan")}, {"mask": None}, {"q": None},
               {"k": None}, {"ip": None}, {"out": None}, {"qs": 4095}, {"qs": 4100}, {"os": 100}, {"q": A + 8}, {"mask": A + 2},
               {"kn": A, "kns": 1024}, {**new, "kns": 1000}, {**new, "vn": A + 8}, {**new, "vns": 1028}, {"rows": A},
               {"rows": A, "width": 4}, {"pages": -1}):
        assert call(**kw) == -1, kw
    for kw in ({"d": 96, "qs": 8192, "os": 8192}, {"hkv": 1}, {"max_q": 1025, "words": 99}, {"P": 1 << 28}):
        assert call(**kw) == -2, kw


def test_workspace_sizes():
    from nanoslg_amd import _lib
    size = _lib.load().nslg_paged_tree_workspace_size
    assert 0 < size(1, 32, 8, 128, 12, 16, 16, 0) < size(1, 32, 8, 128, 4096, 16, 16, 0)
    assert _lib.load().nslg_verify_tree_workspace_size(1, 4000) == 0 < _lib.load().nslg_verify_tree_workspace_size(1, 5000)
    assert size(64, 32, 8, 128, 100_000, 16, 64, 0) < 1 << 29
    for bad in ((0, 32, 8, 128, 9, 16, 16, 0), (1, 32, 8, 96, 9, 16, 16, 0), (1, 32, 8, 128, 9, 16, 2000, 0), (1, 30, 8, 128, 9, 16, 9, 0),
                (1, 32, 8, 128, 9, 16, 9, 5)):
        assert size(*bad) == 0


def test_verify_refusals():
    from nanoslg_amd import _lib
    lib, fast = _lib.load(), _lib.fast_tree()
    ok = dict(tokens=A, parents=A, qo=A, rows=None, total=10, max_q=6, batch=2, p=A, ps=100, q=None, qs=0, n=10, vocab=100, dtype=2, ua=A,
              un=A, path=A, count=A, next=A, ws=None, wsb=0)

    def call(**kw):
        args = (*{**ok, **kw}.values(), None)
        rc = lib.nslg_verify_tree(*args)
        assert fast.verify_tree(*args) == rc
        if rc:
            assert "verify_tree" in _lib.last_error()
        return rc

    assert call(batch=0, total=0) == 0
    for kw in ({"dtype": 9}, {"batch": -1}, {"total": 13}, {"vocab": 0}, {"n": 9}, {"ps": 99}, {"q": A, "qs": 99}, {"p": A + 2}, {"tokens": None},
               {"parents": None}, {"p": None}, {"ua": None}, {"un": None}, {"path": None}, {"count": None}, {"next": None}, {"n": -1}):
        assert call(**kw) == -1, kw
    assert call(max_q=1025) == -2 and call(vocab=(1 << 20) + 1, ps=1 << 21) == -2


def test_move_refusals():
    from nanoslg_amd import _lib
    lib, fast = _lib.load(), _lib.fast_tree()
    ok = dict(k=A, v=A, L=2, P=100, ps=16, hkv=8, d=128, dtype=0, path=A, stride=6, count=A, qo=A, ip=A, ix=A, last=A, batch=2)

    def call(**kw):
        args = (*{**ok, **kw}.values(), None)
        rc = lib.nslg_move_accepted(*args)
        assert fast.move_accepted(*args) == rc
        if rc:
            assert "move_accepted" in _lib.last_error()
        return rc

    assert call(batch=0) == 0 and call(stride=0) == 0
    for kw in ({"dtype": 9}, {"L": 0}, {"P": 0}, {"ps": 0}, {"hkv": 0}, {"d": 0}, {"batch": -1}, {"stride": -1}, {"k": None}, {"path": None},
               {"count": None}, {"qo": None}, {"last": None}):
        assert call(**kw) == -1, kw
    assert call(batch=70000) == -2 and call(P=1 << 28) == -2


def test_fast_binding_signatures_match_the_header():
    from ctypes import c_float, c_int32, c_int64, c_size_t, c_void_p
    from nanoslg_amd import _lib
    code = {c_void_p: "p", c_int64: "q", c_int32: "i", c_size_t: "z", c_float: "f"}
    found = re.findall(r'parse\("(\w+)", "(\w+)"', (ROOT / "nanoslg_amd" / "csrc" / "fastcall_tree.c").read_text())
    assert [fn for fn, _ in found] == ["tree_plan", "paged_tree_attention", "verify_tree", "move_accepted"]
    for fn, sig in found:
        assert sig == "".join(code[t] for t in _lib.SIGNATURES["nslg_" + fn][1]), fn


def test_wrappers_need_device_tensors():
    from nanoslg_amd import kernels
    t = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensors"):
        kernels.tree_plan(t, t, t, 4, 4)
