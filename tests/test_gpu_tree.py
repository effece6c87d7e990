"""Trees of drafted tokens on the GPU against 64-bit oracles: masks and positions, attention (16-bit and fp32 caches,
ragged and grid rows, fused writes, masks of any form, values that are not finite), verification, and the move of
accepted rows; then a whole step captured into a graph and replayed.

Tolerances of the attention, from the arithmetic: with A = sum p |v| / sum p and S = max sum |q_d k_d| scale of a row
(both from the oracle), u the type's half step (2^-11 fp16, 2^-8 bf16, 2^-24 fp32), a result is off by at most
  u |o|                      rounding the output
  2 uP A                     rounding the probabilities (2^-11 fp16; 2^-16 bf16, taken in two terms; none fp32) in the sum
                             and in the normaliser
  2 e A, e = (D + 8) 2^-24 S + 2^-21   the scores' sums in fp32, exp2 and its argument, in both
  (N + 16) 2^-24 A           sums over N keys and joins in fp32
  N 2^-25 max|v| (fp16)      probabilities below fp16's normal range (the largest of a row is at least 1 before
                             normalising)."""
import math
import random

import pytest
import torch

from oracle import tree_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
UP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -16, torch.float32: 0.0}


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def random_tree(rng, n):
    return [-1] + [max(0, j - 1 - int(rng.expovariate(0.3))) for j in range(1, n)] if n else []


def chain(n):
    return list(range(-1, n - 1))


class Setup:
    """A batch of trees behind ctx cached tokens each: pools, tables, rows."""

    def __init__(self, seed, ctx, trees, dtype=torch.float16, Hq=8, Hkv=2, D=128, ps=16, grid=0, offsets=None, layers=None):
        rng = random.Random(seed)
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.ctx, self.trees, self.dtype, self.Hq, self.Hkv, self.D, self.ps = ctx, trees, dtype, Hq, Hkv, D, ps
        self.B = B = len(ctx)
        self.n = [len(t) for t in trees]
        self.lens = [c + n for c, n in zip(ctx, self.n)]
        npg = [-(-x // ps) for x in self.lens]
        self.total_pages = sum(npg)
        P = self.P = self.total_pages + 5
        ids = list(range(1, P))
        rng.shuffle(ids)
        self.table = [ids[sum(npg[:b]):sum(npg[:b + 1])] for b in range(B)]
        shape = ((layers,) if layers else ()) + (P, ps, Hkv, D)
        self.k, self.v = (torch.randn(shape, generator=g, device=DEV).to(dtype) for _ in range(2))
        self.indptr = _i32([sum(npg[:b]) for b in range(B + 1)])
        self.indices = _i32([p for t in self.table for p in t] or [0])
        self.last = _i32([x - (p - 1) * ps if p else 0 for x, p in zip(self.lens, npg)])
        self.qo = _i32([sum(self.n[:b]) for b in range(B + 1)])
        self.T, self.max_q = sum(self.n), max(self.n)
        self.grid = grid
        offsets = offsets or [0] * B
        self.rows = [b * grid + offsets[b] + t for b in range(B) for t in range(self.n[b])] if grid else list(range(self.T))
        self.n_rows = B * grid if grid else self.T
        assert all(r < self.n_rows for r in self.rows) and all(o + n <= grid for o, n in zip(offsets, self.n) if grid)
        self.kw = {"q_rows": _i32(self.rows), "grid_width": grid} if grid else {}
        self.q = torch.randn(self.n_rows, Hq, D, generator=g, device=DEV).to(dtype)
        self.k_new, self.v_new = (torch.randn(self.n_rows, Hkv, D, generator=g, device=DEV).to(dtype) for _ in range(2))
        see = []
        for t in trees:
            m = torch.zeros(len(t), len(t), dtype=torch.bool)
            for j, s in enumerate(O.ancestors(t)):
                m[j, list(s)] = True
            see.append(m)
        self.see = see
        self.mask = O.mask_words(trees, self.max_q).to(DEV)

    def slots(self, b):
        return torch.tensor([self.table[b][i // self.ps] * self.ps + i % self.ps for i in range(self.lens[b])], dtype=torch.long,
                            device=DEV)

    def run(self, fused=True, **kw):
        from nanoslg_amd import kernels
        new = {"k_new": self.k_new, "v_new": self.v_new} if fused else {}
        args = dict(q=self.q, mask=self.mask, qo_indptr=self.qo, total_q=self.T, max_q=self.max_q, k_layer=self.k,
                    v_layer=self.v, kv_indptr=self.indptr, kv_indices=self.indices, kv_last_page_len=self.last,
                    total_pages=self.total_pages)
        return kernels.paged_tree_attention(**{**args, **new, **self.kw, **kw})

    def written(self):
        """The pools with the nodes' rows in."""
        k, v = self.k.clone().view(-1, self.Hkv, self.D), self.v.clone().view(-1, self.Hkv, self.D)
        row = 0
        for b in range(self.B):
            at = self.slots(b)[self.ctx[b]:]
            src = torch.tensor(self.rows[row:row + self.n[b]], dtype=torch.long, device=DEV)
            k[at], v[at] = self.k_new[src], self.v_new[src]
            row += self.n[b]
        return k.view(self.k.shape), v.view(self.v.shape)

    def check(self, out, k, v, scale=None, skip=()):
        """out against the oracle over pools k, v (the nodes' rows in); rows in `skip` are not compared."""
        want = torch.zeros(self.n_rows, self.Hq, self.D, dtype=torch.float64, device=DEV)
        tol = torch.zeros_like(want)
        row = 0
        for b in range(self.B):
            at = self.slots(b)
            src = torch.tensor(self.rows[row:row + self.n[b]], dtype=torch.long, device=DEV)
            kb, vb = k.view(-1, self.Hkv, self.D)[at], v.view(-1, self.Hkv, self.D)[at]
            o, mag, big = O.attention(self.q[src], kb, vb, self.see[b], scale)
            N = self.lens[b]
            e = (self.D + 8) * 2.0 ** -24 * big + 2.0 ** -21
            t = U[self.dtype] * o.abs() + (2 * UP[self.dtype] + 2 * e + (N + 16) * 2.0 ** -24) * mag
            if self.dtype == torch.float16 and N:
                t = t + N * 2.0 ** -25 * vb[vb.isfinite()].abs().max().double()
            want[src], tol[src] = o, t
            row += self.n[b]
        keep = torch.ones(self.n_rows, dtype=torch.bool, device=DEV)
        keep[list(skip)] = False
        err = (out.double() - want).abs()
        bad = (~(err <= tol + 1e-30) & keep[:, None, None]).nonzero()
        assert bad.numel() == 0, (bad[:5].tolist(), err[keep].max().item())


RNG = random.Random(11)
CASES = {
    # name: ctx, trees, dtype, Hq, Hkv, D, ps, grid, offsets
    "one_node_alone": ([0], [[-1]], torch.float16, 8, 2, 128, 16, 0, None),
    "one_node": ([37], [[-1]], torch.bfloat16, 8, 2, 128, 16, 0, None),
    "fresh_trees": ([0, 0, 0], [random_tree(RNG, 5), random_tree(RNG, 33), chain(64)], torch.float16, 8, 2, 128, 16, 0, None),
    "mixed": ([64, 63, 65, 0, 700, 31], [random_tree(RNG, n) for n in (16, 7, 1, 0, 40, 33)], torch.float16, 32, 8, 128, 16, 0, None),
    "grid": ([100, 5, 300, 47], [random_tree(RNG, n) for n in (9, 30, 0, 17)], torch.bfloat16, 8, 2, 128, 16, 37, [3, 0, 5, 20]),
    "group3_page5": ([120, 61], [random_tree(RNG, 21), random_tree(RNG, 45)], torch.float16, 6, 2, 128, 5, 0, None),
    "group16_page1": ([77, 200], [random_tree(RNG, 20), chain(9)], torch.bfloat16, 16, 1, 64, 1, 0, None),
    "heads_alone_d64": ([500, 1000], [random_tree(RNG, 70), random_tree(RNG, 130)], torch.float16, 4, 4, 64, 16, 0, None),
    "d256": ([90, 333], [random_tree(RNG, 33), random_tree(RNG, 64)], torch.float16, 8, 2, 256, 32, 0, None),
    "d256_bf16": ([257, 12], [random_tree(RNG, 100), chain(3)], torch.bfloat16, 4, 2, 256, 16, 101, None),
    "large_tree": ([50], [random_tree(RNG, 300)], torch.float16, 8, 2, 128, 16, 0, None),
    "long": ([9001, 17], [random_tree(RNG, 12), random_tree(RNG, 12)], torch.bfloat16, 4, 1, 128, 16, 0, None),
    "slots_as_pages": ([400, 3], [random_tree(RNG, 20), random_tree(RNG, 20)], torch.float16, 8, 2, 128, 512, 0, None),
    "batch_past_a_wave": ([RNG.randint(0, 90) for _ in range(70)], [random_tree(RNG, RNG.randint(0, 9)) for _ in range(70)],
                          torch.float16, 4, 2, 64, 16, 0, None),
    "fp32": ([100, 0, 640], [random_tree(RNG, n) for n in (20, 33, 5)], torch.float32, 8, 2, 128, 16, 0, None),
    "fp32_grid_d64": ([33, 500], [chain(9), random_tree(RNG, 40)], torch.float32, 6, 2, 64, 20, 43, [1, 2]),
    "fp32_d256": ([170, 29], [random_tree(RNG, 18), random_tree(RNG, 50)], torch.float32, 4, 2, 256, 16, 0, None),
}


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("name", CASES)
def test_attention(name, fused):
    ctx, trees, dtype, Hq, Hkv, D, ps, grid, offsets = CASES[name]
    s = Setup(len(name), ctx, trees, dtype, Hq, Hkv, D, ps, grid, offsets)
    k, v = s.written()
    if not fused:
        s.k, s.v = k.clone(), v.clone()
    out = s.run(fused)
    s.check(out, k, v)
    assert torch.equal(s.k, k) and torch.equal(s.v, v)  # the rows in their slots, nothing else touched
    assert torch.equal(out, s.run(fused))
    if grid:
        pads = torch.ones(s.n_rows, dtype=torch.bool, device=DEV)
        pads[s.rows] = False
        assert not out[pads].any()


@pytest.mark.parametrize("dtype,Hq,Hkv,D,B,most,nodes", [
    (torch.float16, 16, 8, 128, 70, 900, 20), (torch.bfloat16, 16, 8, 128, 130, 500, 9), (torch.float16, 32, 8, 128, 12, 2500, 90),
    (torch.bfloat16, 8, 4, 256, 9, 1500, 150), (torch.float32, 16, 8, 128, 67, 400, 9), (torch.float16, 32, 32, 64, 66, 1200, 8),
    (torch.float16, 16, 4, 64, 3, 6000, 700)])
def test_long_spans(dtype, Hq, Hkv, D, B, most, nodes):
    """Spans of many blocks over several sequences and row tiles, that end where a row tile begins, in its first blocks and in its
    last; batches of more sequences than a wave has lanes."""
    rng = random.Random(B)
    ctx = [rng.choice([0, rng.randint(0, 60), rng.randint(0, most), most]) for _ in range(B)]
    trees = [random_tree(rng, rng.choice([0, 1, rng.randint(1, nodes), nodes])) for _ in range(B)]
    s = Setup(B, ctx, trees, dtype, Hq, Hkv, D)
    k, v = s.written()
    out = s.run()
    s.check(out, k, v)
    assert torch.equal(s.k, k) and torch.equal(s.v, v)
    for pages in (1, 400):  # longer spans
        s.check(s.run(False, total_pages=pages), k, v)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_masks_of_any_form(dtype):
    """Rows that see nothing at all, later nodes, not themselves; masks wider than needed."""
    s = Setup(5, [0, 40, 0], [chain(40), chain(40), [-1]], dtype)
    g = torch.Generator().manual_seed(3)
    s.see = [torch.rand(len(t), len(t), generator=g) < 0.2 for t in s.trees]
    s.see[0][:3] = False
    s.see[2][:] = False
    words = torch.full((s.T, 3), -1, dtype=torch.int64)  # bits past the tree's nodes are set
    row = 0
    for m in s.see:
        for r in m:
            for j, b in enumerate(r.tolist()):
                if not b:
                    words[row, j // 32] &= ~(1 << j % 32)
            row += 1
    s.mask = words.int().to(DEV)
    k, v = s.written()
    out = s.run()
    s.check(out, k, v)
    assert not out[:3].any() and not out[-1].any()


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("dtype,D", [(torch.float16, 128), (torch.bfloat16, 64), (torch.float32, 128), (torch.bfloat16, 256)])
def test_what_is_not_seen_does_not_matter(dtype, D, fused):
    """NaN and infinities in unseen nodes, behind the last token and in unused pages reach no row; the rows that see such
    a node get what the formula gives."""
    trees = [[-1, 0, 0, 1, 2, 3, 4, 4], random_tree(random.Random(4), 40), chain(5)]
    s = Setup(9, [61, 130, 16], trees, dtype, 8, 2, D, 16)
    nan, inf = math.nan, math.inf
    s.k_new[3, 1, 5], s.v_new[2, 0, 7], s.v_new[2, 1, 33], s.v_new[6, 0, 2] = nan, nan, inf, -inf
    s.v_new[8 + 39] = nan  # a last node, of the last key tile
    k, v = s.written()
    for pool in (k, v) if not fused else (s.k, s.v):
        flat = pool.view(-1, s.Hkv, D)
        used = torch.cat([s.slots(b) for b in range(s.B)])
        free = torch.ones(flat.shape[0], dtype=torch.bool, device=DEV)
        free[used] = False
        flat[free] = nan
    if not fused:
        s.k, s.v = k, v
    out = s.run(fused)
    k, v = s.written()
    touched = set()
    for b, row in ((0, 0), (1, 8)):
        for j, seen in enumerate(O.ancestors(trees[b])):
            if seen & ({2, 3, 6} if b == 0 else {39}):
                touched.add(row + j)
    s.check(out, k, v, skip=touched)
    o = out.double().cpu()
    row = {j: set(a) for j, a in enumerate(O.ancestors(trees[0]))}
    for j, seen in row.items():
        for h in range(8):
            if 3 in seen and h >= 4:  # its K of head 1: the whole row
                assert o[j, h].isnan().all()
            else:
                assert bool(o[j, h, 7].isnan()) == (2 in seen and h < 4)
                assert (o[j, h, 33] == inf) == (2 in seen and h >= 4)
                assert (o[j, h, 2] == -inf) == (6 in seen and h < 4)
                assert o[j, h, [0, 1, 3, 4, 5, 6, 8]].isfinite().all()
    assert o[8 + 39].isnan().all()


def test_rows_behind_the_last_tree_stay():
    s = Setup(2, [40, 9], [random_tree(RNG, 6), chain(4)])
    s.q = torch.randn(s.T + 7, 8, 128, device=DEV).half()
    out = torch.full_like(s.q, 7.0)
    s.k, s.v = s.written()
    s.n_rows = s.T
    got = s.run(False, out=out)
    assert got is out and (out[s.T:] == 7).all()
    s.q, full = s.q[:s.T], out
    s.check(full[:s.T], s.k, s.v)


def test_strided_rows_and_scale():
    """q, k_new and v_new as slices of one projection, an output with wide rows, another scale."""
    s = Setup(6, [200, 33], [random_tree(RNG, 30), random_tree(RNG, 11)])
    qkv = torch.randn(s.T, 12, 128, device=DEV).half()
    s.q, s.k_new, s.v_new = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    out = torch.zeros(s.T, 10, 128, device=DEV).half()
    k, v = s.written()
    got = s.run(out=out[:, :8], sm_scale=0.3)
    s.check(got, k, v, scale=0.3)
    assert not out[:, 8:].any() and torch.equal(s.k, k)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("bytes_", [0, 700_000, 3_000_000])
def test_workspaces_of_any_size(dtype, bytes_):
    """Null and small workspaces: fewer chunks, the same rows; the first word is cleared for a recorded decode layout."""
    from nanoslg_amd import _lib, kernels
    s = Setup(8, [2000, 350], [random_tree(RNG, 14), random_tree(RNG, 3)], dtype)
    s.k, s.v = s.written()
    out = torch.empty_like(s.q)
    ws = torch.full((bytes_ + 512,), 77, dtype=torch.uint8, device=DEV)
    base = (ws.data_ptr() + 255) // 256 * 256
    rc = _lib.load().nslg_paged_tree_attention(
        s.q.data_ptr(), 8 * 128, s.mask.data_ptr(), s.mask.shape[1], s.qo.data_ptr(), None, 0, s.T, s.max_q, None, 0, None, 0,
        s.k.data_ptr(), s.v.data_ptr(), s.P, 16, s.indptr.data_ptr(), s.indices.data_ptr(), s.last.data_ptr(), s.total_pages,
        2, 8, 2, 128, 1 / math.sqrt(128), kernels.dtype_code(dtype), out.data_ptr(), 8 * 128, base if bytes_ else None, bytes_,
        torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    s.check(out, s.k, s.v)
    assert (ws[base - ws.data_ptr() + bytes_:] == 77).all()
    if bytes_:
        assert not ws[base - ws.data_ptr():][:8].any()


def test_page_counts_that_are_off_cost_time_only():
    s = Setup(12, [1500, 800], [random_tree(RNG, 10), random_tree(RNG, 25)])
    s.k, s.v = s.written()
    for pages in (1, 10, 100_000):
        s.check(s.run(False, total_pages=pages), s.k, s.v)


def test_offsets_past_32_bits():
    """Pages at both ends of a pool of more than 4 GiB."""
    s = Setup(13, [100, 45], [random_tree(RNG, 20), random_tree(RNG, 9)], Hq=32, Hkv=8)
    P = 150_000
    k, v = s.written()
    where = [P - 1 - p if p % 2 else p for p in range(s.P)]
    big_k, big_v = (torch.empty(P, 16, 8, 128, dtype=torch.float16, device=DEV) for _ in range(2))
    for p in range(s.P):
        big_k[where[p]], big_v[where[p]] = s.k[p], s.v[p]
    out = s.run(k_layer=big_k, v_layer=big_v, kv_indices=_i32([where[p] for p in s.indices.tolist()]))
    s.check(out, k, v)
    for p in range(s.P):
        assert torch.equal(big_k[where[p]], k[p]) and torch.equal(big_v[where[p]], v[p])


@pytest.mark.parametrize("trees,grid", [([chain(1)], 0), ([random_tree(RNG, 26)], 0), ([chain(1024), random_tree(RNG, 1000)], 0),
                                        ([random_tree(RNG, n) for n in (5, 0, 33, 64, 65)], 70),
                                        ([[-1, 0, 5, 2, 9, -7, 4], [-1, -1, 1, 0]], 9)])
def test_plan(trees, grid):
    from nanoslg_amd import kernels
    lens = [len(t) for t in trees]
    B, T, S = len(trees), sum(lens), max(lens)
    start = [10 * b + 3 for b in range(B)]
    off = [2 if grid and n + 2 <= grid else 0 for n in lens]
    rows = [b * grid + off[b] + t for b in range(B) for t in range(lens[b])] if grid else list(range(T))
    kw = {"q_rows": _i32(rows), "grid_width": grid} if grid else {}
    mask, pos = kernels.tree_plan(_i32([p for t in trees for p in t]), _i32([sum(lens[:b]) for b in range(B + 1)]), _i32(start),
                                  T, S, **kw)
    want = [0] * (B * grid if grid else T)
    row = 0
    for b, t in enumerate(trees):
        for d in O.depths(t):
            want[rows[row]] = start[b] + d
            row += 1
    assert torch.equal(mask.cpu(), O.mask_words(trees, S)) and pos.tolist() == want


# ---- verification ----------------------------------------------------------------------


def _rows_like_a_model(g, n, V, dtype, noise=0.7, empty=0.0):
    z = 1.5 * torch.randn(n, V, generator=g)
    z[:, torch.randperm(V, generator=g)[:8]] += 4 + math.log(V)
    q = torch.softmax(z, -1)
    p = torch.softmax(z + noise * torch.randn(n, V, generator=g), -1)
    if empty:  # as after a top-k filter
        p = torch.where(p >= p.quantile(empty, -1, keepdim=True) if V < 100000 else p > 1e-5, p, 0)
    return p.to(dtype), q.to(dtype)


def _verify(trees, tokens, p, q, ua, un, rows=None):
    """The kernel with one workgroup a sequence and with several, against the oracle."""
    from nanoslg_amd import kernels
    for ws in (None, kernels.Workspace(torch.device(DEV))):
        for _ in range(2 if ws else 1):
            got = _verify1(trees, tokens, p, q, ua, un, rows, ws)
        if ws and ws.verify_buf is not None:
            assert not ws.verify_buf[:4 * len(trees)].any()  # the counters, for the next call
    return got


def _verify1(trees, tokens, p, q, ua, un, rows, workspace):
    from nanoslg_amd import kernels
    lens = [len(t) for t in trees]
    B, T, S = len(trees), sum(lens), max(lens)
    dp, dq = p.to(DEV), None if q is None else q.to(DEV)
    path, count, token = kernels.verify_tree(_i32(tokens), _i32([x for t in trees for x in t]),
                                             _i32([sum(lens[:b]) for b in range(B + 1)]), T, S, dp, ua.to(DEV), un.to(DEV),
                                             draft_probs=dq, q_rows=None if rows is None else _i32(rows), workspace=workspace)
    path, count, token = path.tolist(), count.tolist(), token.tolist()
    first = 0
    for b, t in enumerate(trees):
        n = len(t)
        at = list(range(first, first + n)) if rows is None else rows[first:first + n]
        want, nxt = O.verify(t, tokens[first:first + n], p, ua[first:first + n].tolist(), float(un[b]), q, at)
        assert path[b] == want + [-1] * (S - len(want)) and count[b] == len(want) and token[b] == nxt, (b, path[b], want, token[b], nxt)
        first += n
    return path, count, token


def _drafted(g, rng, trees, q, rows, drawn):
    """Tokens of the trees: drawn from q's rows, or their most likely ones; some siblings the same."""
    tokens, first = [], 0
    for t in trees:
        tried = [0] * len(t)
        for j, parent in enumerate(t):
            if parent < 0:
                tokens.append(0)
                continue
            row = q[rows[first + parent]].float()
            k = min(tried[parent], row.numel() - 1)
            tokens.append(int(torch.multinomial(row, 1, generator=g)) if drawn else int(row.topk(k + 1).indices[k]))
            if rng.random() > 0.15:  # else the next sibling repeats it
                tried[parent] += 1
        first += len(t)
    return tokens


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("V,dtype,shape", [(1, torch.float32, "random"), (7, torch.float32, "wide"), (255, torch.bfloat16, "random"),
                                           (256, torch.float32, "wide"), (257, torch.float16, "random"), (1000, torch.float32, "chain"),
                                           (32000, torch.float32, "wide"), (128256, torch.float32, "random"),
                                           (50257, torch.bfloat16, "wide")])
def test_verify(V, dtype, shape, drawn):
    rng, g = random.Random(V), torch.Generator().manual_seed(V + drawn)
    make = {"random": lambda n: random_tree(rng, n), "chain": chain, "wide": lambda n: ([-1] + [(j - 1) // 4 for j in range(1, n)])[:n]}
    trees = [make[shape](n) for n in ((1, 12, 0, 5, 30) if V > 10000 else (1, 12, 0, 5, 30, 64, 65, 130))]
    T = sum(map(len, trees))
    p, q = _rows_like_a_model(g, T, V, dtype, empty=0.5 if V == 1000 else 0.0) if V >= 8 else (
        torch.softmax(torch.randn(T, V, generator=g), -1), torch.softmax(torch.randn(T, V, generator=g), -1))
    rows = list(range(T))
    for round_ in range(3):
        tokens = _drafted(g, rng, trees, q, rows, drawn)
        ua, un = torch.rand(T, generator=g), torch.rand(len(trees), generator=g)
        if round_ == 1:
            ua[:], un[:] = 0.0, 0.0
        if round_ == 2:
            ua[:], un[:] = 1 - 2.0 ** -24, 1 - 2.0 ** -24
        _verify(trees, tokens, p, q if drawn else None, ua, un)


@pytest.mark.parametrize("drawn", [True, False])
def test_verify_odd_rows(drawn):
    """Rows on a grid with strides; rows of zeros, of NaN, with negative and infinite entries; draft rows equal to
    the target's; tokens outside the vocabulary; one token of probability 1."""
    rng, g = random.Random(3), torch.Generator().manual_seed(31)
    V, S = 300, 20
    trees = [random_tree(rng, n) for n in (20, 13, 20, 7)]
    trees[1][5] = -1  # a node of no tree: never reached
    lens = [len(t) for t in trees]
    rows = [b * S + t for b, n in enumerate(lens) for t in range(n)]
    p, q = _rows_like_a_model(g, 4 * S, V, torch.float32)
    wide = torch.zeros(4 * S, V + 13)
    wide[:, :V] = p
    p = wide[:, :V]
    for _ in range(20):
        r = p.clone()
        kind = torch.randint(0, 7, (4 * S,), generator=g)
        r[kind == 0] = 0
        r[kind == 1, 5:9] = math.nan
        r[kind == 2, 100:] = -r[kind == 2, 100:]
        r[kind == 3, 17] = math.inf
        r[kind == 4] = q[kind == 4]
        r[kind == 5] = 0
        r[kind == 5, int(torch.randint(0, V, (1,), generator=g))] = 1.0
        wide[:, :V] = r
        tokens = _drafted(g, rng, trees, q, rows, drawn)
        for k in range(0, len(tokens), 9):
            tokens[k] = rng.choice([-1, V, V + 5, 1 << 30])
        _verify(trees, tokens, p, q if drawn else None, torch.rand(len(rows), generator=g), torch.rand(4, generator=g), rows)


def test_tokens_without_weight_are_rejected_whatever_their_number():
    """Numbers outside [0, 1) (1 from a rounding, say) accept nothing that the target cannot give."""
    p = torch.zeros(6, 5)
    p[:, 0], p[:, 1] = 0.75, 0.25
    for q in (None, torch.full((6, 5), 0.2)):
        for u in (-1.0, 0.0, 1.0, 2.0, float("nan")):
            path, count, token = _verify([[-1, 0, 0, 0, 0, 0]], [0, 2, 9, -1, 0, 1], p, q, torch.tensor([0.0] + [u] * 5), torch.tensor([0.5]))
            assert path[0][:count[0]] in ([0], [0, 4], [0, 5]) and token[0] in (0, 1)


def test_a_workspace_is_not_made_in_a_capture():
    """Its zeros would be written by replays only."""
    from nanoslg_amd import kernels
    V, ws = 40000, kernels.Workspace(torch.device(DEV))
    args = (_i32([0, 1]), _i32([-1, 0]), _i32([0, 2]), 2, 2, torch.full((2, V), 1 / V, device=DEV), torch.zeros(2, device=DEV), torch.zeros(1, device=DEV))
    kernels.verify_tree(*args)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="before"):
            kernels.verify_tree(*args, workspace=ws)
        args[5].add_(0)
    want = kernels.verify_tree(*args)
    assert all(torch.equal(a, b) for a, b in zip(want, kernels.verify_tree(*args, workspace=ws)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = kernels.verify_tree(*args, workspace=ws)
    used = ws.verify_buf.data_ptr()
    ws.get_verify(2 * ws.verify_buf.numel())  # the graph's memory stays its own
    other = torch.zeros(ws.verify_buf.numel() // 4, device=DEV)
    assert used not in (ws.verify_buf.data_ptr(), other.data_ptr())
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held)) and not other.any()


def test_verify_with_one_workspace_for_other_batches():
    """A workspace that a call left is another batch's: its counters are where the sums were not."""
    from nanoslg_amd import kernels
    rng, g = random.Random(0), torch.Generator().manual_seed(0)
    ws = kernels.Workspace(torch.device(DEV))
    for B, V in ((1, 40000), (200, 9000), (256, 12000), (2, 1 << 20), (100, 5000), (1, 9000), (300, 9000)):
        trees = [random_tree(rng, 3) for _ in range(B)]
        p = torch.softmax(2 * torch.randn(3 * B, V, generator=g), -1)
        tokens = [int(p[i].argmax()) for i in range(3 * B)]
        _verify1(trees, tokens, p, None, torch.rand(3 * B, generator=g) * 0.01, torch.rand(B, generator=g), None, ws)


@pytest.mark.parametrize("drawn", [True, False])
def test_verified_tokens_have_the_targets_distribution(drawn):
    """The first token behind the root over 40000 trees of four children: its frequencies are the target's within five
    standard deviations."""
    from nanoslg_amd import kernels
    g = torch.Generator(device=DEV).manual_seed(5)
    V, B, n = 6, 40000, 5
    p = torch.tensor([0.35, 0.05, 0.2, 0.1, 0.25, 0.05], device=DEV)
    q = torch.tensor([0.1, 0.3, 0.1, 0.2, 0.1, 0.2], device=DEV)
    drafted = torch.multinomial(q, B * 4, replacement=True, generator=g).view(B, 4) if drawn else \
        torch.tensor([[1, 4, 0, 3]], device=DEV).expand(B, 4)
    tokens = torch.cat([torch.zeros(B, 1, device=DEV), drafted], 1).int().view(-1).contiguous()
    rows = p.expand(B * n, V).contiguous()
    path, count, token = kernels.verify_tree(tokens, _i32([-1, 0, 0, 0, 0]).repeat(B), torch.arange(0, B * n + 1, n, dtype=torch.int32, device=DEV),
                                             B * n, n, rows, torch.rand(B * n, generator=g, device=DEV), torch.rand(B, generator=g, device=DEV),
                                             draft_probs=q.expand(B * n, V).contiguous() if drawn else None)
    first = torch.where(count > 1, tokens.view(B, n)[torch.arange(B, device=DEV), path[:, 1].clamp(min=0).long()], token)
    freq = torch.bincount(first.long(), minlength=V).double() / B
    assert ((freq - p.double()).abs() <= 5 * (p.double() * (1 - p.double()) / B).sqrt()).all(), freq.tolist()


# ---- the move ----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,Hkv,D,ps", [(torch.float16, 2, 64, 16), (torch.bfloat16, 8, 128, 5), (torch.float32, 1, 64, 1),
                                            (torch.float16, 3, 128, 64), (torch.float16, 1, 5, 16), (torch.float16, 1, 6, 16)])
def test_move(dtype, Hkv, D, ps):
    from nanoslg_amd import kernels
    rng = random.Random(D)
    ns = [1, 30, 0, 64, 17, 40, 9, 20, 33]
    s = Setup(4, [rng.randint(0, 70) for _ in ns], [chain(n) for n in ns], dtype, Hkv, Hkv, D, ps, layers=3)
    paths = [[0], sorted(rng.sample(range(30), 12)), [], list(range(1, 64)), [0, 2, 3, 4, 16], [0], [3, 2, 5], [0, 0, 1], [5, 40]]
    counts = [1, 12, 0, 63, 5, 0, 3, 3, 2]  # the last three: no paths
    k, v = s.k.clone(), s.v.clone()
    for b in (0, 1, 3, 4):
        at = s.slots(b)[s.ctx[b]:].tolist()
        for pool in (k, v):
            O.move(pool.view(3, -1, Hkv, D), at, paths[b])
    W = 64
    path = _i32([p + [-1] * (W - len(p)) for p in paths])
    kernels.move_accepted(s.k, s.v, path, _i32(counts), s.qo, s.indptr, s.indices, s.last)
    assert torch.equal(s.k, k) and torch.equal(s.v, v)


# ---- a whole step --------------------------------------------------------------------------


def test_step_in_a_graph_and_on_a_stream():
    """Plan, attention with its writes, verification and the move, on a stream of its own and captured into a graph that is
    replayed with other inputs in its tensors: every replay equals the eager calls."""
    from nanoslg_amd import kernels
    g = torch.Generator(device=DEV).manual_seed(1)
    s = Setup(21, [600, 90, 0], [random_tree(RNG, n) for n in (24, 17, 9)], layers=1)
    V = 3000
    parents = _i32([p for t in s.trees for p in t])
    start = _i32(s.ctx)
    k_in, v_in = s.k.clone(), s.v.clone()
    tokens = torch.zeros(s.T, dtype=torch.int32, device=DEV)
    target, draft = torch.zeros(s.T, V, device=DEV), torch.zeros(s.T, V, device=DEV)
    ua, un = torch.zeros(s.T, device=DEV), torch.zeros(3, device=DEV)
    ws = kernels.Workspace(torch.device(DEV))

    def fill():
        for x in (s.q, s.k_new, s.v_new):
            x.copy_(torch.randn(x.shape, generator=g, device=DEV))
        z = 3 * torch.randn(s.T, V, generator=g, device=DEV)
        draft.copy_(torch.softmax(z, -1))
        target.copy_(torch.softmax(z + 0.5 * torch.randn(s.T, V, generator=g, device=DEV), -1))
        up = parents.clamp(min=0).long() + torch.repeat_interleave(s.qo[:-1].long(), torch.tensor(s.n, device=DEV))
        tokens.copy_(torch.multinomial(draft[up], 1, generator=g)[:, 0])
        ua.copy_(torch.rand(s.T, generator=g, device=DEV))
        un.copy_(torch.rand(3, generator=g, device=DEV))

    def step():
        s.k.copy_(k_in)
        s.v.copy_(v_in)
        mask, pos = kernels.tree_plan(parents, s.qo, start, s.T, s.max_q)
        out = s.run(k_layer=s.k[0], v_layer=s.v[0], mask=mask, workspace=ws)
        path, count, token = kernels.verify_tree(tokens, parents, s.qo, s.T, s.max_q, target, ua, un, draft_probs=draft, workspace=ws)
        kernels.move_accepted(s.k, s.v, path, count, s.qo, s.indptr, s.indices, s.last)
        return mask, pos, out, path, count, token, s.k, s.v

    fill()
    want = [x.clone() for x in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(4):
        fill()
        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held))


def test_refusals():
    from nanoslg_amd import kernels
    s = Setup(3, [20, 20], [chain(4), chain(6)])
    for err, kw in [(TypeError, {"q": s.q.float()}), (ValueError, {"q": s.q[:5]}), (ValueError, {"mask": s.mask.long()}),
                    (ValueError, {"mask": s.mask[:3]}), (ValueError, {"max_q": 4}), (ValueError, {"max_q": 1025}),
                    (ValueError, {"k_new": None}), (ValueError, {"k_new": s.k_new[:3]}), (TypeError, {"v_new": s.v_new.float()}),
                    (ValueError, {"mask": s.mask.cpu()}), (ValueError, {"q_rows": _i32(list(range(10))), "grid_width": 4}),
                    (ValueError, {"out": s.q[:, :4]}), (ValueError, {"kv_indptr": s.indptr[:2]}), (ValueError, {"q": s.q[:, :, :64]}),
                    (kernels._lib.KernelLibraryError, {"sm_scale": -1.0})]:
        with pytest.raises(err):
            s.run(**kw)
    big = Setup(3, [20], [chain(40)])
    with pytest.raises(kernels._lib.KernelLibraryError, match="masks of 1 words"):
        big.run(mask=big.mask[:, :1].contiguous())
    par, st = _i32(chain(4) + chain(6)), _i32([20, 20])
    p = torch.full((10, 9), 1 / 9, device=DEV)
    u, un = torch.rand(10, device=DEV), torch.rand(2, device=DEV)
    with pytest.raises(ValueError):
        kernels.tree_plan(par[:9], s.qo, st, 10, 6)
    with pytest.raises(ValueError):
        kernels.tree_plan(par, s.qo, st, 10, 6, q_rows=_i32(list(range(10))), grid_width=0)
    ok = dict(tokens=par, parents=par, qo_indptr=s.qo, total_q=10, max_q=6, target_probs=p, u_accept=u, u_next=un)
    for err, kw in [(ValueError, {"target_probs": p[:9]}), (TypeError, {"target_probs": p.double()}), (ValueError, {"u_accept": u[:9]}),
                    (ValueError, {"u_next": un[:1]}), (ValueError, {"u_accept": u.half()}), (ValueError, {"draft_probs": p[:, :8]}),
                    (TypeError, {"draft_probs": p.half()}), (ValueError, {"tokens": par.long()}), (ValueError, {"target_probs": p.t()}),
                    (ValueError, {"parents": par.cpu()})]:
        with pytest.raises(err):
            kernels.verify_tree(**{**ok, **kw})
    pool = torch.zeros(1, s.P, 16, 2, 128, dtype=torch.float16, device=DEV)
    table = (s.indptr, s.indices, s.last)
    path, count = _i32([[0], [0]]), _i32([1, 1])
    with pytest.raises(TypeError):
        kernels.move_accepted(pool.to(torch.int8), pool.to(torch.int8), path, count, s.qo, *table)
    with pytest.raises(ValueError):
        kernels.move_accepted(pool, pool, path[:1], count, s.qo, *table)
    with pytest.raises(ValueError):
        kernels.move_accepted(pool[0], pool[0], path, count, s.qo, *table)
