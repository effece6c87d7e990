"""Speculative decoding over the KV cache as measurable cases: trees of drafted tokens.

A tree has n nodes, each one token: node 0 is the sequence's last sampled token (its root), the others
are drafted. parents[j] < j is node j's parent (-1 for the root); children of a node are tried in the
order of their indices. The trees of a batch are ragged: nodes of sequence b are rows qo[b] .. qo[b + 1] - 1. A model's
inputs and outputs are those rows, or the rows of a padded [batch, width] grid (row map q_rows).

Kinds of case, each one call:

* "plan": the trees' ancestor masks (bit j % 32 of word j / 32 of a node's row: it sees node j) and
  positions (start + depth);
* "attend": attention of the nodes over a paged cache that holds their K/V as the sequences' last
  tokens: each sees every token before its tree, its ancestors and itself;
* "step": the nodes' K/V rows written into the pages, and that attention;
* "verify": the drafted tokens against the target's probabilities, from given uniform numbers (see
  _verify), giving the accepted path, its length and the next token;
* "move": the accepted nodes' K/V moved to the slots behind the sequence's tokens, in every layer.

Shapes are those of this repository's workloads, tests and benchmark, with trees of 2 to 256 nodes.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _case(name=None, kind="attend", dtype="fp16", hq=32, hkv=8, d=128, page=16, batch=1, ctx_lo=0, ctx_hi=0, nodes_lo=16,
          nodes_hi=16, shape="random", grid=False, layers=1, vocab=0, draft=False, lens_seed=0):
    """ctx_lo..ctx_hi: tokens that a sequence has cached (log-uniform); nodes_lo..nodes_hi: nodes of its tree;
    shape: "chain", "wide" (four children a node) or "random"; grid: model rows on a padded grid; draft:
    drafted tokens are drawn from given distributions (else they are the draft's most likely ones)."""
    c = dict(kind=kind, dtype=dtype, hq=hq, hkv=hkv, d=d, page=page, batch=batch, ctx_lo=ctx_lo, ctx_hi=ctx_hi,
             nodes_lo=nodes_lo, nodes_hi=nodes_hi, shape=shape, grid=grid, layers=layers, vocab=vocab, draft=draft,
             lens_seed=lens_seed)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the tables of a loaded server's step, and of the largest one
        _case("plan_b16_n32", "plan", batch=16, ctx_lo=256, ctx_hi=8191, nodes_lo=20, nodes_hi=32, grid=True),
        _case("plan_b256_n256", "plan", batch=256, ctx_lo=256, ctx_hi=8191, nodes_lo=100, nodes_hi=256, shape="wide"),
        # one conversation, a tree of 16: latency
        _case("step_fp16_b1_n16_2k", "step", ctx_lo=2048, ctx_hi=2048),
        # mixed conversations in the default dtype, trees of several sizes on a padded grid
        _case("step_bf16_b8_grid", "step", dtype="bf16", batch=8, ctx_lo=256, ctx_hi=8191, nodes_lo=24, nodes_hi=60, grid=True,
              lens_seed=1),
        # a loaded server with long conversations
        _case("attend_fp16_b32_n32_16k", batch=32, ctx_lo=2048, ctx_hi=16383, nodes_lo=32, nodes_hi=32, lens_seed=2),
        # 256-wide heads in pages of 32, large trees
        _case("attend_bf16_d256_b4_n128", dtype="bf16", hq=16, hkv=4, d=256, page=32, batch=4, ctx_lo=1000, ctx_hi=6000,
              nodes_lo=128, nodes_hi=128, shape="wide", lens_seed=3),
        # an fp32 model's cache, short chains of drafted tokens
        _case("step_fp32_b4_chain", "step", dtype="fp32", batch=4, ctx_lo=700, ctx_hi=3000, nodes_lo=5, nodes_hi=9,
              shape="chain", lens_seed=4),
        # one request's tree of the most likely tokens
        _case("verify_b1_n26", "verify", dtype="fp32", nodes_lo=26, nodes_hi=26, vocab=128256, lens_seed=5),
        # chains drawn by a draft model, a loaded server
        _case("verify_draft_b64_chain", "verify", dtype="fp32", batch=64, nodes_lo=4, nodes_hi=8, shape="chain", vocab=128256,
              draft=True, lens_seed=6),
        # trees drawn by a draft model, probabilities as a model of 16 bits gives them
        _case("verify_draft_bf16_b16_n32", "verify", dtype="bf16", batch=16, nodes_lo=32, nodes_hi=32, shape="wide", vocab=32000,
              draft=True, grid=True, lens_seed=7),
        # the accepted rows of one request in all layers, and of a loaded server
        _case("move_fp16_b1_l32", "move", layers=32, ctx_lo=100, ctx_hi=100, nodes_lo=26, nodes_hi=26, lens_seed=8),
        _case("move_bf16_b64_l16", "move", dtype="bf16", layers=16, batch=64, ctx_lo=1, ctx_hi=120, nodes_lo=16, nodes_hi=48,
              lens_seed=9),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


#: (query heads, KV heads, head dim): mostly the grouped 128-wide heads
_HEADS = [(32, 8, 128)] * 5 + [(64, 8, 128), (8, 8, 128), (16, 1, 128), (32, 8, 64), (16, 4, 256)]


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= 8e8 and w["flops"] <= 1e11 and _state_bytes(c) <= 1.5e9:
            return c


def _draw(rng):
    kind = rng.choice(["step", "step", "step", "attend", "attend", "attend", "verify", "verify", "verify", "move", "plan"])
    hq, hkv, d = rng.choice(_HEADS)
    n = _log_int(rng, 2, 256 if kind == "plan" else 64 if kind == "verify" else 128)
    c = dict(kind=kind, dtype=rng.choice(["fp16", "fp16", "bf16", "bf16", "fp32"]), hq=hq, hkv=hkv, d=d,
             page=rng.choice([16, 16, 16, 8, 20, 32, 64]), nodes_lo=rng.choice([n, max(1, n // 3)]), nodes_hi=n,
             shape=rng.choice(["chain", "wide", "random", "random"]), grid=rng.random() < 0.4, lens_seed=rng.randrange(1 << 20))
    hi = _log_int(rng, 64, 60000)
    c.update(batch=_log_int(rng, 1, 64), ctx_lo=max(1, hi // rng.choice([1, 2, 4, 16])), ctx_hi=hi)
    if kind == "verify":
        c.update(dtype=rng.choice(["fp32", "fp32", "fp16", "bf16"]), vocab=_log_int(rng, 500, 152000), draft=rng.random() < 0.6)
    elif kind == "move":
        c.update(layers=_log_int(rng, 1, 48), ctx_lo=1, ctx_hi=rng.randint(1, 150))
    elif kind == "plan":
        c.update(batch=_log_int(rng, 1, 256))
    return _case(**c)


# ---- sizes and trees -----------------------------------------------------------------


def _lens(case):
    """Per sequence: tokens cached before the tree, the tree's parents."""
    rng = random.Random(case["lens_seed"])
    ctx, trees = [], []
    for _ in range(case["batch"]):
        ctx.append(_log_int(rng, case["ctx_lo"], case["ctx_hi"]) if case["ctx_lo"] else 0)
        n = rng.randint(case["nodes_lo"], case["nodes_hi"])
        if case["shape"] == "chain":
            trees.append([j - 1 for j in range(n)])
        elif case["shape"] == "wide":
            trees.append([-1] + [(j - 1) // 4 for j in range(1, n)])
        else:  # nodes hang mostly on recent ones: several levels, few children each
            trees.append([-1] + [max(0, j - 1 - int(rng.expovariate(0.3))) for j in range(1, n)])
    return ctx, trees


def _depths(parents):
    out = []
    for p in parents:
        out.append(out[p] + 1 if p >= 0 else 0)
    return out


def _state_bytes(case):
    ctx, trees = _lens(case)
    size = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "verify":
        rows = case["batch"] * case["nodes_hi"] if case["grid"] else sum(map(len, trees))
        return rows * case["vocab"] * (8 + 2 * size)
    if case["kind"] == "plan":
        return 0
    return 2.2 * case["layers"] * case["hkv"] * case["d"] * size * sum(c + len(t) + case["page"] for c, t in zip(ctx, trees))


def work(case):
    """plan: parents read, masks and positions written. attend, step: K/V of the tokens seen, new rows read and written, q and
    the outputs; 4 * D flops per query head, node and token seen. verify: the last node's row (and its draft row) and one
    probability a drafted token, an addition an element. move: the accepted rows behind others (a path is about
    one node a level) read and written."""
    ctx, trees = _lens(case)
    size = DTYPES[case["dtype"]].itemsize
    n, B = sum(map(len, trees)), case["batch"]
    depths = [_depths(t) for t in trees]
    if case["kind"] == "plan":
        words = -(-max(map(len, trees)) // 32)
        return {"bytes": 4 * (n + n * words + n + 2 * B), "flops": sum(sum(x) + len(x) for x in depths)}
    if case["kind"] == "verify":
        rows = 2 if case["draft"] else 1
        return {"bytes": B * rows * case["vocab"] * size + n * (8 + rows * size), "flops": B * rows * case["vocab"]}
    row = 2 * case["hkv"] * case["d"] * size
    if case["kind"] == "move":
        moved = sum(max(x) for x in depths)
        return {"bytes": 2 * case["layers"] * moved * row + 4 * n, "flops": 0}
    seen = sum(c * len(t) + sum(x) + len(x) for c, t, x in zip(ctx, trees, depths))
    qo = 2 * case["hq"] * case["d"] * size
    put = n * row if case["kind"] == "step" else 0
    return {"bytes": (sum(ctx) + n) * row + put + n * qo, "flops": 4 * case["hq"] * case["d"] * seen}


# ---- inputs --------------------------------------------------------------------------


def _rand(g, shape, dtype):
    """Unit normal values of `dtype`, made in pieces."""
    out = torch.empty(shape, dtype=dtype, device=DEV)
    flat = out.view(-1)
    for a in range(0, flat.numel(), 1 << 27):
        b = min(flat.numel(), a + (1 << 27))
        flat[a:b] = torch.randn(b - a, generator=g, device=DEV)
    return out


def _padded(trees, width):
    """Parents [B, width], -2 past a tree's nodes."""
    return torch.tensor([t + [-2] * (width - len(t)) for t in trees], device=DEV)


def _see(parents):
    """[B, S, S]: row j sees node i. A node sees what its parent sees, and itself."""
    B, S = parents.shape
    see = torch.eye(S, dtype=torch.bool, device=DEV).repeat(B, 1, 1)
    for j in range(1, S):
        up = parents[:, j].clamp(min=0)
        see[:, j] |= see[torch.arange(B, device=DEV), up] & (parents[:, j] >= 0)[:, None]
    return see


def _words(see, lens, width):
    """The masks of the ragged nodes as int32 words."""
    W = -(-width // 32)
    bits = torch.nn.functional.pad(see, (0, 32 * W - width)).view(see.shape[0], width, W, 32).long()
    words = (bits << torch.arange(32, device=DEV)).sum(-1)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).int()
    return torch.cat([words[b, :n] for b, n in enumerate(lens)])


def prepare(case, seed):
    ctx, trees = _lens(case)
    g = torch.Generator(device=DEV).manual_seed(1_000_003 * seed + 31)
    kind, B, dt = case["kind"], case["batch"], DTYPES[case["dtype"]]
    lens = [len(t) for t in trees]
    width, T = max(lens), sum(lens)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    if kind == "plan":  # (its inputs are the trees themselves)
        ctx = [c + int(x) for c, x in zip(ctx, torch.randint(0, 100, (B,), generator=g, device=DEV).tolist())]
    rows = [b * width + t for b, n in enumerate(lens) for t in range(n)] if case["grid"] else list(range(T))
    s = {"case": case, "parents": i32([p for t in trees for p in t]), "qo": i32([sum(lens[:b]) for b in range(B + 1)]),
         "total": T, "width": width, "lens": lens, "ctx": ctx, "start": i32(ctx), "q_rows": i32(rows), "up": _padded(trees, width),
         # grid row of ragged row t, and of every node of a [B, width] grid its ragged row
         "node": torch.tensor([[sum(lens[:b]) + min(t, n - 1) for t in range(width)] for b, n in enumerate(lens)], device=DEV),
         "real": torch.tensor([[t < n for t in range(width)] for n in lens], device=DEV), "workspace": None}
    if kind == "plan":
        return s
    if kind == "verify":
        return {**s, **_probabilities(case, g, s, trees)}
    ps, hkv, hq, d, L = case["page"], case["hkv"], case["hq"], case["d"], case["layers"]
    held = [a + n for a, n in zip(ctx, lens)]
    npg = [-(-n // ps) for n in held]
    total = sum(npg)
    P = total + total // 9 + 4  # a pool in use to about nine tenths; page 0 is the null page
    shape = (L, P, ps, hkv, d) if kind == "move" else (P, ps, hkv, d)
    table = torch.randperm(P - 1, generator=g, device=DEV)[:total] + 1
    s.update(k=_rand(g, shape, dt), v=_rand(g, shape, dt), indptr=i32([sum(npg[:b]) for b in range(B + 1)]),
             indices=table.int(), last=i32([n - (p - 1) * ps for n, p in zip(held, npg)]), total_pages=total, held=held)
    # slots of every sequence's tokens, [B, longest] (slot 0 past its length)
    pos = torch.arange(max(held), device=DEV)[None]
    inside = pos < torch.tensor(held, device=DEV)[:, None]
    slots = torch.where(inside, table[(s["indptr"][:-1, None] + pos // ps).clamp(max=total - 1).long()] * ps + pos % ps, 0)
    s["slots"] = slots
    s["put"] = torch.cat([slots[b, a:a + n] for b, (a, n) in enumerate(zip(ctx, lens))])
    if kind == "move":
        # accepted paths: from the root down, a child in the order of its index or the end
        coin = torch.rand(T, generator=g, device=DEV).tolist()
        paths = []
        for b, t in enumerate(trees):
            path = [0]
            for j in range(1, len(t)):
                if t[j] == path[-1] and coin[sum(lens[:b]) + j] < 0.6:
                    path.append(j)
            paths.append(path)
        s["path"] = i32([p + [-1] * (width - len(p)) for p in paths])
        s["count"] = i32([len(p) for p in paths])
        s["paths"] = paths
        return s
    see = _see(s["up"])
    s["see"], s["mask"] = see, _words(see, lens, width)
    n_rows = B * width if case["grid"] else T
    s["q"] = _rand(g, (n_rows, hq, d), dt)
    if kind == "step":
        s["k_new"], s["v_new"] = _rand(g, (n_rows, hkv, d), dt), _rand(g, (n_rows, hkv, d), dt)
    return s


def _probabilities(case, g, s, trees):
    """The target's probabilities of every model row, the draft's, and tokens drafted from those: peaked rows,
    the draft's near the target's, so that about two of three drafted tokens are accepted."""
    V, dt, T, B = case["vocab"], DTYPES[case["dtype"]], s["total"], case["batch"]
    n_rows = B * s["width"] if case["grid"] else T
    target, draft = (torch.empty(n_rows, V, dtype=dt, device=DEV) for _ in range(2))
    step = max(1, (1 << 26) // V)
    likely = torch.randperm(V, generator=g, device=DEV)[:8]
    for a in range(0, n_rows, step):
        z = 1.5 * torch.randn(min(step, n_rows - a), V, generator=g, device=DEV)
        z[:, likely] += 4 + math.log(V) - torch.arange(8, device=DEV)
        draft[a:a + step] = torch.softmax(z, -1)
        target[a:a + step] = torch.softmax(z + 0.7 * torch.randn(z.shape, generator=g, device=DEV), -1)
    at = s["q_rows"].tolist()
    most = max(t.count(p) for t in trees for p in t[1:] + [-1])
    tokens = torch.zeros(T, dtype=torch.int32, device=DEV)
    drawn = torch.empty(n_rows, most, dtype=torch.int64, device=DEV)
    for a in range(0, n_rows, step):
        q = draft[a:a + step].float()
        drawn[a:a + step] = torch.multinomial(q, most, replacement=True, generator=g) if case["draft"] else q.topk(most).indices
    drawn, ids, row = drawn.tolist(), tokens.tolist(), 0
    for t in trees:
        tried = [0] * len(t)
        for j, p in enumerate(t):
            if p >= 0:
                ids[row + j] = drawn[at[row + p]][tried[p]]
                tried[p] += 1
        row += len(t)
    return {"target": target, "draft": draft if case["draft"] else None, "tokens": torch.tensor(ids, dtype=torch.int32, device=DEV),
            "u_accept": torch.rand(T, generator=g, device=DEV), "u_next": torch.rand(B, generator=g, device=DEV)}


# ---- one pass: the plain form --------------------------------------------------------


def _plan(s):
    up, real = s["up"], s["real"]
    see = _see(up)
    depth = see.sum(-1) - 1
    positions = torch.where(real, s["start"][:, None] + depth, 0).int()
    if not s["case"]["grid"]:
        positions = positions[real]
    return {"mask": _words(see, s["lens"], s["width"]), "positions": positions.reshape(-1)}


def _attend(s):
    """Grid rows [B, width, Hq, D] in 32 bits over the sequences' tokens, in the inputs' type."""
    case, q = s["case"], s["q"]
    B, S, hq, hkv, d = case["batch"], s["width"], case["hq"], case["hkv"], case["d"]
    at = torch.arange(B * S, device=DEV).view(B, S) if case["grid"] else s["node"]
    x = q[at].float().view(B, S, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(B, hkv, -1, d)
    k = s["k"].view(-1, hkv, d)[s["slots"]].float().permute(0, 2, 3, 1).contiguous()
    x = torch.matmul(x, k).view(B, hkv, hq // hkv, S, -1) * (1 / math.sqrt(d))
    M = x.shape[-1]
    pos, start = torch.arange(M, device=DEV), s["start"].long()
    node = (pos[None] - start[:, None]).clamp(0, S - 1)
    seen = torch.gather(s["see"], 2, node[:, None].expand(B, S, M)) & (pos[None] < start[:, None] + S)[:, None]
    seen |= (pos[None] < start[:, None])[:, None]
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    total = x.sum(-1, keepdim=True)
    v = s["v"].view(-1, hkv, d)[s["slots"]].float().permute(0, 2, 1, 3).contiguous()
    o = torch.matmul(x.view(B, hkv, -1, M), v).view(B, hkv, hq // hkv, S, d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(B, S, hq, d).to(q.dtype)
    if case["grid"]:
        return torch.where(s["real"][..., None, None], o, 0).reshape(B * S, hq, d)
    return o[s["real"]]


def _verify(s):
    """At a node with target probabilities p, its drafted children in the order of their indices. Without draft
    probabilities: child x is accepted if u W < r(x), r = p and W = 1 at first; once rejected, W
    loses r(x) and r(x) becomes 0. With them (q, of which the children were drawn): accepted if u q(x) W < r(x);
    once rejected, r = max(r / W - q, 0) and W is its sum. The accepted child is the next node. Where none is, the
    next token is the first one whose running sum of r exceeds u_next times r's sum."""
    case, B, S = s["case"], s["case"]["batch"], s["width"]
    at = s["q_rows"].long()
    b = torch.arange(B, device=DEV)
    cur = torch.zeros(B, dtype=torch.long, device=DEV)  # node of the tree
    path = torch.full((B, S), -1, dtype=torch.int32, device=DEV)
    path[:, 0] = 0
    count = torch.ones(B, dtype=torch.int32, device=DEV)
    rows = at[s["node"][:, 0]]
    r, W = s["target"][rows].double(), torch.ones(B, dtype=torch.float64, device=DEV)
    q = s["draft"][rows].double() if case["draft"] else None
    for j in range(1, S):
        tried = s["real"][:, j] & (s["up"][:, j] == cur)
        x, u = s["tokens"][s["node"][:, j]].long(), s["u_accept"][s["node"][:, j]].double()
        has = r[b, x]
        ok = tried & (u * W * q[b, x] < has if case["draft"] else u * W < has)
        lost = tried & ~ok
        if case["draft"]:
            new = (r / W[:, None] - q).clamp(min=0)
            W = torch.where(lost, new.sum(-1), W)
            r = torch.where(lost[:, None], new, r)
        else:
            W = torch.where(lost, W - has, W)
            r[b, x] = torch.where(lost, 0.0, has)
        cur = torch.where(ok, j, cur)
        path[b[ok], count[ok].long()] = j
        count += ok.int()
        rows = at[s["node"][b, cur]]
        r = torch.where(ok[:, None], s["target"][rows].double(), r)
        W = torch.where(ok, 1.0, W)
        if case["draft"]:
            q = torch.where(ok[:, None], s["draft"][rows].double(), q)
    total = r.cumsum(-1)
    past = total > (s["u_next"].double() * total[:, -1])[:, None]
    return {"path": path, "count": count, "next": past.int().argmax(-1).int()}


def _move(s):
    case = s["case"]
    b = torch.arange(case["batch"], device=DEV)[:, None]
    i = torch.arange(s["width"], device=DEV)[None]
    keep = i < s["count"][:, None]
    start = s["start"][:, None].long()
    src = s["slots"][b, start + s["path"].long().clamp(min=0)][keep]
    dst = s["slots"][b, start + i * keep][keep]
    for pool in (s["k"], s["v"]):
        flat = pool.view(case["layers"], -1, case["hkv"], case["d"])
        flat[:, dst] = flat[:, src]
    return {"k": s["k"], "v": s["v"]}


def _plain(s):
    kind = s["case"]["kind"]
    if kind in ("plan", "verify", "move"):
        return {"plan": _plan, "verify": _verify, "move": _move}[kind](s)
    if kind == "attend":
        return {"out": _attend(s)}
    at = s["q_rows"].long()
    for pool, new in ((s["k"], s["k_new"]), (s["v"], s["v_new"])):
        pool.view(-1, *pool.shape[2:])[s["put"]] = new[at]
    return {"out": _attend(s), "k": s["k"], "v": s["v"]}


# ---- one pass ------------------------------------------------------------------------


def run(state):
    if not own:
        return _plain(state)
    from nanoslg_amd import kernels

    s, case, kind = state, state["case"], state["case"]["kind"]
    grid = {"q_rows": s["q_rows"], "grid_width": s["width"]} if case["grid"] else {}
    if kind == "plan":
        mask, positions = kernels.tree_plan(s["parents"], s["qo"], s["start"], s["total"], s["width"], **grid)
        return {"mask": mask, "positions": positions}
    if s["workspace"] is None:  # kept by the program, as its caches keep theirs
        s["workspace"] = kernels.Workspace(torch.device(DEV))
    if kind == "verify":
        path, count, token = kernels.verify_tree(s["tokens"], s["parents"], s["qo"], s["total"], s["width"], s["target"],
                                                 s["u_accept"], s["u_next"], draft_probs=s["draft"],
                                                 q_rows=s["q_rows"] if case["grid"] else None, workspace=s["workspace"])
        return {"path": path, "count": count, "next": token}
    table = (s["indptr"], s["indices"], s["last"])
    if kind == "move":
        kernels.move_accepted(s["k"], s["v"], s["path"], s["count"], s["qo"], *table)
        return {"k": s["k"], "v": s["v"]}
    new = {"k_new": s["k_new"], "v_new": s["v_new"]} if kind == "step" else {}
    out = kernels.paged_tree_attention(s["q"], s["mask"], s["qo"], s["total"], s["width"], s["k"], s["v"], *table,
                                       s["total_pages"], workspace=s["workspace"], **grid, **new)
    return {"out": out, "k": s["k"], "v": s["v"]} if kind == "step" else {"out": out}


# ---- the same in 64 bits -------------------------------------------------------------


def _exact_plan(s, trees):
    mask = torch.zeros(s["total"], -(-s["width"] // 32), dtype=torch.int64)
    positions = torch.zeros(s["case"]["batch"] * s["width"] if s["case"]["grid"] else s["total"], dtype=torch.int64)
    at, row = s["q_rows"].tolist(), 0
    for b, t in enumerate(trees):
        for j in range(len(t)):
            a, depth = j, -1
            while a >= 0:
                mask[row + j, a // 32] |= 1 << a % 32
                a, depth = t[a], depth + 1
            positions[at[row + j]] = s["ctx"][b] + depth
        row += len(t)
    mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask)
    return {"mask": mask.int().to(DEV), "positions": positions.int().to(DEV)}


def _exact_verify(s, trees):
    """One sequence after the other; what is left of p after rejections of drawn tokens is max(p - c q, 0) up to a factor,
    with c growing by the sum of that at every rejection."""
    at, first = s["q_rows"].tolist(), 0
    path = torch.full((len(trees), s["width"]), -1, dtype=torch.int32)
    count, token = [], []
    tokens, u = s["tokens"].tolist(), s["u_accept"].tolist()
    for b, t in enumerate(trees):
        node, way, j = 0, [0], 1
        while True:
            p = s["target"][at[first + node]].double()
            q = s["draft"][at[first + node]].double() if s["draft"] is not None else None
            c, W, left, down = 0.0, 1.0, p.clone(), None
            for j in range(node + 1, len(t)):
                if t[j] != node:
                    continue
                x, uj = tokens[first + j], u[first + j]
                if uj * W * (float(q[x]) if q is not None else 1.0) < float(left[x]):
                    down = j
                    break
                if q is None:
                    W -= float(left[x])
                    left[x] = 0
                else:
                    c += W
                    left = (p - c * q).clamp(min=0)
                    W = float(left.sum())
            if down is None:
                break
            node = down
            way.append(node)
        sums = left.cumsum(0)
        token.append(int((sums > float(s["u_next"][b].double()) * sums[-1]).int().argmax()))
        path[b, :len(way)] = torch.tensor(way, dtype=torch.int32)
        count.append(len(way))
        first += len(t)
    as_i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return {"path": path.to(DEV), "count": as_i32(count), "next": as_i32(token)}


def exact(case, seed):
    s = prepare(case, seed)
    _, trees = _lens(case)
    kind, hkv, hq, d, B = case["kind"], case["hkv"], case["hq"], case["d"], case["batch"]
    if kind == "plan":
        return _exact_plan(s, trees)
    if kind == "verify":
        return _exact_verify(s, trees)
    if kind == "move":  # row by row: a path's nodes lie at or behind the slots they go to
        for b, way in enumerate(s["paths"]):
            slots = s["slots"][b, s["ctx"][b]:].tolist()
            for pool in (s["k"], s["v"]):
                flat = pool.view(case["layers"], -1, hkv, d)
                for i, node in enumerate(way):
                    flat[:, slots[i]] = flat[:, slots[node]].clone()
        return {"k": s["k"], "v": s["v"]}
    k, v = s["k"].view(-1, hkv, d), s["v"].view(-1, hkv, d)
    at = s["q_rows"].tolist()
    if kind == "step":
        k[s["put"]] = s["k_new"][s["q_rows"].long()]
        v[s["put"]] = s["v_new"][s["q_rows"].long()]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    first, G = 0, hq // hkv
    for b, t in enumerate(trees):
        m, n, c = s["held"][b], len(t), s["ctx"][b]
        slots = s["slots"][b, :m]
        hidden = torch.ones(n, m, dtype=torch.bool)
        hidden[:, :c] = False
        for j in range(n):
            a = j
            while a >= 0:
                hidden[j, c + a] = False
                a = t[a]
        hidden = hidden.to(DEV).repeat_interleave(G, 0)
        rows = torch.tensor(at[first:first + n], device=DEV)
        for h in range(hkv):
            q = s["q"][rows][:, h * G:(h + 1) * G].double().reshape(n * G, d)
            x = (q @ k[slots, h].double().t().contiguous() / math.sqrt(d)).masked_fill_(hidden, -math.inf)
            o = torch.softmax(x, -1) @ v[slots, h].double()
            out[rows, h * G:(h + 1) * G] = o.view(n, G, d)
        first += n
    return {"out": out, "k": s["k"], "v": s["v"]} if kind == "step" else {"out": out}
