"""The 8-bit KV cache as measurable cases: writing it, reading it back, attention over it.

A cache layer in 8 bits is four tensors: codes k and v [P, page, Hkv, D] (float8_e4m3fn or
int8) and scales k_scale and v_scale [P, nb, Hkv] (float32, nb = ceil(page / 16)): one scale
for each block of 16 slots of a page and KV head. A stored value is code * scale. Scales
are powers of two (or 0), so dividing by one is exact.

Writing a sequence's next tokens, block by block and head by head: `need` is the smallest
power of two with amax(|new rows|) <= M * need, M = 448 (e4m3) or 127 (int8). A block
written from its first slot takes that scale; one that holds earlier tokens takes the larger of
its own and `need`, and its earlier tokens' codes are rounded to the new scale where it
grew. New codes are row / scale, rounded to nearest, ties to even.

Kinds of case, each one call (or two, where rows are written and read back) of one layer:

* "step": a decode step: every sequence's new row written, and one query row a sequence
  attended over all of its tokens; the e4m3 pools come back as they are, with their scales;
* "decode": that attention alone, for a program that wrote the rows before;
* "prefill": causal attention of a forward's new tokens (already written) over their
  sequences, ragged, or on the padded [batch, width] grid of a left-padded batch;
* "append": a forward's rows written. e4m3 pools come back as in "step"; int8 ones are read back
  (the values that the codes stand for);
* "read": the cached sequences as contiguous 16-bit rows.

Shapes are those of this repository's workloads, tests and benchmark.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
MOST = {"e4m3": 448.0, "int8": 127.0}
BLOCK = 16


def _case(name=None, kind="decode", dtype="fp16", code="e4m3", hq=32, hkv=8, d=128, page=16, batch=1, ctx_lo=0, ctx_hi=0,
          new_lo=0, new_hi=0, grid=False, lens_seed=0):
    """ctx_lo..ctx_hi: tokens that a sequence has cached (log-uniform); new_lo..new_hi: its new
    tokens; grid: rows on a left-padded grid instead of ragged ones."""
    c = dict(kind=kind, dtype=dtype, code=code, hq=hq, hkv=hkv, d=d, page=page, batch=batch, ctx_lo=ctx_lo, ctx_hi=ctx_hi,
             new_lo=new_lo, new_hi=new_hi, grid=grid, lens_seed=lens_seed)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # a lightly loaded server, one token for each of 4 conversations of 1k to 4k tokens: latency
        _case("step_e4m3_fp16_b4", "step", batch=4, ctx_lo=1024, ctx_hi=4095, new_lo=1, new_hi=1),
        # mixed conversations in the default dtype
        _case("step_e4m3_bf16_b16", "step", dtype="bf16", batch=16, ctx_lo=256, ctx_hi=8191, new_lo=1, new_hi=1, lens_seed=1),
        # a loaded server under KV pressure: 64 conversations of 2k to 32k tokens
        _case("decode_e4m3_fp16_b64_32k", batch=64, ctx_lo=2048, ctx_hi=32767),
        # one very long conversation
        _case("decode_int8_bf16_b1_128k", dtype="bf16", code="int8", ctx_lo=131071, ctx_hi=131071),
        # 256-wide heads in pages of 32
        _case("decode_int8_fp16_d256_b16", code="int8", hq=16, hkv=4, d=256, page=32, batch=16, ctx_lo=700, ctx_hi=6000,
              lens_seed=2),
        # a batch of 4096-token prompts, its last 512-token chunk
        _case("prefill_e4m3_fp16_8x512", "prefill", batch=8, ctx_lo=3584, ctx_hi=3584, new_lo=512, new_hi=512),
        # one long request's next chunk, in the default dtype
        _case("prefill_e4m3_bf16_b1_over_6k", "prefill", dtype="bf16", ctx_lo=6007, ctx_hi=6007, new_lo=512, new_hi=512),
        # the suffixes of requests on one system prompt: ragged, left-padded rows
        _case("prefill_int8_fp16_grid_b16", "prefill", code="int8", batch=16, ctx_lo=2040, ctx_hi=2040, new_lo=128, new_hi=1024,
              grid=True, lens_seed=3),
        # a chunk of each of 8 prompts written behind what is cached, from inside a block on
        _case("append_e4m3_fp16_8x512", "append", batch=8, ctx_lo=900, ctx_hi=1100, new_lo=512, new_hi=512, lens_seed=4),
        # a padded batch of fresh prompts of a model with 64-wide heads, written and read back
        _case("append_int8_bf16_d64_b4", "append", dtype="bf16", code="int8", d=64, batch=4, new_lo=250, new_hi=2000,
              grid=True, lens_seed=5),
        # a short conversation handed out in 16 bits
        _case("read_e4m3_bf16_b1", "read", dtype="bf16", ctx_lo=777, ctx_hi=777),
        # a batch of long ones
        _case("read_int8_fp16_b16_16k", "read", code="int8", batch=16, ctx_lo=2048, ctx_hi=16000, lens_seed=6),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


#: (query heads, KV heads, head dim): mostly the grouped 128-wide heads
_HEADS = [(32, 8, 128)] * 5 + [(64, 8, 128), (8, 8, 128), (16, 1, 128), (32, 8, 64), (16, 4, 256)]


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= 1.3e9 and w["flops"] <= 2e11:
            return c


def _draw(rng):
    kind = rng.choice(["step", "step", "decode", "decode", "prefill", "prefill", "append", "read"])
    hq, hkv, d = rng.choice(_HEADS)
    c = dict(kind=kind, dtype=rng.choice(["fp16", "bf16"]), code=rng.choice(["e4m3", "int8"]), hq=hq, hkv=hkv, d=d,
             page=rng.choice([16, 16, 16, 8, 20, 32, 64]), lens_seed=rng.randrange(1 << 20))
    if kind in ("step", "decode"):
        hi = _log_int(rng, 64, 60000)
        c.update(batch=_log_int(rng, 1, 64), ctx_lo=max(1, hi // rng.choice([1, 2, 4, 16])), ctx_hi=hi)
        if kind == "step":
            c.update(new_lo=1, new_hi=1, code="e4m3")
    elif kind == "prefill":
        n, hi = _log_int(rng, 16, 1024), _log_int(rng, 64, 16000)
        c.update(batch=_log_int(rng, 1, 16), ctx_lo=max(1, hi // rng.choice([1, 3])), ctx_hi=hi,
                 new_lo=rng.choice([n, max(1, n // 3)]), new_hi=n, grid=rng.random() < 0.4)
    elif kind == "append":
        n = _log_int(rng, 1, 2048)
        hi = _log_int(rng, 1, 400 if c["code"] == "int8" else 4000)
        c.update(batch=_log_int(rng, 1, 16), ctx_lo=max(1, hi // 3), ctx_hi=hi, new_lo=rng.choice([n, max(1, n // 3)]), new_hi=n,
                 grid=rng.random() < 0.4)
    else:
        hi = _log_int(rng, 24, 16000)
        c.update(batch=_log_int(rng, 1, 16), ctx_lo=max(1, hi // 3), ctx_hi=hi)
    return _case(**c)


# ---- sizes ---------------------------------------------------------------------------


def _lens(case):
    """Per sequence: tokens cached before the new ones, new tokens."""
    rng = random.Random(case["lens_seed"])
    ctx, new = [], []
    for _ in range(case["batch"]):
        ctx.append(_log_int(rng, case["ctx_lo"], case["ctx_hi"]) if case["ctx_lo"] else 0)
        new.append(rng.randint(case["new_lo"], case["new_hi"]) if case["new_lo"] else 0)
    return ctx, new


def work(case):
    """Codes (1 byte) and scales (4 a block) of the tokens attended or read, the new rows read and written,
    q and the 16-bit outputs; 4 * D flops per query head and visible key."""
    ctx, new = _lens(case)
    rows = 2 * case["hkv"] * case["d"]  # elements of a token's K and V
    held = sum(a + n for a, n in zip(ctx, new)) * (rows + 2 * case["hkv"] * 4 / BLOCK)
    put = sum(new) * (3 * rows + 2 * case["hkv"] * 4 / BLOCK)
    qo = 4 * case["hq"] * case["d"]  # a query row read and its output written
    flops = 4 * case["hq"] * case["d"]
    kind = case["kind"]
    if kind in ("step", "decode"):
        return {"bytes": held + (put if kind == "step" else 0) + case["batch"] * qo,
                "flops": flops * sum(a + n for a, n in zip(ctx, new))}
    if kind == "prefill":
        return {"bytes": held + sum(new) * qo, "flops": flops * sum(a * n + n * (n + 1) // 2 for a, n in zip(ctx, new))}
    if kind == "append":  # a multiplication and a comparison an element
        back = held + 2 * rows * sum(a + n for a, n in zip(ctx, new)) if case["code"] == "int8" else 0
        return {"bytes": put + back, "flops": 2 * rows * sum(new)}
    return {"bytes": held + 2 * rows * sum(ctx), "flops": rows * sum(ctx)}


# ---- the format ----------------------------------------------------------------------


def _need(amax, code):
    """Smallest power of two s with amax <= MOST * s, at least 2^-126; 0 where amax is 0."""
    m, x = torch.frexp(amax.float())  # amax = m 2^x, 0.5 <= m < 1
    mm, mx = math.frexp(MOST[code])
    e = (x - mx + (m > mm).int()).clamp(min=-126)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(m), e), torch.zeros_like(m))


def _encode(x, scale, code):
    y = torch.where(scale > 0, x / scale, torch.zeros_like(x))
    return y.to(CODES[code]) if code == "e4m3" else y.round().to(torch.int8)


def _flat(pool):
    """Slots of a pool as rows of plain bytes [P * page, Hkv, D]."""
    return pool.view(torch.int8).view(-1, *pool.shape[2:])


def _block_of(slots, page):
    """Flat block number of each slot."""
    return slots // page * (-(-page // BLOCK)) + slots % page // BLOCK


def _values(pool, scale, slots):
    """What the codes at `slots` (any shape) stand for, in 32 bits."""
    codes = _flat(pool)[slots].view(pool.dtype).float()
    return codes * scale.view(-1, scale.shape[2])[_block_of(slots, pool.shape[1])][..., None]


# ---- inputs --------------------------------------------------------------------------


def _rows(g, case, n):
    """Rows [n, Hkv, D] as a model's projections give them: some channels much larger than the others,
    some tokens too."""
    hkv, d = case["hkv"], case["d"]
    wide = 1 + 7 * (torch.rand(hkv, d, generator=g, device=DEV) < 0.03)
    x = torch.randn(n, hkv, d, generator=g, device=DEV) * wide
    return x * torch.exp(0.5 * torch.randn(n, 1, 1, generator=g, device=DEV))


def _pool(g, case, pages):
    """A pool in use: every slot written, block by block (slots past a sequence's end by earlier requests)."""
    ps, hkv, d, code = case["page"], case["hkv"], case["d"], case["code"]
    nb = -(-ps // BLOCK)
    codes = torch.empty(pages, ps, hkv, d, dtype=CODES[code], device=DEV)
    scale = torch.empty(pages, nb, hkv, device=DEV)
    step = max(1, (1 << 27) // (ps * hkv * d))
    for a in range(0, pages, step):
        b = min(pages, a + step)
        x = _rows(g, case, (b - a) * ps).to(DTYPES[case["dtype"]]).float().view(b - a, ps, hkv, d)
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, nb * BLOCK - ps)).view(b - a, nb, BLOCK, hkv, d)
        s = _need(x.abs().amax((2, 4)), code)
        scale[a:b] = s
        codes.view(torch.int8)[a:b] = _encode(x, s[:, :, None, :, None], code).view(torch.int8).view(b - a, nb * BLOCK, hkv, d)[:, :ps]
    return codes, scale


def prepare(case, seed):
    ctx, new = _lens(case)
    g = torch.Generator(device=DEV).manual_seed(1_000_003 * seed + 29)
    ps, hkv, hq, d, B = case["page"], case["hkv"], case["hq"], case["d"], case["batch"]
    lens = [a + n for a, n in zip(ctx, new)]
    npg = [-(-n // ps) for n in lens]
    total = sum(npg)
    P = total + total // 9 + 4  # a pool in use to about nine tenths; page 0 is the null page
    k, k_scale = _pool(g, case, P)
    v, v_scale = _pool(g, case, P)
    table = torch.randperm(P - 1, generator=g, device=DEV)[:total] + 1
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    first = [sum(npg[:b]) for b in range(B + 1)]
    s = {"case": case, "k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale, "indptr": i32(first), "indices": table.int(),
         "last": i32([n - (p - 1) * ps for n, p in zip(lens, npg)]), "total_pages": total, "lens": lens, "new": new,
         "max_len": max(lens), "workspace": None}
    # slots of every sequence's tokens, [B, max_len] (slot 0 past its length)
    pos = torch.arange(max(lens), device=DEV)[None]
    seen = pos < torch.tensor(lens, device=DEV)[:, None]
    s["slots"] = torch.where(seen, table[(s["indptr"][:-1, None] + pos // ps).clamp(max=total - 1).long()] * ps + pos % ps, 0)
    s["seen"] = seen
    if case["kind"] in ("decode", "step"):
        s["q"] = torch.randn(B, hq, d, generator=g, device=DEV).to(DTYPES[case["dtype"]])
    if any(new):
        width = max(new)
        rows = [b * width + width - n + t for b, n in enumerate(new) for t in range(n)] if case["grid"] else list(range(sum(new)))
        n_rows = B * width if case["grid"] else sum(new)
        s.update(width=width, q_rows=i32(rows), qo=i32([sum(new[:b]) for b in range(B + 1)]), total_q=sum(new),
                 # the new tokens' slots, and those of the tokens before them in their first blocks
                 put=torch.cat([s["slots"][b, a:a + n] for b, (a, n) in enumerate(zip(ctx, new))]),
                 held=torch.cat([s["slots"][b, a - a % ps % BLOCK:a] for b, (a, n) in enumerate(zip(ctx, new)) if n]))
        if case["kind"] == "prefill":
            s["q"] = torch.randn(n_rows, hq, d, generator=g, device=DEV).to(DTYPES[case["dtype"]])
        else:
            s["k_new"], s["v_new"] = (_rows(g, case, n_rows).to(DTYPES[case["dtype"]]) for _ in range(2))
    return s


# ---- one pass: the plain form --------------------------------------------------------


def _append(s, pool, scale, rows):
    """Rows [T, Hkv, D] of the new tokens into the pool, in place."""
    case = s["case"]
    code, ps = case["code"], case["page"]
    x = rows.float()
    flat = scale.view(-1, scale.shape[2])
    at = _block_of(s["put"], ps)
    amax = torch.zeros_like(flat).index_reduce_(0, at, x.abs().amax(-1), "amax")
    need = _need(amax, code)
    touched = torch.zeros(flat.shape[0], 1, device=DEV).index_fill_(0, at, 1.0) > 0
    starts = (s["put"] % ps % BLOCK == 0).float()
    fresh = torch.zeros(flat.shape[0], device=DEV).index_reduce_(0, at, starts, "amax")[:, None] > 0
    grown = torch.where(touched, torch.where(fresh, need, torch.maximum(flat, need)), flat)
    bytes_ = _flat(pool)
    held = _values(pool, scale, s["held"])
    bytes_[s["held"]] = _encode(held, grown[_block_of(s["held"], ps)][..., None], code).view(torch.int8)
    bytes_[s["put"]] = _encode(x, grown[at][..., None], code).view(torch.int8)
    flat.copy_(grown)


def _attend(q, k, v, seen):
    """q [B, S, Hq, D] over k, v [B, M, Hkv, D] in 32 bits; seen [B, S, M]: which keys a row sees. A row that
    sees none is zero."""
    B, S, hq, d = q.shape
    hkv = k.shape[2]
    x = q.float().view(B, S, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(B, hkv, -1, d)
    x = torch.matmul(x, k.permute(0, 2, 3, 1)).view(B, hkv, hq // hkv, S, -1) * (1 / math.sqrt(d))
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, hkv, -1, x.shape[-1]), v.permute(0, 2, 1, 3)).view(B, hkv, hq // hkv, S, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(B, S, hq, d)


def _plain(s):
    case, kind = s["case"], s["case"]["kind"]
    dt = DTYPES[case["dtype"]]
    if kind in ("append", "step"):
        at = s["q_rows"].long()
        _append(s, s["k"], s["k_scale"], s["k_new"][at])
        _append(s, s["v"], s["v_scale"], s["v_new"][at])
        state = {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        if kind == "append" and case["code"] == "e4m3":
            return state
    k = _values(s["k"], s["k_scale"], s["slots"])
    v = _values(s["v"], s["v_scale"], s["slots"])
    if kind in ("append", "read"):
        keep = s["seen"][..., None, None]
        out = {"k": torch.where(keep, k, 0).to(dt), "v": torch.where(keep, v, 0).to(dt)}
        return out if kind == "read" else {**out, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if kind in ("decode", "step"):
        o = _attend(s["q"][:, None], k, v, s["seen"][:, None])[:, 0].to(dt)
        return {"out": o, **state} if kind == "step" else {"out": o}
    # rows on a grid of the widest sequence, right-aligned: row w of sequence b sees keys up to len - width + w
    B, W = case["batch"], s["width"]
    n, length = (torch.tensor(x, device=DEV)[:, None] for x in (s["new"], s["lens"]))
    w = torch.arange(W, device=DEV)[None]
    token = (s["qo"][:-1, None] + w - (W - n)).clamp(min=0)  # ragged row of grid row (b, w)
    at = torch.arange(B * W, device=DEV).view(B, W) if case["grid"] else token
    limit = torch.where(w >= W - n, length - W + w, -1)
    seen = torch.arange(k.shape[1], device=DEV)[None, None] <= limit[..., None]
    o = _attend(s["q"][at.long()], k, v, seen).to(dt).reshape(B * W, *s["q"].shape[1:])
    if case["grid"]:
        return {"out": o}
    seq = torch.repeat_interleave(torch.arange(B, device=DEV), n[:, 0], output_size=s["total_q"])
    return {"out": o[seq * W + W - n[seq, 0] + torch.arange(s["total_q"], device=DEV) - s["qo"][seq]]}


# ---- one pass ------------------------------------------------------------------------


def run(state):
    if not own:
        return _plain(state)
    from nanoslg_amd import kernels

    s, case, kind = state, state["case"], state["case"]["kind"]
    cache = (s["k"], s["v"], s["k_scale"], s["v_scale"])
    table = (s["indptr"], s["indices"], s["last"])
    if s["workspace"] is None:  # kept by the program, as its caches keep theirs
        s["workspace"] = kernels.Workspace(torch.device(DEV))
    grid = {"q_rows": s["q_rows"], "grid_width": s["width"]} if case["grid"] else {}
    if kind == "step":
        out = kernels.paged_decode_append_q8(s["q"], s["k_new"], s["v_new"], *cache, *table, s["total_pages"],
                                             workspace=s["workspace"])
        return {"out": out, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if kind == "decode":
        return {"out": kernels.paged_decode_q8(s["q"], *cache, *table, s["total_pages"], workspace=s["workspace"])}
    if kind == "prefill":
        return {"out": kernels.paged_prefill_q8(s["q"], s["qo"], s["total_q"], s["width"], *cache, *table,
                                                workspace=s["workspace"], **grid)}
    state = {}
    if kind == "append":
        kernels.append_kv_q8(s["k_new"], s["v_new"], s["qo"], s["total_q"], *cache, *table, **grid)
        state = {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        if case["code"] == "e4m3":
            return state
    k, v = kernels.gather_kv_q8(*cache, *table, s["max_len"], DTYPES[case["dtype"]])
    return {**state, "k": k, "v": v}


# ---- the same in 64 bits -------------------------------------------------------------


def _round64(y, code):
    """y rounded to the code type's values, ties to even."""
    if code == "int8":
        return y.round()
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return (y / step).round() * step


def _write64(s, b, values, scales, pool, scale, rows):
    """Sequence b's new rows [n, Hkv, D] into values [P, page, Hkv, D] (code values) and scales, block by block."""
    case = s["case"]
    code, ps = case["code"], case["page"]
    n, L = s["new"][b], s["lens"][b]
    pages = s["indices"][s["indptr"][b]:s["indptr"][b + 1]].tolist()
    t = L - n
    while t < L:
        page, slot = pages[t // ps], t % ps
        i = slot // BLOCK
        end = min(L, t - slot + min(ps, (i + 1) * BLOCK))
        x = rows[t - (L - n):end - (L - n)].double()
        amax = x.abs().amax((0, 2))
        e = torch.ceil(torch.log2(amax / MOST[code]))
        need = torch.where(amax > 0, torch.exp2(e.clamp(min=-126)), 0.0)
        old = scale[page, i].double()
        new = need if slot % BLOCK == 0 else torch.maximum(old, need)
        at = values[page, i * BLOCK:slot]
        at.copy_(_round64(torch.nan_to_num(at * (old / new)[:, None]), code))
        values[page, slot:slot + end - t] = _round64(torch.nan_to_num(x / new[:, None]), code)
        scales[page, i] = new
        t = end


def _attend64(q, k, v):
    """Causal attention, bottom-right aligned: q [n, Hq, D] over k, v [m, Hkv, D]."""
    n, hq, d = q.shape
    m, hkv = k.shape[:2]
    G = hq // hkv
    out = torch.empty(n, hq, d, dtype=torch.float64, device=q.device)
    step = max(1, (1 << 27) // max(1, m * G))
    for h in range(hkv):
        kt, vh = k[:, h].t().contiguous(), v[:, h].contiguous()
        for a in range(0, n, step):
            b = min(n, a + step)
            x = q[a:b, h * G:(h + 1) * G].double().reshape(-1, d) @ kt / math.sqrt(d)
            x = x.view(b - a, G, m)
            ahead = torch.arange(m, device=q.device)[None] > torch.arange(m - n + a, m - n + b, device=q.device)[:, None]
            x.masked_fill_(ahead[:, None], -math.inf)
            out[a:b, h * G:(h + 1) * G] = (torch.softmax(x, -1).view(-1, m) @ vh).view(b - a, G, d)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind, ps, B = case["kind"], case["page"], case["batch"]
    got = {}
    for name in ("k", "v"):
        pool, scale = s[name], s[name + "_scale"]
        if kind not in ("append", "step"):
            got[name] = (pool, scale)
            continue
        values, scales = pool.double(), scale.double()
        for b in range(B):
            rows = s[name + "_new"][s["q_rows"][s["qo"][b]:s["qo"][b + 1]].long()]
            _write64(s, b, values, scales, pool, scale, rows)
        got[name] = (values, scales)

    def cached(name, b):
        values, scales = got[name]
        pages = s["indices"][s["indptr"][b]:s["indptr"][b + 1]].long()
        x = values.view(torch.int8)[pages].view(values.dtype) if values.element_size() == 1 else values[pages]
        sc = scales[pages].double().repeat_interleave(BLOCK, 1)[:, :ps]
        return (x.double() * sc[..., None]).flatten(0, 1)[:s["lens"][b]]

    scales = {} if kind in ("decode", "prefill", "read") else {"k_scale": got["k"][1], "v_scale": got["v"][1]}
    codes = {"k": got["k"][0], "v": got["v"][0]} if kind in ("append", "step") else {}
    if kind == "append" and case["code"] == "e4m3":
        return {**codes, **scales}
    if kind in ("append", "read"):
        out = {}
        for name in ("k", "v"):
            out[name] = torch.zeros(B, s["max_len"], case["hkv"], case["d"], dtype=torch.float64, device=DEV)
            for b in range(B):
                out[name][b, :s["lens"][b]] = cached(name, b)
        return {**out, **scales}
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b in range(B):
        at = slice(b, b + 1) if kind != "prefill" else s["q_rows"][s["qo"][b]:s["qo"][b + 1]].long()
        o[at] = _attend64(s["q"][at], cached("k", b), cached("v", b))
    return {"out": o, **codes, **scales}
