"""Trees of drafted tokens in 64 bits: masks, attention, verification and the move of accepted rows, sequence by
sequence, as the definitions in include/nslg_kv.h state them. Test infrastructure only."""
from __future__ import annotations

import math

import torch


def ancestors(parents):
    """Per node the set of nodes that it sees. A parent that is not before its child counts as none."""
    out = []
    for j, p in enumerate(parents):
        out.append({j} | (out[p] if 0 <= p < j else set()))
    return out


def mask_words(trees, max_q):
    """int32 [total, ceil(max_q / 32)]."""
    W = -(-max_q // 32)
    rows = []
    for t in trees:
        for seen in ancestors(t):
            words = [0] * W
            for a in seen:
                words[a // 32] |= 1 << a % 32
            rows.append([w - (1 << 32) if w >= 1 << 31 else w for w in words])
    return torch.tensor(rows, dtype=torch.int32).view(len(rows), W)


def depths(parents):
    return [len(s) - 1 for s in ancestors(parents)]


def attention(q, k, v, see, scale=None):
    """q [n, Hq, D] of a tree's nodes over k, v [m, Hkv, D], its sequence's tokens, the nodes last; see bool [n, n] (node
    i sees node j). Returns the output [n, Hq, D] in 64 bits (zero where a row sees nothing) and two bounds for a
    kernel's error: sum p |v| / sum p, [n, Hq, D], and the largest sum |q_d k_d| scale of a row's seen keys,
    [n, Hq, 1]. What a row does not see does not enter, whatever it is."""
    n, hq, d = q.shape
    m, hkv = k.shape[:2]
    G = hq // hkv
    scale = 1 / math.sqrt(d) if scale is None else scale
    out, mag = torch.zeros(n, hq, d, dtype=torch.float64, device=q.device), torch.zeros(n, hq, d, dtype=torch.float64, device=q.device)
    big = torch.zeros(n, hq, 1, dtype=torch.float64, device=q.device)
    for i in range(n):
        keys = torch.cat([torch.arange(m - n, device=q.device), m - n + see[i].nonzero()[:, 0].to(q.device)])
        if keys.numel() == 0:
            continue
        ki, vi = k[keys].double(), v[keys].double()
        for h in range(hkv):
            qh = q[i, h * G:(h + 1) * G].double()
            kt = ki[:, h].t().contiguous()
            p = torch.softmax(qh @ kt * scale, -1)
            out[i, h * G:(h + 1) * G] = p @ vi[:, h]
            mag[i, h * G:(h + 1) * G] = p @ vi[:, h].abs()
            big[i, h * G:(h + 1) * G, 0] = (qh.abs() @ kt.abs() * scale).amax(-1)
    return out, mag, big


def verify(parents, tokens, target, u_accept, u_next, draft=None, rows=None):
    """One tree: (path, next token). target, draft: 64-bit rows, node j's being rows[j] (default j)."""
    rows = list(range(len(parents))) if rows is None else rows
    if not parents:
        return [], -1

    def clean(x):
        return torch.where((x > 0) & (x < math.inf), x, torch.zeros_like(x))

    path = [0]
    while True:
        node = path[-1]
        r, W = clean(target[rows[node]].double()), 1.0
        q = draft[rows[node]].double() if draft is not None else None
        down = None
        for j in range(node + 1, len(parents)):
            if parents[j] != node:
                continue
            x = tokens[j]
            has = float(r[x]) if 0 <= x < r.numel() else 0.0
            qx = (float(q[x]) if 0 <= x < r.numel() else 1.0) if q is not None else 1.0
            if has > 0 and u_accept[j] * qx * W < has:
                down = j
                break
            if q is None:
                W -= has
                if 0 <= x < r.numel():
                    r[x] = 0
            elif W > 0:
                r = clean(r / W - q)
                W = float(r.sum())
        if down is None:
            break
        path.append(down)
    for left in (r, clean(target[rows[path[-1]]].double())):
        sums = left.cumsum(0)
        if sums[-1] > 0:
            past = (sums > u_next * sums[-1]) & (left > 0)
            return path, int(past.int().argmax()) if past.any() else int((left > 0).nonzero()[-1])
    return path, -1


def move(pool, slots, path):
    """pool [L, slots, ...] in place: the row at slots[path[i]] to slots[i], one after the other."""
    for i, node in enumerate(path):
        pool[:, slots[i]] = pool[:, slots[node]].clone()
