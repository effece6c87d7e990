"""The 8-bit KV cache in plain 64-bit arithmetic on the CPU (test infrastructure only).

A layer: code values k, v [P, page, Hkv, D] (float64 holding what the codes are) and scales
[P, nb, Hkv]. Written from the definition, token by token and block by block: no vectorisation
over sequences, no code of the package."""
from __future__ import annotations

import math

import numpy as np

BLOCK = 16
MOST = {"e4m3": 448.0, "int8": 127.0}


def write_kv(k, v, table, start, k_rows, v_rows):
    """A sequence's new rows into layers k and v."""
    k.write(table, start, k_rows, v_rows)
    v.write(table, start, v_rows)


def need_scale(amax: float, code: str) -> float:
    """Smallest power of two s >= 2^-126 with amax <= MOST * s; 0 for amax 0."""
    if amax == 0:
        return 0.0
    e = -126
    while MOST[code] * math.ldexp(1.0, e) < amax:
        e += 1
    return math.ldexp(1.0, e)


def round_code(y: np.ndarray, code: str) -> np.ndarray:
    """y (|y| <= MOST) rounded to the code type's values, ties to even."""
    y = np.asarray(y, np.float64)
    if code == "int8":
        return np.rint(y)
    mag = np.where(np.isfinite(y), np.maximum(np.abs(y), 2.0 ** -6), 1.0)
    _, x = np.frexp(mag)  # mag = m 2^x, 0.5 <= m < 1: 3 mantissa bits behind the leading one
    step = np.ldexp(1.0, x - 1 - 3)
    return np.rint(y / step) * step


class Layer:
    """K or V of one layer."""

    def __init__(self, values, scale, code):
        self.values, self.scale, self.code = np.array(values, np.float64), np.array(scale, np.float64), code
        self.page = self.values.shape[1]

    def write(self, table, start, rows, twin=None):
        """rows [n, Hkv, D] as the tokens at positions start .. start + n - 1 of a sequence with page table `table`.
        K is given V's rows as `twin`: a value that is not finite, in either, is K's to show (chunk by chunk of 8 elements
        for V's); in V it is 0."""
        is_k = twin is not None
        t, n = start, len(rows)
        while t < start + n:
            pid, slot = table[t // self.page], t % self.page
            blk = slot // BLOCK
            stop = min(start + n, t - slot + min(self.page, BLOCK * (blk + 1)))
            for h in range(self.values.shape[2]):
                x = np.asarray(rows[t - start:stop - start, h], np.float64)
                fin = np.isfinite(x)
                spoilt = np.zeros_like(fin)
                if is_k:
                    bad = ~np.isfinite(np.asarray(twin[t - start:stop - start, h], np.float64))
                    spoilt = np.repeat(bad.reshape(len(x), -1, 8).any(2), 8, 1)
                need = need_scale(float(np.abs(np.where(fin, x, 0)).max()), self.code)
                old = float(self.scale[pid, blk, h]) if slot % BLOCK else 0.0
                new = max(need, old)
                if self.code == "int8" and is_k and (not fin.all() or spoilt.any() or math.isnan(old)):
                    new = math.nan
                held = self.values[pid, BLOCK * blk:slot, h]
                if slot % BLOCK and new > old:
                    self.values[pid, BLOCK * blk:slot, h] = round_code(held * old / new, self.code)
                if not new > 0:  # 0 or NaN: zero codes
                    y = np.zeros_like(x)
                else:
                    y = np.where(fin, x, 0) / new
                y = round_code(y, self.code)
                if self.code == "e4m3" and is_k:
                    y = np.where(fin & ~spoilt, y, np.nan)
                self.values[pid, slot:slot + stop - t, h] = y
                self.scale[pid, blk, h] = new
            t = stop

    def read(self, table, length):
        """The values of a sequence's tokens [length, Hkv, D]."""
        out = np.empty((length, *self.values.shape[2:]))
        for t in range(length):
            pid, slot = table[t // self.page], t % self.page
            out[t] = self.values[pid, slot] * self.scale[pid, slot // BLOCK][:, None]
        return out


#: Weights (relative to the row's largest) under `below` are rounded by up to `by`, absolutely: half's subnormals; fp32's
#: range, under which exp2 and the low half of a bf16 pair may be 0. "bf16half": bf16 rows with half weights.
LOW = {"fp16": (2.0 ** -14, 2.0 ** -25), "bf16": (2.0 ** -118, 2.0 ** -125), "bf16half": (2.0 ** -14, 2.0 ** -25)}
#: "bf16up": such weights times 2^7, where V's scales lie within 2^8 of each other (else a bf16 pair's: "bf16"); "bf16runs":
#: either of them by the run of keys, each run with a weight near its largest on every key that counts.
LOW["bf16up"], LOW["bf16runs"] = (2.0 ** -21, 2.0 ** -32), LOW["bf16"]


def attend(q, k, v, scale=None, dtype="fp16"):
    """Causal attention, bottom-right aligned: q [n, Hq, D] over k, v [m, Hkv, D]. Returns out [n, Hq, D] and what
    attention_bound takes: mag = sum_j p_j |v_j|, big = the row's largest sum_d |q_d k_jd| * scale, and low =
    sum_j min(r_j, by) |v_j| over the keys of r_j = p_j / max p < below (LOW[dtype])."""
    n, hq, d = q.shape
    m, hkv = k.shape[:2]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out, mag, low = (np.zeros((n, hq, d)) for _ in range(3))
    big = np.zeros((n, hq, 1))
    ahead = np.arange(m)[None] > np.arange(m - n, m)[:, None]
    for h in range(hq):
        kh, vh = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
        x = q[:, h].astype(np.float64) @ kh.T * scale
        big[:, h, 0] = np.where(ahead, 0, np.abs(q[:, h].astype(np.float64)) @ np.abs(kh).T * scale).max(1, initial=0)
        x = np.where(ahead, -np.inf, x)
        r = np.exp(x - x.max(1, keepdims=True))
        p = r / r.sum(1, keepdims=True)
        out[:, h], mag[:, h] = p @ vh, p @ np.abs(vh)
        low[:, h] = np.where(r < LOW[dtype][0], np.minimum(r, LOW[dtype][1]), 0) @ np.abs(vh)
    return out, mag, big, low


def attention_bound(out, mag, big, low, keys, dtype):
    """How far a kernel's output may be from attend()'s, element by element.

    Scores: products of 16-bit numbers are exact in fp32; a sum of D <= 256 of them (in any order) is off by at
    most 256 * 2^-24 * sum |q k|, the scalings and the exponent's argument by 4 * 2^-24 of its size, exp2 by 2^-22
    relative: delta = (260 * big + 4) * 2^-24, and a softmax weight by 2 * delta relative (numerator and sum).
    Probabilities are rounded to 16 bits: half 2^-11 relative, or below 2^-14 an absolute 2^-25 (or all of them; the
    reference is at most the maximum, so r <= the kernel's value: `low`); a pair of bf16 2^-16 relative, or an absolute
    2^-125 where a part leaves fp32's normal range; and once more where the kernel sums the rounded ones. P.V adds `keys` terms in fp32 and the merge of runs a few more:
    (keys + 64) * 2^-24. All of these are relative to sum p |v|.
    The output is rounded once, 2^-11 (half) or 2^-8 (bf16) of its value; half's subnormals count 2^-25 for it
    and 2^-24 for V at half its scale. "bf16half": a bf16 prefill, whose weights are half's (V exact in half: its
    scales are brought to 2^-15 .. 2^5, or the weights stay in bf16 pairs, which are closer)."""
    u_p, u_o, tiny = {"fp16": (2.0 ** -11, 2.0 ** -11, 2.0 ** -24 + 2.0 ** -25), "bf16": (2.0 ** -16, 2.0 ** -8, 1e-37),
                      "bf16half": (2.0 ** -11, 2.0 ** -8, 1e-37), "bf16up": (2.0 ** -11, 2.0 ** -8, 1e-37),
                      "bf16runs": (2.0 ** -11, 2.0 ** -8, 1e-37)}[dtype]
    delta = (260 * big + 4) * 2.0 ** -24
    err = mag * (2 * delta + 2 * u_p + (keys + 64) * 2.0 ** -24)
    err = err + 2 * low + keys * LOW[dtype][1] * mag  # (in the sum of P.V, and in the sum of the weights)
    return err + u_o * (np.abs(out) + err) + tiny
