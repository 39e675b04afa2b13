"""Plain 64-bit restatements of the paged serving step's operators, for its
tests: Q4_0 rows, the pages' byte layout, attention, page tables, sampling."""
from __future__ import annotations

import numpy as np

PAGE = 64


def quantise(x):
    """Nibbles (0..15) and f16 scales of blocks of 32 along the last axis; a
    NaN counts as 0 and the scale stops at 65504. The products x * (1 / d) and
    + 8.5 are rounded to f32, as the format's quantiser does."""
    x = np.where(np.isnan(x), 0, np.asarray(x, np.float32)).astype(np.float32)
    x = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    if not x.size:
        return np.zeros(x.shape, np.uint8), np.zeros(x.shape[:-1], np.float16)
    at = np.abs(x).argmax(-1)[..., None]
    with np.errstate(over="ignore"):
        d = np.clip(np.take_along_axis(x, at, -1) / np.float32(-8), -65504, 65504).astype(np.float16)
    f = d.astype(np.float32)
    inv = np.divide(np.float32(1), f, out=np.zeros_like(f), where=f != 0)
    with np.errstate(over="ignore", invalid="ignore"):
        q = np.clip(np.trunc((x * inv).astype(np.float32) + np.float32(8.5)), 0, 15).astype(np.uint8)
    return q, d[..., 0]


def values(q, d):
    return ((q.astype(np.float64) - 8) * d.astype(np.float64)[..., None]).reshape(*q.shape[:-2], 32 * q.shape[-2])


def put(pages, slot, kq, kd, vq, vd):
    """One row's nibbles [G, NB, 32] and scales [G, NB] at `slot` of pages (uint8 [n_pages, bytes])."""
    g_, nb = kd.shape
    r, tile = slot % 16, slot % PAGE // 16
    for h in range(g_):
        p = pages[slot // PAGE, (h * 4 + tile) * 576 * nb:][: 576 * nb]
        for b in range(nb):
            for x in range(32):
                w = 4 * ((r * 4 + x // 8) * nb + b) + x % 8 // 2
                p[w] = (p[w] & (0xF0 if x % 2 == 0 else 0x0F)) | kq[h, b, x] << 4 * (x % 2)
                w = 288 * nb + 4 * ((r // 2 * 8 + x // 4) * nb + b) + 2 * (r % 2) + x % 4 // 2
                p[w] = (p[w] & (0xF0 if x % 2 == 0 else 0x0F)) | vq[h, b, x] << 4 * (x % 2)
            p[256 * nb + 2 * (r * nb + b):][:2] = np.frombuffer(kd[h, b].tobytes(), np.uint8)
            p[544 * nb + 2 * (r * nb + b):][:2] = np.frombuffer(vd[h, b].tobytes(), np.uint8)


def attention(q, k, v, kv_len, q_start, scale, window=0):
    """q [rows, H, d]; k, v: per sequence [len, G, d] (64 bits). Also the largest
    sum of |q k| * scale of a score, for error bounds."""
    out = np.zeros(q.shape, np.float64)
    worst = 0.0
    for b, n in enumerate(kv_len):
        lo, hi = q_start[b], q_start[b + 1]
        if n == 0:
            continue
        grp = q.shape[1] // k[b].shape[1]
        for i in range(lo, hi):
            last = n - (hi - lo) + (i - lo)
            first = max(0, last - window + 1) if window else 0
            if last < first:
                continue
            for h in range(q.shape[1]):
                kk, vv = k[b][first:last + 1, h // grp], v[b][first:last + 1, h // grp]
                x = kk @ q[i, h].astype(np.float64) * scale
                worst = max(worst, float((np.abs(kk) @ np.abs(q[i, h].astype(np.float64))).max() * abs(scale)))
                p = np.exp(x - x.max())
                out[i, h] = p @ vv / p.sum()
    return out, worst


def extend(lens, add, table, free, n_free, max_tokens):
    """(status, lens, table, n_free, q_start, slots, positions, seqs)"""
    lens, table, n = list(lens), table.copy(), len(lens)
    blank = [-1] * max_tokens
    need = [-(-(a + b) // PAGE) for a, b in zip(lens, add)]
    status = 0
    if any(x > table.shape[1] for x in need):
        status = 2
    elif sum(add) > max_tokens:
        status = 3
    elif sum(x - -(-a // PAGE) for x, a in zip(need, lens)) > n_free:
        status = 1
    if status:
        return status, lens, table, n_free, [0] * (n + 1), blank, blank, blank
    starts, slots, pos, seqs = [0], [], [], []
    for b in range(n):
        for j in range(-(-lens[b] // PAGE), need[b]):
            n_free -= 1
            table[b, j] = free[n_free]
        for t in range(lens[b], lens[b] + add[b]):
            slots.append(table[b, t // PAGE] * PAGE + t % PAGE)
            pos.append(t)
            seqs.append(b)
        starts.append(len(slots))
        lens[b] += add[b]
    pad = [-1] * (max_tokens - len(slots))
    return 0, lens, table, n_free, starts, slots + pad, pos + pad, seqs + pad


def sample(z, u, t, k, p, m, eps=0.0):
    """The tokens that the rule can draw for one row when every cumulative
    boundary may move by `eps` of the total, and {token: logprob}."""
    z = np.where(np.isnan(z), -np.inf, np.asarray(z, np.float64))
    n, top = len(z), z.max()
    if top == -np.inf:
        return {-1: -np.inf}
    if not t > 0:
        return {int(n - 1 - np.argmax(z[::-1])): 0.0}
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(z == top, 1.0, np.where((z == -np.inf) | (top == np.inf), 0.0, np.exp((z - top) / t)))
    if k > 0 or p < 1 or m > 0:
        order = np.lexsort((np.arange(n), -z))
        c = np.cumsum(w[order])
        end = n if k <= 0 else min(n, k)
        if m > 0:
            end = min(end, max(1, int((w >= min(m, 1.0)).sum())))
        ends = {end}
        if p < 1:
            a, b = (int(np.searchsorted(c, (p + e) * c[-1], side="left")) + 1 for e in (-eps, eps))
            ends = {min(end, max(1, x)) for x in range(a, b + 1)}
    else:
        order, ends = np.arange(n), {n}
    got = {}
    for end in ends:
        c = np.cumsum(w[order[:end]])
        for e in (-eps, eps):
            i = min(int(np.searchsorted(c, (u + e) * c[-1], side="right")), end - 1)
            while w[order[i]] == 0 and i > 0:  # u at the very end
                i -= 1
            got[int(order[i])] = float(np.log(w[order[i]]) - np.log(c[-1]))
    return got
