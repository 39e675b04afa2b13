"""The serving step's operators over a key/value cache held in 4 bits, as measured cases.

A paged serving loop runs, every step: page tables and slot maps for the rows that arrive (pages_release,
pages_extend), the rows' keys and values into the cache (kv4_store; kv4_load reads rows back), attention over
the cache (kv4_attention), and the next tokens (sample_rows). Each case is one pass through one of them.

`own` False: the plain form, elementary torch operations. `own` True: the calls of inferox_b200.ops.

The cache's memory, which both forms work on: pages of 64 rows. A page holds, for each kv head, four tiles of
16 rows; a tile holds, with NB = head_dim / 32 blocks of 32 values per row,
  key words    [row][t][b]          u32: values 32 b + 8 t + i in nibble i             (256 NB bytes)
  key scales   [row][b]             f16                                                 (32 NB bytes)
  value words  [row pair][g][b]     u32: values 32 b + 4 g + j of the even row in nibble j of the low half,
                                    of the odd row in the high half                     (256 NB bytes)
  value scales [row][b]             f16                                                 (32 NB bytes)
A block is quantised as Q4_0: d = f16(m / -8) with m the first value of the largest magnitude, the stored
nibble trunc(x / d + 8.5) within 0..15, and the nibble q stands for (q - 8) d.
"""
import math

import numpy as np
import torch

own = False

PAGE = 64
DEV = "cuda"


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of a full batch: every sequence takes one token, a few need a page
        dict(name="pages_decode_32", op="pages", seqs=32, max_pages=64, prefill=0, done=2, ctx=2000),
        # a mixed step of a large server: 480 decoding, 32 prompts admitted, 32 finished
        dict(name="pages_mixed_512", op="pages", seqs=512, max_pages=512, prefill=32, done=32, ctx=6000),
        # the rows of one decode step of 16 sequences, 8B geometry
        dict(name="store_decode_16", op="store", n=16, G=8, hd=128, type="f32", pad=0),
        # a prompt chunk with padding at its end
        dict(name="store_prompt_4096", op="store", n=4096, G=8, hd=128, type="f32", pad=37),
        # the shortest attention: one sequence at a 1024-token prompt, 8B geometry (32 heads on 8)
        dict(name="attn_b1_1k", op="attn", seqs=1, ctx=1100, ragged=0.0, qlen=1, G=8, grp=4, hd=128, type="f32", window=0),
        # batched decode of 16 sequences of uneven length, 8B geometry
        dict(name="attn_b16_2k", op="attn", seqs=16, ctx=2300, ragged=0.8, qlen=1, G=8, grp=4, hd=128, type="f32", window=0),
        # a large server, 70B geometry (64 heads on 8), long and short sequences together
        dict(name="attn_b64_8k", op="attn", seqs=64, ctx=8192, ragged=0.9, qlen=1, G=8, grp=8, hd=128, type="f32", window=0),
        # one very long context
        dict(name="attn_b1_128k", op="attn", seqs=1, ctx=131072, ragged=0.0, qlen=1, G=8, grp=4, hd=128, type="f16", window=0),
        # a chunk of new rows of each sequence against its cache (prompt in chunks), 1B geometry (32 heads of 64 on 8)
        dict(name="attn_chunk_128", op="attn", seqs=4, ctx=3001, ragged=0.3, qlen=128, G=8, grp=4, hd=64, type="f32", window=0),
        # one request's next token, every filter on
        dict(name="sample_1", op="sample", rows=1, vocab=32000, mix="chat"),
        # a batch's next tokens, filters differing by row
        dict(name="sample_64", op="sample", rows=64, vocab=128256, mix="mixed"),
        # many rows drawn from the whole distribution (no filter)
        dict(name="sample_256_free", op="sample", rows=256, vocab=128256, mix="free"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pages", "store", "attn", "attn", "attn", "sample", "sample"])
    if op == "pages":
        seqs = _log(rng, 1, 512)
        return dict(op=op, seqs=seqs, max_pages=rng.choice([64, 200, 512]), prefill=rng.randint(0, max(1, seqs // 16)),
                    done=rng.randint(0, max(1, seqs // 16)), ctx=_log(rng, 10, 4000))
    if op == "store":
        n = _log(rng, 1, 4096)
        return dict(op=op, n=n, G=rng.choice([1, 2, 3, 4, 8]), hd=rng.choice([32, 64, 96, 128]), type=rng.choice(["f32", "f16"]),
                    pad=rng.randint(0, n // 4))
    if op == "sample":
        return dict(op=op, rows=_log(rng, 1, 200), vocab=rng.choice([_log(rng, 50, 128256), 32000, 128256]),
                    mix=rng.choice(["chat", "mixed", "free", "masked"]))
    G, grp = rng.choice([(1, 8), (2, 4), (4, 1), (4, 7), (8, 4), (8, 8), (8, 2), (2, 16), (6, 1), (3, 5)])
    hd = rng.choice([32, 64, 96, 128, 128, 256])
    qlen = rng.choice([1, 1, 1, rng.randint(2, 8), rng.randint(9, 100)])
    seqs = _log(rng, 1, 48)
    if qlen > 8:
        seqs = min(seqs, 4)
    # cached rows x heads of 32 values: at most what the largest listed case has, its chunk's work for chunks
    most = (64 * 4500 * 8 * 4 if qlen <= 8 else 4 * 2700 * 8 * 2 * 128 // qlen) // (seqs * G * (hd // 32) * (1 if qlen == 1 else 4))
    ctx = _log(rng, 2, min(40000, max(300, most)))
    return dict(op=op, seqs=seqs, ctx=max(ctx, qlen), ragged=rng.choice([0.0, 0.5, 0.95]), qlen=qlen, G=G, grp=grp, hd=hd,
                type=rng.choice(["f32", "f32", "f16"]), window=rng.choice([0, 0, 0, rng.randint(1, 2000)]))


# ----------------------------------------------------------------- inputs
def _dtype(case):
    return torch.float16 if case["type"] == "f16" else torch.float32


def _lens(case, rng):
    """Lengths of the sequences (rows in the cache, the new ones among them): even, or spread downwards by `ragged`."""
    u = rng.random(case["seqs"])
    n = np.maximum(case["qlen"], np.round(case["ctx"] * (1.0 - case["ragged"] * u)).astype(np.int64))
    n[0] = case["ctx"]
    return n


def _pages_lens(case, rng):
    cap = case["max_pages"] * PAGE
    lens = np.minimum(cap - 1, rng.integers(0, 2 * case["ctx"], case["seqs"]))
    new = np.ones(case["seqs"], np.int64)
    at = rng.permutation(case["seqs"])
    fill, gone = at[: case["prefill"]], at[case["prefill"]:][: case["done"]]
    lens[fill] = 0
    new[fill] = rng.integers(1, 2 * min(512, cap // 2), len(fill))
    done = np.zeros(case["seqs"], np.int64)
    done[gone] = 1
    new[gone] = 0
    return lens, new, done


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    s = dict(case)
    i32 = dict(dtype=torch.int32, device=DEV)

    def up(a):
        return torch.from_numpy(np.ascontiguousarray(a)).to(**i32)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    if case["op"] == "pages":
        lens, new, done = _pages_lens(case, rng)
        held = -(-lens // PAGE)
        n_pages = int(held.sum() + (-(-(lens + new) // PAGE)).sum() + 8)
        perm = rng.permutation(n_pages)
        table = np.full((case["seqs"], case["max_pages"]), -1, np.int64)
        table[np.arange(case["max_pages"])[None, :] < held[:, None]] = perm[: held.sum()]
        free = np.concatenate([perm[held.sum():], np.full(held.sum(), -1)])
        s.update(lens=up(lens), new=up(new), done=up(done), table=up(table), free=up(free), n_free=up([n_pages - held.sum()]),
                 max_tokens=case["seqs"] + case["prefill"] * 2 * min(512, case["max_pages"] * PAGE // 2))
    elif case["op"] == "store":
        n, G, hd = case["n"], case["G"], case["hd"]
        # keys have a few channels far larger than the others, as rotary models' keys do
        channel = torch.exp(0.7 * normal(1, G, hd))
        s["k"] = (normal(n, G, hd) * channel).to(_dtype(case))
        s["v"] = normal(n, G, hd).to(_dtype(case))
        n_pages = -(-n // PAGE) + 3
        slots = rng.permutation(n_pages * PAGE)[:n] if n <= 64 else np.arange(n) + 17  # scattered decode rows; a prompt's rows in order
        slots[n - case["pad"]:] = -1
        s["slots"] = up(slots)
        s["pages"] = torch.zeros(n_pages, G * 2304 * (hd // 32), dtype=torch.uint8, device=DEV)
    elif case["op"] == "attn":
        G, grp, hd = case["G"], case["grp"], case["hd"]
        lens = _lens(case, rng)
        held = -(-lens // PAGE)
        n_pages = int(held.sum())
        width = int(held.max()) + 1
        table = np.full((case["seqs"], width), -1, np.int64)
        table[np.arange(width)[None, :] < held[:, None]] = rng.permutation(n_pages)
        s["table"], s["kv_len"] = up(table), up(lens)
        s["q_start"] = None if case["qlen"] == 1 else up(np.arange(case["seqs"] + 1) * case["qlen"])
        s["q"] = (1.5 * normal(case["seqs"] * case["qlen"], G * grp, hd)).to(_dtype(case))
        s["pages"] = torch.zeros(n_pages, G * 2304 * (hd // 32), dtype=torch.uint8, device=DEV)
        step = max(1, (1 << 26) // (PAGE * G * hd))  # the cache is filled some pages at a time
        for a in range(0, n_pages, step):
            b = min(n_pages, a + step)
            k, v = normal((b - a) * PAGE, G, hd), normal((b - a) * PAGE, G, hd)
            _put(s["pages"][a:b], torch.arange((b - a) * PAGE, device=DEV), k, v)
    else:
        rows, n = case["rows"], case["vocab"]
        # a long flat body and some tokens that stand out
        z = 2.2 * normal(rows, n)
        top = torch.randint(0, n, (rows, 24), generator=g, device=DEV)
        z.scatter_add_(1, top, 6.0 + 3.0 * normal(rows, 24))
        if case["mix"] == "masked":  # a grammar's mask: most tokens at minus infinity or at the type's lowest value
            hide = torch.rand(rows, n, generator=g, device=DEV) < 0.9
            low = torch.where(torch.arange(rows, device=DEV) % 2 == 0, -math.inf, torch.finfo(torch.float32).min)
            z = torch.where(hide, low[:, None], z)
        s["logits"] = z
        s["u"] = torch.rand(rows, generator=g, device=DEV)
        one = np.ones(rows)
        t, k, p, m = rng.choice([0.6, 0.8, 1.0, 1.3], rows), 40 * one, 0.95 * one, 0.02 * one
        if case["mix"] in ("mixed", "masked"):
            t = np.where(rng.random(rows) < 0.1, 0.0, t)
            k = rng.choice([0, 0, 1, 20, 50, 500], rows)
            p = rng.choice([1.0, 1.0, 0.5, 0.9, 0.99], rows)
            m = rng.choice([0.0, 0.0, 0.05, 0.3], rows)
        elif case["mix"] == "free":
            t, k, p, m = one, 0 * one, one, 0 * one
        f32 = dict(dtype=torch.float32, device=DEV)
        s.update(temperature=torch.tensor(t, **f32), top_k=up(k), top_p=torch.tensor(p, **f32), min_p=torch.tensor(m, **f32))
    return s


# ------------------------------------------------------------------ plain forms
def _quantise(x):
    """Nibbles and scales of the blocks of 32 along the last axis, in 32 bits."""
    x = x.float().unflatten(-1, (-1, 32))
    m = x.gather(-1, x.abs().argmax(-1, keepdim=True))
    d = (m / -8.0).clamp(-65504.0, 65504.0).half()
    inv = torch.where(d == 0, 0.0, 1.0 / d.float())
    return (x * inv + 8.5).trunc().clamp(0, 15).to(torch.uint8), d.squeeze(-1)


def _parts(pages, hd):
    """Views of the parts of every tile: key words [P, G, 4, 16, 4, NB, 4 bytes], key scales [.., 16, NB], value words
    [.., 8 pairs, 8, NB, 2 rows, 2 bytes], value scales."""
    nb = hd // 32
    t = pages.view(pages.shape[0], -1, 4, 576 * nb)
    a, b, c = 256 * nb, 288 * nb, 544 * nb
    return (t[..., :a].unflatten(-1, (16, 4, nb, 4)), t[..., a:b].unflatten(-1, (16, nb, 2)),
            t[..., b:c].unflatten(-1, (8, 8, nb, 2, 2)), t[..., c:].unflatten(-1, (16, nb, 2)))


def _put(pages, slots, k, v):
    """Rows k, v [n, G, hd] quantised into the rows `slots` of the pages."""
    kw, ks, vw, vs = _parts(pages, k.shape[-1])
    page, tile, row = slots // PAGE, slots % PAGE // 16, slots % 16
    for words, scales, x, axes in ((kw, ks, k, (4, 8)), (vw, vs, v, (8, 4))):
        q, d = _quantise(x)  # [n, G, NB, 32]
        q = q.unflatten(-1, axes).transpose(2, 3)  # [n, G, lane, NB, nibbles]
        byte = q[..., 0::2] | (q[..., 1::2] << 4)
        if words is kw:
            words[page, :, tile, row] = byte
        else:
            words[page, :, tile, row // 2, :, :, row % 2] = byte
        scales[page, :, tile, row] = d.contiguous().view(torch.uint8).unflatten(-1, (-1, 2))


def _values(byte, d, dtype):
    """[.., lane, NB, bytes] and scales [.., NB, 2 bytes] -> [.., hd]"""
    q = torch.stack([byte & 15, byte >> 4], -1).flatten(-2).transpose(-3, -2).flatten(-2)  # [.., NB, 32]
    return ((q.to(dtype) - 8.0) * d.contiguous().view(torch.float16).to(dtype)).flatten(-2)


def _get(pages, slots, hd, dtype=torch.float32):
    """The rows `slots` [n] of the pages as keys and values [n, G, hd]."""
    kw, ks, vw, vs = _parts(pages, hd)
    page, tile, row = slots // PAGE, slots % PAGE // 16, slots % 16
    return (_values(kw[page, :, tile, row], ks[page, :, tile, row], dtype),
            _values(vw[page, :, tile, row // 2, :, :, row % 2], vs[page, :, tile, row], dtype))


def _plain_store(s):
    keep = s["slots"] >= 0
    _put(s["pages"], s["slots"][keep].long(), s["k"][keep], s["v"][keep])
    k, v = _get(s["pages"], s["slots"].long().clamp(min=0), s["hd"])
    keep = keep[:, None, None]
    return {"k": torch.where(keep, k, 0.0), "v": torch.where(keep, v, 0.0)}


def _plain_attn(s):
    B, ql, G, grp, hd = s["seqs"], s["qlen"], s["G"], s["grp"], s["hd"]
    L = int(s["table"].shape[1]) * PAGE
    at = torch.arange(L, device=DEV)
    slots = s["table"].long().clamp(min=0)[:, at // PAGE] * PAGE + at % PAGE
    k, v = _get(s["pages"], slots.flatten(), hd)
    k, v = k.view(B, L, G, hd).transpose(1, 2), v.view(B, L, G, hd).transpose(1, 2)
    q = s["q"].float().view(B, ql, G, grp, hd).permute(0, 2, 1, 3, 4).reshape(B, G, ql * grp, hd)
    x = (q @ k.transpose(-1, -2)).view(B, G, ql, grp, L) / math.sqrt(hd)
    pos = s["kv_len"].long()[:, None] - ql + torch.arange(ql, device=DEV)  # [B, ql]
    seen = at <= pos[..., None]
    if s["window"]:
        seen &= at > pos[..., None] - s["window"]
    x = x.masked_fill(~seen[:, None, :, None, :], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = p.view(B, G, ql * grp, L) @ v / p.sum(-1).view(B, G, ql * grp, 1)
    return o.view(B, G, ql, grp, hd).transpose(1, 2).reshape(B * ql, G * grp, hd).to(s["q"].dtype)


def _plain_pages(s):
    lens, table, free, B = s["lens"].long(), s["table"], s["free"], s["seqs"]
    width = s["max_pages"]
    # finished sequences give their pages back, in the order of sequences and positions
    held = -(-lens // PAGE)
    gone = torch.where(s["done"] != 0, held, 0)
    n_free = s["n_free"].long()
    col = torch.arange(width, device=DEV)
    give = col[None, :] < gone[:, None]
    at = n_free + (gone.cumsum(0) - gone)[:, None] + col[None, :]
    free[at[give]] = table[give]
    n_free = n_free + gone.sum()
    lens = torch.where(s["done"] != 0, 0, lens)
    # the others take pages from the end of the free list for their new rows
    new = s["new"].long()
    held, need = -(-lens // PAGE), -(-(lens + new) // PAGE)
    take = need - held
    fits = (take.sum() <= n_free) & (need.max() <= width)
    new, take = new * fits, take * fits
    fresh = (col[None, :] >= held[:, None]) & (col[None, :] < (held + take)[:, None])
    at = n_free - 1 - (take.cumsum(0) - take)[:, None] - (col[None, :] - held[:, None])
    table[fresh] = free[at[fresh]]
    q_start = torch.cat([new.new_zeros(1), new.cumsum(0)])
    t = torch.arange(s["max_tokens"], device=DEV)
    seq = torch.searchsorted(q_start, t, right=True) - 1
    live = t < q_start[-1]
    seq_of = seq.clamp(max=B - 1)
    pos = lens[seq_of] + t - q_start[seq_of]
    slot = table[seq_of, (pos // PAGE).clamp(max=width - 1)].long() * PAGE + pos % PAGE
    out = dict(lens=lens + new, n_free=n_free - take.sum(), q_start=q_start, slots=torch.where(live, slot, -1),
               positions=torch.where(live, pos, -1), seqs=torch.where(live, seq, -1), status=1 - fits.long().view(1))
    return {"table": table} | {k: v.int() for k, v in out.items()}


def _plain_sample(s):
    z = s["logits"].double()
    rows, n = z.shape
    t, k, p, m = s["temperature"].double()[:, None], s["top_k"].long(), s["top_p"].double()[:, None], s["min_p"].double()[:, None]
    greedy = t <= 0
    top = z.amax(-1, keepdim=True)
    w = torch.exp((z - top) / torch.where(greedy, 1.0, t))
    order = z.sort(dim=-1, descending=True, stable=True).indices
    free = (k[:, None] <= 0) & (p >= 1) & (m <= 0)
    order = torch.where(free, torch.arange(n, device=DEV), order)
    w = w.gather(1, order)
    c = w.cumsum(-1)
    rank = torch.arange(n, device=DEV)[None, :]
    kept = torch.where(k > 0, k, n).clamp(max=n)[:, None]
    kept = torch.where(p < 1, torch.minimum(kept, (c < p * c[:, -1:]).sum(-1, keepdim=True) + 1), kept)
    kept = torch.where(free, n, torch.minimum(kept, (w >= m).sum(-1, keepdim=True)))
    mass = c.gather(1, kept - 1)
    at = torch.minimum(((c <= s["u"].double()[:, None] * mass) & (rank < kept)).sum(-1, keepdim=True), kept - 1)
    token, logp = order.gather(1, at), torch.log(w.gather(1, at) / mass)
    last = n - 1 - (z == top).flip(1).int().argmax(-1, keepdim=True)
    return {"token": torch.where(greedy, last, token)[:, 0].int(), "logprob": torch.where(greedy, 0.0, logp)[:, 0].float()}


# ------------------------------------------------------------------ a pass
def run(s):
    if own:
        from inferox_b200 import ops

        if s["op"] == "pages":
            lens, n_free = ops.pages_release(s["done"], s["lens"], s["table"], s["free"], s["n_free"])
            r = ops.pages_extend(lens, s["new"], s["table"], s["free"], n_free, s["max_tokens"])
            return {"table": s["table"], "lens": r.lens, "n_free": r.n_free, "q_start": r.q_start, "slots": r.slots,
                    "positions": r.positions, "seqs": r.seqs, "status": r.status}
        if s["op"] == "store":
            ops.kv4_store(s["k"], s["v"], s["slots"], s["pages"])
            k, v = ops.kv4_load(s["slots"], s["pages"], s["G"], s["hd"])
            return {"k": k, "v": v}
        if s["op"] == "attn":
            return ops.kv4_attention(s["q"], s["pages"], s["table"], s["kv_len"], s["G"], q_start=s["q_start"], window=s["window"])
        token, logp = ops.sample_rows(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        return {"token": token, "logprob": logp}
    return {"pages": _plain_pages, "store": _plain_store, "attn": _plain_attn, "sample": _plain_sample}[s["op"]](s)


# ------------------------------------------------------------------ least work
def work(case):
    if case["op"] == "pages":
        tokens = case["seqs"] + case["prefill"] * min(512, case["max_pages"] * PAGE // 2)
        pages = (tokens + case["done"] * case["ctx"]) // PAGE + case["seqs"] // PAGE
        return {"bytes": 24 * case["seqs"] + 12 * tokens + 8 * pages + 16, "flops": 0}
    if case["op"] == "store":
        values = 2 * case["n"] * case["G"] * case["hd"]
        size = 2 if case["type"] == "f16" else 4
        return {"bytes": values * (size + 2 * 4.5 / 8 + 4) + 8 * case["n"], "flops": 5 * values}
    if case["op"] == "attn":
        # every cached row that a query row sees, once, at 4.5 bits a value; the average length of `ragged`
        G, grp, hd, ql, B = case["G"], case["grp"], case["hd"], case["qlen"], case["seqs"]
        mean = (case["ctx"] + (B - 1) * max(ql, case["ctx"] * (1 - case["ragged"] / 2))) / B
        seen = min(mean, case["window"]) if case["window"] else max(1.0, mean - (ql - 1) / 2)
        rows = min(mean, case["window"] + ql - 1) if case["window"] else mean
        size = 2 if case["type"] == "f16" else 4
        return {"bytes": B * (rows * 2 * G * hd * 4.5 / 8 + 2 * ql * G * grp * hd * size), "flops": 4 * B * ql * G * grp * hd * seen}
    return {"bytes": 4 * case["rows"] * (case["vocab"] + 7), "flops": 20 * case["rows"] * case["vocab"]}


# ------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        # what the rows stand for; the scale and the product x / d are rounded to 16 and 32 bits by definition
        out = {}
        for name in ("k", "v"):
            x = s[name].float().cpu().numpy().reshape(case["n"], case["G"], -1, 32)
            big = np.take_along_axis(x, np.abs(x).argmax(-1)[..., None], -1).astype(np.float64)
            d = np.clip(big / -8, -65504, 65504).astype(np.float16).astype(np.float32)
            inv = np.divide(np.float32(1), d, out=np.zeros_like(d), where=d != 0)
            q = np.clip(np.floor((x * inv).astype(np.float32) + np.float32(8.5)), 0, 15)
            y = (q.astype(np.float64) - 8) * d
            y[s["slots"].cpu().numpy() < 0] = 0
            out[name] = y.reshape(s[name].shape)
        return out
    if case["op"] == "attn":
        G, grp, hd, ql = case["G"], case["grp"], case["hd"], case["qlen"]
        if case["seqs"] * case["ctx"] * G * hd > 1 << 30:
            return None
        lens, table = s["kv_len"].tolist(), s["table"].long()
        q = s["q"].double().view(case["seqs"], ql, G, grp, hd)
        out = torch.zeros_like(q)
        for b, n in enumerate(lens):
            at = torch.arange(n, device=DEV)
            k, v = _exact_rows(s["pages"], table[b, at // PAGE] * PAGE + at % PAGE, G, hd)  # [n, G, hd]
            for i in range(ql):
                last = n - ql + i
                first = max(0, last - case["window"] + 1) if case["window"] else 0
                x = torch.einsum("ghd,ngd->ghn", q[b, i], k[first:last + 1]) / hd ** 0.5
                out[b, i] = torch.einsum("ghn,ngd->ghd", torch.softmax(x, -1), v[first:last + 1])
        return out.view(case["seqs"] * ql, G * grp, hd)
    if case["op"] == "sample":
        z = s["logits"].cpu().numpy().astype(np.float64)
        cols = [s[x].cpu().numpy() for x in ("temperature", "top_k", "top_p", "min_p", "u")]
        token, logp = np.zeros(len(z), np.int32), np.zeros(len(z))
        for r, (t, k, p, m, u) in enumerate(zip(*(c.tolist() for c in cols))):
            row = z[r]
            if t <= 0:
                token[r] = len(row) - 1 - np.argmax(row[::-1])
                continue
            w = np.exp((row - row.max()) / t)
            if k > 0 or p < 1 or m > 0:
                order = np.lexsort((np.arange(len(row)), -row))
                c, ends = np.cumsum(w[order]), [len(row)]
                if k > 0:
                    ends.append(k)
                if p < 1:
                    ends.append(np.searchsorted(c, p * c[-1], side="left") + 1)
                if m > 0:
                    ends.append(np.count_nonzero(w >= m))
                order = order[:max(1, min(ends))]
            else:
                order = np.arange(len(row))
            c = np.cumsum(w[order])
            i = min(int(np.searchsorted(c, u * c[-1], side="right")), len(order) - 1)
            token[r], logp[r] = order[i], np.log(w[order[i]]) - np.log(c[-1])
        return {"token": token, "logprob": logp}
    return None


def _exact_rows(pages, slots, G, hd):
    """Rows of the cache in 64 bits, word by word as the layout at the top of this file says."""
    nb = hd // 32
    base = (slots // PAGE * G)[:, None] * 4 * 576 * nb + torch.arange(G, device=DEV) * 4 * 576 * nb + ((slots % PAGE // 16) * 576 * nb)[:, None]
    base, row, flat = base[..., None], (slots % 16)[:, None, None], pages.view(-1)
    x = torch.arange(hd, device=DEV)
    b, r = x // 32, x % 32

    def half(at):
        u = flat[at].int() | (flat[at + 1].int() << 8)
        return u.to(torch.int16).view(torch.float16).double()

    def nibble(word, n):
        return (flat[word + n // 2] >> (4 * (n % 2)).to(torch.uint8)) & 15

    k = nibble(base + 4 * ((row * 4 + r // 8) * nb + b), r % 8).double() - 8
    v = nibble(base + 288 * nb + 4 * ((row // 2 * 8 + r // 4) * nb + b) + 2 * (row % 2), r % 4).double() - 8
    return (k * half(base + 256 * nb + 2 * (row * nb + b)), v * half(base + 544 * nb + 2 * (row * nb + b)))
