"""The paged serving step's operators (ops.pages_extend / pages_release,
kv4_store / kv4_load, kv4_attention, sample_rows) against plain 64-bit
restatements (serve_rule.py)."""
import numpy as np
import pytest
import torch

import serve_rule as SR
from inferox_b200 import IfxError, ops

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def cuda(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).to(DEV)


def i32(a):
    return cuda(np.asarray(a, np.int64), torch.int32)


# ------------------------------------------------------------------ rows
@pytest.mark.parametrize("G,hd,n", [(1, 32, 1), (8, 128, 16), (3, 96, 33), (2, 64, 130), (1, 256, 7), (5, 160, 20)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_store_writes_the_layout_and_nothing_else(G, hd, n, dtype):
    rng = np.random.default_rng(G * hd + n)
    k, v = (rng.standard_normal((2, n, G, hd)) * np.exp(rng.standard_normal((2, 1, G, hd)))).astype(np.float32)
    k[0, 0, :32] = 0  # a block of zeros
    if n > 4:
        k[1, 0, :3] = (np.nan, 2, -2)  # a NaN, and a tie of the largest magnitude
        v[2, 0, 5] = np.inf if dtype == torch.float32 else 60000
        v[3, 0, :32] = 1e-7 * np.arange(32) if dtype == torch.float32 else 6e-8
    kt, vt = cuda(k).to(dtype), cuda(v).to(dtype)
    n_pages = (n + 63) // 64 + 1
    slots = rng.permutation(n_pages * 64)[:n]
    if n > 6:
        slots[4], slots[5] = -1, n_pages * 64  # skipped
    start = rng.integers(0, 256, (n_pages, ops.kv4_page_bytes(G, hd))).astype(np.uint8)
    want, pages = start.copy(), cuda(start)
    (kq, kd), (vq, vd) = SR.quantise(kt.float().cpu().numpy()), SR.quantise(vt.float().cpu().numpy())
    for i, s in enumerate(slots):
        if 0 <= s < n_pages * 64:
            SR.put(want, s, kq[i], kd[i], vq[i], vd[i])
    ops.kv4_store(kt, vt, i32(slots), pages)
    assert np.array_equal(pages.cpu().numpy(), want)
    for back in (torch.float32, torch.float16):
        lk, lv = ops.kv4_load(i32(slots), pages, G, hd, back)
        live = ((slots >= 0) & (slots < n_pages * 64))[:, None, None]
        with np.errstate(over="ignore"):
            for got, q, d in ((lk, kq, kd), (lv, vq, vd)):
                # the product of a 4-bit and an 11-bit number is exact in f32; f16 rounds it once
                ref = np.where(live, SR.values(q, d), 0).astype(np.float32 if back == torch.float32 else np.float16)
                assert np.array_equal(got.cpu().numpy(), ref)


def test_store_of_slices_of_one_projection():
    """K and V as column slices of the fused projection's rows."""
    n, H, G, hd = 9, 4, 2, 64
    qkv = torch.randn(n, (H + 2 * G) * hd, device=DEV)
    k = qkv[:, H * hd:(H + G) * hd].unflatten(1, (G, hd))
    v = qkv[:, (H + G) * hd:].unflatten(1, (G, hd))
    a, b = ops.kv4_pages(1, G, hd), ops.kv4_pages(1, G, hd)
    ops.kv4_store(k, v, i32(range(n)), a)
    ops.kv4_store(k.contiguous(), v.contiguous(), i32(range(n)), b)
    assert torch.equal(a, b) and a.any()


def test_rows_refuse():
    G, hd = 2, 64
    pages, k = ops.kv4_pages(2, G, hd), torch.zeros(3, G, hd, device=DEV)
    s = i32([0, 1, 2])
    with pytest.raises(IfxError, match="InvalidArgument"):
        ops.kv4_store(k.cpu(), k.cpu(), s, pages)
    with pytest.raises(IfxError, match="Shape"):
        ops.kv4_store(k, k[:2], s, pages)
    with pytest.raises(IfxError, match="Shape"):
        ops.kv4_store(k[:, :1], k[:, :1], s, pages)
    with pytest.raises(IfxError, match="Unsupported"):
        ops.kv4_store(k.double(), k.double(), s, pages)
    with pytest.raises(IfxError, match="InvalidArgument"):
        ops.kv4_store(k, k, s.long(), pages)
    with pytest.raises(IfxError, match="InvalidArgument"):
        ops.kv4_store(k.transpose(1, 2).contiguous().transpose(1, 2), k, s, pages)
    with pytest.raises(IfxError, match="Unsupported"):
        ops.kv4_pages(2, G, 40)
    ops.kv4_store(k[:0], k[:0], s[:0], pages)
    assert ops.kv4_load(s[:0], pages, G, hd)[0].shape == (0, G, hd)


# ------------------------------------------------------------- attention
def filled(rng, lens, G, hd, extra=2, width=None):
    """A cache of sequences of these lengths in shuffled pages; every byte that
    belongs to no row is 0xff (NaN scales)."""
    held = [-(-n // 64) for n in lens]
    n_pages = sum(held) + extra
    perm = rng.permutation(n_pages)
    table = np.full((len(lens), width or max(1, max(held, default=1)) + 1), -1, np.int64)
    pages = torch.full((n_pages, ops.kv4_page_bytes(G, hd)), 255, dtype=torch.uint8, device=DEV)
    K, V, at = [], [], 0
    for b, n in enumerate(lens):
        table[b, :held[b]] = perm[at:at + held[b]]
        at += held[b]
        k = (rng.standard_normal((n, G, hd)) * np.exp(0.5 * rng.standard_normal((1, G, hd)))).astype(np.float32)
        v = rng.standard_normal((n, G, hd)).astype(np.float32)
        t = np.arange(n)
        ops.kv4_store(cuda(k), cuda(v), i32(table[b, t // 64] * 64 + t % 64), pages)
        K.append(SR.values(*SR.quantise(k)))
        V.append(SR.values(*SR.quantise(v)))
    return pages, table, K, V


def bound(ref, K, V, worst, dtype):
    """Score: the products of hd terms in f32 with a split query are off by at
    most (hd + 16) 2^-24 of the sum of magnitudes; a probability by twice that
    plus 2^-21 (exponential, split), the sums over n rows by a random walk of
    f32 roundings, eight deviations of it; the result is rounded once."""
    n = max(len(k) for k in K)
    hd = ref.shape[-1]
    vmax = max(float(np.abs(v).max()) if v.size else 0.0 for v in V)
    rel = 2 * (hd + 16) * 2.0 ** -24 * worst + 2.0 ** -21 + 8 * np.sqrt(n + 1) * 2.0 ** -24
    return vmax * rel + np.abs(ref) * (2.0 ** -11 if dtype == torch.float16 else 2.0 ** -24) + (
        2.0 ** -25 if dtype == torch.float16 else 0)


def check_attention(lens, qlens, H, G, hd, dtype=torch.float32, window=0, scale=None, seed=0, amp=1.0):
    rng = np.random.default_rng(seed + sum(lens) + hd)
    pages, table, K, V = filled(rng, lens, G, hd)
    start = np.concatenate([[0], np.cumsum(qlens)])
    rows = int(start[-1])
    q = cuda((amp * rng.standard_normal((rows, H, hd))).astype(np.float32)).to(dtype)
    one = all(x == 1 for x in qlens)
    ref, worst = SR.attention(q.float().cpu().numpy(), K, V, lens, start, hd ** -0.5 if scale is None else scale, window)
    for qs in ([None] if one else []) + [i32(start)]:
        got = ops.kv4_attention(q, pages, i32(table), i32(lens), G, q_start=qs, scale=scale, window=window)
        got = got.float().cpu().numpy().astype(np.float64)
        err = np.abs(got - ref)
        assert np.all(err <= bound(ref, K, V, worst, dtype)), (float(err.max()), float((err / bound(ref, K, V, worst, dtype)).max()))


@pytest.mark.parametrize("H,G,hd", [(4, 4, 64), (8, 2, 128), (8, 1, 128), (7, 1, 64), (5, 1, 96), (16, 1, 128), (32, 8, 64),
                                    (3, 3, 32), (4, 2, 256), (20, 1, 64), (6, 2, 192), (6, 2, 160)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_attention_one_row(H, G, hd, dtype):
    check_attention([1, 15, 16, 17, 63, 64, 65, 200], [1] * 8, H, G, hd, dtype)


@pytest.mark.parametrize("H,G,hd", [(8, 2, 128), (8, 1, 64), (3, 3, 96), (12, 1, 128)])
@pytest.mark.parametrize("window", [0, 1, 30, 64])
def test_attention_several_rows(H, G, hd, window):
    check_attention([5, 64, 130, 81, 3], [5, 2, 1, 17, 3], H, G, hd, window=window)


@pytest.mark.parametrize("hd,dtype", [(64, torch.float32), (128, torch.float32), (128, torch.float16), (96, torch.float32)])
def test_attention_chunks(hd, dtype):
    check_attention([100, 333, 64], [100, 70, 64], 8, 2, hd, dtype)


@pytest.mark.parametrize("H,G,hd", [(4, 4, 64), (16, 4, 128), (8, 4, 32), (8, 4, 96), (4, 4, 256), (4, 4, 160)])
@pytest.mark.parametrize("window", [0, 50])
def test_attention_chunks_of_many_sequences(H, G, hd, window):
    """Enough query rows for the kernel that takes 64 of them at a time."""
    per = {64: 70, 128: 20, 32: 40, 96: 40, 256: 66, 160: 66}[hd]
    qlens = [per] * 14 + [1, 0, per + 30, 3]
    lens = [q + 37 * i % 150 for i, q in enumerate(qlens)]
    lens[3], qlens[3] = per - 9, per  # rows before the cache's first
    lens[15] = 0
    check_attention(lens, qlens, H, G, hd, torch.float16 if hd == 32 else torch.float32, window=window)


@pytest.mark.parametrize("hd", range(32, 257, 32))
@pytest.mark.parametrize("dtype,window", [(torch.float32, 0), (torch.float32, 70), (torch.float16, 0)])
def test_attention_chunks_every_head_size(hd, dtype, window):
    """Tiles of 128 query rows: groups of three, lengths from none to many
    pages, more query rows than cached ones."""
    H, G = (30, 10) if hd <= 64 else (12, 4)
    check_attention([290, 40, 0, 130, 30, 777], [90, 1, 0, 130, 64, 17], H, G, hd, dtype, window=window)


def test_attention_chunks_whole_prompts_and_one_tile():
    check_attention([200, 129, 1, 64], [200, 129, 1, 64], 16, 8, 128)  # nothing cached before: each row sees up to itself
    check_attention([128], [128], 32, 8, 64)
    check_attention([64] * 12, [64] * 12, 8, 8, 64)  # a page a tile: no partial results
    check_attention([70 + 9 * i for i in range(32)], [1] * 32, 64, 1, 128)  # many heads on one, a row per sequence


def test_attention_chunks_streams_and_graph():
    """Calls that overlap on two streams, each with its own workspace, and a
    captured one give the bits of a call alone."""
    calls = []
    for seed, (H, G, hd) in enumerate([(32, 8, 64), (16, 4, 128)]):
        lens = [500, 333, 128, 64]
        pages, table, _, _ = filled(np.random.default_rng(seed), lens, G, hd)
        q = torch.randn(4 * 64, H, hd, device=DEV)
        args = (q, pages, i32(table), i32(lens), G)
        kw = dict(q_start=i32(64 * np.arange(5)), workspace=ops.kv4_workspace(H, G, hd))
        calls.append((args, kw, ops.kv4_attention(*args, **kw)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    outs = []
    for _ in range(8):
        for st, (args, kw, _) in zip(streams, calls):
            with torch.cuda.stream(st):
                outs.append(ops.kv4_attention(*args, **kw))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out, calls[i % 2][2])
    args, kw, want = calls[0]
    out = torch.zeros_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.kv4_attention(*args, **kw, out=out)
    out.fill_(3.0)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_attention_chunks_gaps_and_magnitudes():
    """The same kernel: a missing page, rows behind the last sequence, a query
    that is not finite, queries and values of very different sizes, a scale
    below 0."""
    H, G, hd, n, ql = 8, 8, 64, 20, 64
    lens = [64 + 7 * i for i in range(n)]
    rng = np.random.default_rng(6)
    pages, table, K, V = filled(rng, lens, G, hd)
    for b in range(0, n, 3):  # values from 1e-3 to 1e3 by sequence and by row
        v = (10.0 ** rng.uniform(-3, 3) * rng.standard_normal((lens[b], G, hd)) *
             10.0 ** rng.uniform(-1, 0, (lens[b], 1, 1))).astype(np.float32)
        k = rng.standard_normal((lens[b], G, hd)).astype(np.float32)
        t = np.arange(lens[b])
        ops.kv4_store(cuda(k), cuda(v), i32(table[b, t // 64] * 64 + t % 64), pages)
        K[b], V[b] = SR.values(*SR.quantise(k)), SR.values(*SR.quantise(v))
    start = np.arange(n + 1) * ql
    q = rng.standard_normal((n * ql + 5, H, hd)).astype(np.float32) * 10.0 ** rng.uniform(-2, 1, (n * ql + 5, 1, 1)).astype(np.float32)
    table[1, 1] = -1  # rows 64 .. of sequence 1 are hidden: every row sees the first page
    out = torch.full((n * ql + 5, H, hd), 7.0, device=DEV)
    got = ops.kv4_attention(cuda(q), pages, i32(table), i32(lens), G, q_start=i32(start), scale=-0.11, out=out).cpu().numpy()
    assert (got[n * ql:] == 7).all()
    for b in range(n):
        sl = slice(start[b], start[b + 1])
        if b == 1:
            k, v, rows = K[1][:64], V[1][:64], q[sl]
            ref = np.zeros((ql, H, hd))
            for i in range(ql):
                e = lens[1] - ql + i + 1
                r, worst = SR.attention(rows[i:i + 1], [k[:min(e, 64)]], [v[:min(e, 64)]], [min(e, 64)], [0, 1], -0.11)
                ref[i] = r[0]
        else:
            k, v = K[b], V[b]
            ref, worst = SR.attention(q[sl], [k], [v], [lens[b]], [0, ql], -0.11)
        lim = bound(ref, [k], [v], worst, torch.float32)
        assert np.all(np.abs(got[sl] - ref) <= lim), (b, float((np.abs(got[sl] - ref) / lim).max()))
    bad = cuda(q)
    bad[70, 3, 5] = np.nan
    bad[71, 2, 5] = np.inf
    got = ops.kv4_attention(bad, pages, i32(table), i32(lens), G, q_start=i32(start), scale=-0.11)
    nan = torch.isnan(got).all(-1)
    assert nan[70, 3] and nan[71, 2] and nan.sum() == 2 and torch.isnan(got).sum() == 2 * hd


def test_attention_query_that_is_not_finite():
    pages, table, _, _ = filled(np.random.default_rng(1), [90, 200], 2, 64)
    q = torch.randn(2, 8, 64, device=DEV)
    q[0, 3, 7], q[1, 5, 0] = np.nan, -np.inf
    got = torch.isnan(ops.kv4_attention(q, pages, i32(table), i32([90, 200]), 2))
    assert got[0, 3].all() and got[1, 5].all() and got.sum() == 2 * 64


def test_attention_empty_rows_and_gaps():
    """kv_len 0, query rows before the cache's first row, sequences without
    query rows, rows behind the last sequence, and a table entry of -1."""
    H, G, hd, lens = 8, 2, 64, [0, 3, 70, 129]
    rng = np.random.default_rng(5)
    pages, table, K, V = filled(rng, lens, G, hd)
    start = np.array([0, 2, 7, 7, 8])  # two rows of nothing; five rows on three; none; one
    q = torch.randn(10, H, hd, device=DEV)
    ref, worst = SR.attention(q[:8].cpu().numpy(), K, V, lens, start, hd ** -0.5)
    out = torch.full_like(q, 7.0)
    ops.kv4_attention(q, pages, i32(table), i32(lens), G, q_start=i32(start), out=out)
    got = out.cpu().numpy().astype(np.float64)
    assert not got[:4].any() and np.all(got[8:] == 7.0)
    assert np.all(np.abs(got[:8] - ref) <= bound(ref, K, V, worst, torch.float32))
    # a sequence whose first page is gone: the rest is what counts
    table2 = table.copy()
    table2[3, 0] = -1
    K2, V2 = [k.copy() for k in K], [v.copy() for v in V]
    K2[3], V2[3] = K[3][64:], V[3][64:]
    ref, worst = SR.attention(q[7:8].cpu().numpy(), K2[3:], V2[3:], [65], [0, 1], hd ** -0.5)
    got = ops.kv4_attention(q[:8], pages, i32(table2), i32(lens), G, q_start=i32(start)).cpu().numpy()[7:]
    assert np.all(np.abs(got - ref) <= bound(ref, K2[3:], V2[3:], worst, torch.float32))
    # ... and one whose every page is gone gives zeros
    table2[3] = -1
    got = ops.kv4_attention(q[:8], pages, i32(table2), i32(lens), G, q_start=i32(start))
    assert not got[7].any()


@pytest.mark.parametrize("ql,seqs", [(1, 3), (2, 3), (70, 20)])  # a row, some rows, chunks of rows
def test_attention_fresh_out_rows_of_no_sequence(ql, seqs):
    """Rows before the first sequence's and behind the last's are 0 in an out
    that the call makes (its memory held sevens), and kept in a given one."""
    H, G, hd, lead, rest = 8, 8, 64, 4, 300
    lens = [80 + 3 * i for i in range(seqs)]
    pages, table, _, _ = filled(np.random.default_rng(3), lens, G, hd)
    start, rows = i32(lead + ql * np.arange(seqs + 1)), lead + ql * seqs + rest
    for dtype in (torch.float32, torch.float16):
        q = torch.randn(rows, H, hd, device=DEV, dtype=dtype)
        ws = ops.kv4_workspace(H, G, hd)
        given = torch.full_like(q, 7.0)
        ops.kv4_attention(q, pages, i32(table), i32(lens), G, q_start=start, out=given, workspace=ws)
        assert (given[:lead] == 7).all() and (given[-rest:] == 7).all()
        sevens = torch.full_like(q, 7.0)
        del sevens
        got = ops.kv4_attention(q, pages, i32(table), i32(lens), G, q_start=start, workspace=ws)
        assert not got[:lead].any() and not got[-rest:].any()
        assert torch.equal(got[lead:-rest], given[lead:-rest])
        sevens = torch.full_like(q, 7.0)
        del sevens
        none = i32(np.zeros((0, 2)))
        assert not ops.kv4_attention(q, pages, none, i32([]), G, q_start=i32([0]), workspace=ws).any()


@pytest.mark.parametrize("amp,scale", [(1e4, 1e-6), (1e-6, 1e3), (30.0, None), (1.0, 0.0), (1.0, -0.3)])
def test_attention_magnitudes(amp, scale):
    check_attention([70, 150], [1, 1], 8, 2, 128, amp=amp, scale=scale)


@pytest.mark.parametrize("mag", [1e-4, 1.0, 3000.0, 3e5])
def test_attention_value_scales(mag):
    """Values of any size, and sequences whose value sizes differ from row to row."""
    H, G, hd, n = 4, 1, 128, 300
    rng = np.random.default_rng(9)
    pages, table, K, V = filled(rng, [n], G, hd)
    v = (mag * rng.standard_normal((n, G, hd)) * 10.0 ** rng.uniform(-2, 0, (n, 1, 1))).astype(np.float32)
    t = np.arange(n)
    k = rng.standard_normal((n, G, hd)).astype(np.float32)
    ops.kv4_store(cuda(k), cuda(v), i32(table[0, t // 64] * 64 + t % 64), pages)
    K, V = [SR.values(*SR.quantise(k))], [SR.values(*SR.quantise(v))]
    q = torch.randn(1, H, hd, device=DEV)
    ref, worst = SR.attention(q.cpu().numpy(), K, V, [n], [0, 1], hd ** -0.5)
    got = ops.kv4_attention(q, pages, i32(table), i32([n]), G).cpu().numpy()
    assert np.all(np.abs(got - ref) <= bound(ref, K, V, worst, torch.float32))


@pytest.mark.parametrize("lens", [[5000], [4097, 1, 1, 1, 900], [64] * 40, [1] * 100, [2500, 0, 33, 1300]])
def test_attention_split(lens):
    """Long axes are cut among many CTAs and joined; many short sequences share one."""
    check_attention(lens, [1] * len(lens), 8, 2, 64, seed=3)


def test_attention_deterministic_and_strided():
    H, G, hd, lens = 8, 2, 128, [700, 64, 2000]
    rng = np.random.default_rng(2)
    pages, table, _, _ = filled(rng, lens, G, hd)
    qkv = torch.randn(3, (H + 2 * G) * hd, device=DEV)
    q = qkv[:, :H * hd].unflatten(1, (H, hd))
    ws = ops.kv4_workspace(H, G, hd, DEV)
    a = ops.kv4_attention(q, pages, i32(table), i32(lens), G, workspace=ws)
    b = ops.kv4_attention(q.contiguous(), pages, i32(table), i32(lens), G, workspace=ws)
    assert torch.equal(a, b)
    wide = torch.full((3, H + 1, hd), 3.0, device=DEV)
    ops.kv4_attention(q, pages, i32(table), i32(lens), G, out=wide[:, :H])
    assert torch.equal(wide[:, :H], a) and (wide[:, H] == 3).all()


def test_attention_far_pages():
    """Page offsets beyond 32 bits: a pool of over 4 GB, the sequence at its end."""
    G, hd, n = 8, 256, 100
    per = ops.kv4_page_bytes(G, hd)
    n_pages = (1 << 32) // per + 40
    pages = torch.empty(n_pages, per, dtype=torch.uint8, device=DEV)
    rng = np.random.default_rng(4)
    k, v = rng.standard_normal((2, n, G, hd)).astype(np.float32)
    table = np.array([[n_pages - 1, n_pages - 3]])
    t = np.arange(n)
    slots = i32(table[0, t // 64] * 64 + t % 64)
    ops.kv4_store(cuda(k), cuda(v), slots, pages)
    K, V = [SR.values(*SR.quantise(k))], [SR.values(*SR.quantise(v))]
    assert np.array_equal(ops.kv4_load(slots, pages, G, hd)[0].cpu().numpy(), K[0].astype(np.float32))
    q = torch.randn(1, 8, hd, device=DEV)
    ref, worst = SR.attention(q.cpu().numpy(), K, V, [n], [0, 1], hd ** -0.5)
    got = ops.kv4_attention(q, pages, i32(table), i32([n]), G).cpu().numpy()
    assert np.all(np.abs(got - ref) <= bound(ref, K, V, worst, torch.float32))


def test_attention_refuses():
    H, G, hd = 8, 2, 64
    pages, q = ops.kv4_pages(2, G, hd), torch.zeros(2, H, hd, device=DEV)
    table, kl = i32([[0], [1]]), i32([1, 1])
    for bad, what in (
            (dict(q=q.double()), "Unsupported"), (dict(G=3), "Shape"), (dict(kl=i32([1])), "Shape"),
            (dict(table=table.long()), "InvalidArgument"), (dict(kl=kl.cpu()), "InvalidArgument"),
            (dict(q_start=i32([0, 1])), "Shape"), (dict(window=-1), "Shape"), (dict(G=4), "Shape"),
            (dict(out=torch.empty(2, H, hd, device=DEV, dtype=torch.float16)), "Shape"),
            (dict(workspace=torch.empty(0, dtype=torch.uint8, device=DEV)), "InvalidArgument"),
            (dict(scale=float("nan")), "InvalidArgument")):
        a = dict(q=q, pages=pages, table=table, kl=kl, G=G) | bad
        if what == "InvalidArgument" and "workspace" in bad and not ops.kv4_workspace(H, G, hd).numel():
            continue
        with pytest.raises(IfxError, match=what):
            ops.kv4_attention(a.pop("q"), a.pop("pages"), a.pop("table"), a.pop("kl"), a.pop("G"), **a)


# ----------------------------------------------------------------- pages
def check_extend(lens, add, width, n_free, max_tokens, seed=0):
    rng = np.random.default_rng(seed)
    held = [-(-x // 64) for x in lens]
    pool = rng.permutation(sum(held) + n_free + 5)
    table = np.full((len(lens), width), -1, np.int64)
    at = 0
    for b, x in enumerate(held):
        table[b, :x] = pool[at:at + x]
        at += x
    free = np.concatenate([pool[at:at + n_free], np.full(7, -9)])
    want = SR.extend(lens, add, table, free, n_free, max_tokens)
    t, f = i32(table), i32(free)
    r = ops.pages_extend(i32(lens), i32(add), t, f, i32([n_free]), max_tokens)
    got = [int(r.status), r.lens.tolist(), t.cpu().numpy(), int(r.n_free), r.q_start.tolist(), r.slots.tolist(),
           r.positions.tolist(), r.seqs.tolist()]
    for g, w in zip(got, want):
        assert np.array_equal(g, w), (g, w)
    assert np.array_equal(f.cpu().numpy(), free)
    return want[0]


@pytest.mark.parametrize("n", [1, 2, 31, 257, 1000])
def test_extend(n):
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 300, n)
    lens[rng.random(n) < 0.3] = 64 * rng.integers(0, 4, (rng.random(n) < 0.3).sum())[0] if n > 3 else 64
    add = np.where(rng.random(n) < 0.2, rng.integers(0, 400, n), rng.integers(0, 2, n))
    need = int((-(-(lens + add) // 64) - -(-lens // 64)).sum())
    assert check_extend(lens.tolist(), add.tolist(), 12, need, int(add.sum())) == 0  # to the last page and row
    assert check_extend(lens.tolist(), add.tolist(), 12, need + 3, int(add.sum()) + 70) == 0
    if need:
        assert check_extend(lens.tolist(), add.tolist(), 12, need - 1, int(add.sum())) == 1
    if add.sum():
        assert check_extend(lens.tolist(), add.tolist(), 12, need, int(add.sum()) - 1) == 3


def test_extend_edges():
    assert check_extend([], [], 4, 2, 5) == 0
    assert check_extend([0, 0], [0, 0], 4, 0, 0) == 0
    assert check_extend([256], [1], 4, 3, 1) == 2
    assert check_extend([255], [1], 4, 0, 1) == 0
    assert check_extend([0, 64, 128], [200000, 1, 0], 4000, 3200, 200001) == 0
    for n in (4096, 8192):
        assert check_extend([3] * n, [1] * n, 1, 0, n) == 0


@pytest.mark.parametrize("n", [1, 40, 700])
def test_release(n):
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 500, n)
    done = rng.integers(0, 2, n)
    table = rng.permutation(n * 8).reshape(n, 8)
    want = [int(table[b, j]) for b in range(n) if done[b] for j in range(-(-lens[b] // 64))]
    free = np.concatenate([[5, 6, 7], np.full(8 * n, -1)])
    f = i32(free)
    lo, nf = ops.pages_release(i32(done), i32(lens), i32(table), f, i32([3]))
    assert lo.tolist() == np.where(done, 0, lens).tolist() and int(nf) == 3 + len(want)
    assert f.tolist() == [5, 6, 7] + want + [-1] * (8 * n - len(want))


def test_pages_refuse():
    a = i32([1, 2])
    t, f, nf = i32([[0, -1], [1, -1]]), i32([2, 3]), i32([2])
    for args in ((a, i32([1]), t, f, nf, 4), (a, a, t[:1], f, nf, 4), (a, a, t, f, i32([1, 2]), 4), (a, a, t, f, nf, -1)):
        with pytest.raises(IfxError, match="Shape"):
            ops.pages_extend(*args)
    for args in ((a.long(), a, t, f, nf, 4), (a, a, t.t(), f, nf, 4), (a, a, t, f.cpu(), nf, 4)):
        with pytest.raises(IfxError, match="InvalidArgument"):
            ops.pages_extend(*args)
    with pytest.raises(IfxError, match="Shape"):
        ops.pages_release(a[:1], a, t, f, nf)


# -------------------------------------------------------------- sampling
def settings(rng, rows):
    return (rng.choice([0.0, 0.3, 0.8, 1.0, 2.0], rows), rng.choice([0, 0, 1, 2, 40, 10 ** 6], rows),
            rng.choice([1.0, 1.0, 0.0, 0.3, 0.9, 0.999], rows), rng.choice([0.0, 0.0, 0.05, 0.5, 1.0, 2.0], rows))


def check_sample(z, u, t, k, p, m):
    f = torch.float32
    token, logp = ops.sample_rows(cuda(z, f), cuda(u, f), cuda(t, f), i32(k), cuda(p, f), cuda(m, f))
    token, logp = token.tolist(), logp.tolist()
    z, u, t, p, m = (np.asarray(x, np.float32).astype(np.float64) for x in (z, u, t, p, m))
    for r in range(len(z)):
        # masses are kept to 2^-45 of the largest weight: 1e-9 of the total covers their sum
        ok = SR.sample(z[r], u[r], t[r], int(k[r]), p[r], m[r], 1e-9)
        assert token[r] in ok, (r, token[r], ok, t[r], k[r], p[r], m[r], u[r])
        ref = ok[token[r]]
        assert logp[r] == ref or abs(logp[r] - ref) <= 2.0 ** -23 * abs(ref) + 4e-9, (r, logp[r], ref)
    return token


@pytest.mark.parametrize("n", [1, 2, 31, 1000, 2048, 2300, 4097, 32000, 128256, 300001])
def test_sample_settings(n):
    rng = np.random.default_rng(n)
    rows = 40 if n <= 32000 else 12
    z = 3 * rng.standard_normal((rows, n))
    z[rng.random((rows, n)) < 0.1] += 5
    check_sample(z, rng.random(rows).astype(np.float32), *settings(rng, rows))


@pytest.mark.parametrize("n", [5, 700, 20000])
def test_sample_ties(n):
    """Equal logits: few distinct values, all equal, -0 beside 0."""
    rng = np.random.default_rng(n)
    rows = 60
    z = rng.integers(-3, 4, (rows, n)).astype(np.float64) * 0.5
    z[:5] = 1.25
    z[5:10] = np.where(rng.random((5, n)) < 0.5, -0.0, 0.0)
    check_sample(z, rng.random(rows).astype(np.float32), *settings(rng, rows))


def test_sample_masks_and_extremes():
    rng = np.random.default_rng(1)
    n, rows = 3000, 12
    z = rng.standard_normal((rows, n))
    hide = rng.random((rows, n)) < 0.95
    z[0][hide[0]] = -np.inf
    z[1][hide[1]] = np.finfo(np.float32).min
    z[2][hide[2]] = np.nan
    z[3] = -np.inf                        # nothing left: -1
    z[4] = np.nan
    z[5] = np.finfo(np.float32).min       # all at the lowest value: uniform
    z[6, 17] = np.inf
    z[7, [3, 2000]] = np.inf
    z[8] = -np.inf
    z[8, n - 1] = -2e38                   # one left, at the end
    z[9] = np.linspace(-3e38, 3e38, n)
    z[10] = 1e-30 * z[10]
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.01), (0.0, 0, 1.0, 0.0), (np.inf, 0, 1.0, 0.0), (1e-38, 5, 1.0, 0.0)):
        one = np.ones(rows)
        for u in (0.0, 0.5, 1 - 2.0 ** -24):
            tok = check_sample(z, u * one, t * one, (k * one).astype(int), p * one, m * one)
            assert tok[3] == tok[4] == -1 and tok[8] == n - 1


def test_sample_agrees_with_the_single_row_sampler():
    """min-p off: the rule of ops.sample_u, whose weights are rounded to f32
    (2^-24 of each, and the quotient z / T to 2^-24 of itself, at most 20): a
    pick may differ only when the draw is that near to a boundary."""
    rng = np.random.default_rng(8)
    n, rows = 5000, 50
    z = (2 * rng.standard_normal((rows, n))).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    t, k, p = 0.8, 60, 0.95
    got = ops.sample_rows(cuda(z), cuda(u), t, k, p)[0].tolist()
    for r in range(rows):
        one = ops.sample_u(cuda(z[r]), t, k, p, float(u[r]))
        eps = 21 * 2.0 ** -24
        near = set(SR.sample(z[r], u[r], np.float32(t), k, np.float32(p), 0.0, eps))
        assert one == got[r] or {one, got[r]} <= near


def test_sample_greedy_is_argmax():
    z = torch.randn(20, 999, device=DEV).round()
    got = ops.sample_rows(z, torch.rand(20, device=DEV), 0.0, 7, 0.5, 0.1)
    assert got[0].tolist() == [ops.argmax(r.contiguous()) for r in z] and not got[1].any()


def test_sample_strided_and_refusals():
    z = torch.randn(6, 500, device=DEV)
    u = torch.rand(6, device=DEV)
    a = ops.sample_rows(z[:, 100:301], u, 0.9, 30)
    b = ops.sample_rows(z[:, 100:301].contiguous(), u, 0.9, 30)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for bad in ((z.half(), u), (z.t(), u), (z, u.double()), (z.cpu(), u)):
        with pytest.raises(IfxError, match="InvalidArgument"):
            ops.sample_rows(*bad)
    with pytest.raises(IfxError, match="Shape"):
        ops.sample_rows(z, u[:5])
    with pytest.raises(IfxError, match="Shape"):
        ops.sample_rows(z[:, :0], u)
    assert ops.sample_rows(z[:0], u[:0])[0].numel() == 0


# -------------------------------------------------------------- together
class Loop:
    """A serving loop over the four operators: admits, stores, attends, samples."""

    def __init__(self, seqs, width, n_pages, G, hd):
        self.G, self.hd = G, hd
        self.table = i32(np.full((seqs, width), -1))
        self.free, self.n_free = i32(np.arange(n_pages)), i32([n_pages])
        self.lens = i32(np.zeros(seqs))
        self.pages = ops.kv4_pages(n_pages, G, hd)

    def step(self, add, done, q, k, v, logits, u, max_tokens):
        lens, n_free = ops.pages_release(done, self.lens, self.table, self.free, self.n_free)
        r = ops.pages_extend(lens, add, self.table, self.free, n_free, max_tokens)
        ops.kv4_store(k, v, r.slots, self.pages)
        out = ops.kv4_attention(q, self.pages, self.table, r.lens, self.G, q_start=r.q_start)
        tok, logp = ops.sample_rows(logits, u, 0.8, 50, 0.95, 0.02)
        self.lens, self.n_free = r.lens, r.n_free
        return r, out, tok


def test_serving_step_together():
    """Requests of uneven lengths arrive, decode, finish and make room; each
    step's attention is that of every sequence's own rows."""
    seqs, H, G, hd, n_pages = 5, 8, 2, 64, 12
    loop = Loop(seqs, 8, n_pages, G, hd)
    rng = np.random.default_rng(12)
    K = [np.zeros((0, G, hd))] * seqs
    V = [np.zeros((0, G, hd))] * seqs
    plan = [([70, 0, 5, 1, 0], [0] * 5), ([1, 130, 1, 1, 0], [0] * 5), ([1, 1, 1, 1, 64], [0] * 5), ([200, 1, 1, 0, 1], [1, 0, 0, 0, 0]),
            ([1, 0, 1, 0, 1], [0, 1, 0, 1, 0])]
    cap = 216
    for add, done in plan:
        n = sum(add)
        q, k, v = (rng.standard_normal((cap, h, hd)).astype(np.float32) for h in (H, G, G))
        z, u = rng.standard_normal((seqs, 777)).astype(np.float32), rng.random(seqs).astype(np.float32)
        r, out, tok = loop.step(i32(add), i32(done), cuda(q), cuda(k), cuda(v), cuda(z), cuda(u), cap)
        assert int(r.status) == 0
        start = np.concatenate([[0], np.cumsum(add)])
        for b in range(seqs):
            if done[b]:
                K[b], V[b] = K[b][:0], V[b][:0]
            sl = slice(start[b], start[b + 1])
            K[b] = np.concatenate([K[b], SR.values(*SR.quantise(k[sl]))])
            V[b] = np.concatenate([V[b], SR.values(*SR.quantise(v[sl]))])
        assert r.lens.tolist() == [len(x) for x in K]
        assert int(r.n_free) == n_pages - sum(-(-len(x) // 64) for x in K)
        ref, worst = SR.attention(q[:n], K, V, [len(x) for x in K], start, hd ** -0.5)
        got = out.cpu().numpy()
        assert np.all(np.abs(got[:n] - ref) <= bound(ref, K, V, worst, torch.float32))
        assert not got[n:].any()
        for b in range(seqs):
            assert tok.tolist()[b] in SR.sample(z[b], u[b], np.float32(0.8), 50, np.float32(0.95), np.float32(0.02), 1e-9)
    # a pool that is too small: nothing moves
    before = loop.table.clone()
    r = ops.pages_extend(loop.lens, i32([0, 400, 0, 0, 0]), loop.table, loop.free, loop.n_free, 400)
    assert int(r.status) == 1 and torch.equal(r.lens, loop.lens) and torch.equal(loop.table, before) and (r.slots == -1).all()


def test_serving_step_captured_and_on_another_stream():
    """The same steps eagerly, on a side stream, and as a replayed graph whose
    inputs change between replays, give the same results bit for bit."""
    seqs, H, G, hd, V = 6, 8, 2, 128, 5000
    steps = 70  # past a page's end
    g = torch.Generator(device=DEV).manual_seed(3)
    data = [tuple(torch.randn(s, device=DEV, generator=g) for s in ((seqs, H, hd), (seqs, G, hd), (seqs, G, hd), (seqs, V))) +
            (torch.rand(seqs, device=DEV, generator=g),) for _ in range(steps)]
    add, done = i32(np.ones(seqs)), i32(np.zeros(seqs))

    def eager():
        loop, got = Loop(seqs, 4, 20, G, hd), []
        for q, k, v, z, u in data:
            _, out, tok = loop.step(add, done, q, k, v, z, u, seqs)
            got.append((out, tok))
        return got

    want = eager()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = eager()
    side.synchronize()
    loop = Loop(seqs, 4, 20, G, hd)
    buf = [x.clone() for x in data[0]]
    lens, n_free = loop.lens, loop.n_free
    with torch.cuda.stream(side):  # warm-up outside the capture, on a copy of the state
        Loop(seqs, 4, 20, G, hd).step(add, done, *buf, seqs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, out, tok = loop.step(add, done, *buf, seqs)
        lens.copy_(r.lens)
        n_free.copy_(r.n_free)
    for i, d in enumerate(data):
        for a, b in zip(buf, d):
            a.copy_(b)
        graph.replay()
        assert torch.equal(out, want[i][0]) and torch.equal(tok, want[i][1]), i
        assert torch.equal(other[i][0], want[i][0]) and torch.equal(other[i][1], want[i][1]), i
    assert lens.tolist() == [steps] * seqs
