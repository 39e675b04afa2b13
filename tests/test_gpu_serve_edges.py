"""Edges of the paged serving step's operators, against serve_rule.py's 64-bit
restatements: values of very different sizes under the attention's sums."""
import numpy as np
import pytest
import torch

import serve_rule as SR
from inferox_b200 import IfxError, ops
from test_gpu_serve_ops import cuda, filled, i32

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def store(pages, table, b, k, v):
    """Rows k, v of sequence b into its pages; the values they then stand for."""
    t = np.arange(len(k))
    k, v = np.asarray(k, np.float32), np.asarray(v, np.float32)
    ops.kv4_store(cuda(k), cuda(v), i32(table[b, t // 64] * 64 + t % 64), pages)
    return SR.values(*SR.quantise(k)), SR.values(*SR.quantise(v))


def own_bound(q, K, V, lens, start, scale, window=0):
    """The result in 64 bits, and a bound from what each row sees itself: a
    score's error as in test_gpu_serve_ops.bound, and twice that of a
    probability; 2^-20 for the exponential and the planes of 22 bits; per
    page of 64 rows fixed-point roundings of 2^-20 (half of 8 / 4.1e6) of the
    largest term, eight deviations of 64 of them; f32's sums; relative to the
    magnitudes summed, at their largest in a block of 32 dimensions (its
    largest value is what a block's scale is made for)."""
    ref, worst = SR.attention(q, K, V, lens, start, scale, window)
    mag = SR.attention(q, K, [np.abs(v) for v in V], lens, start, scale, window)[0]
    mag = np.repeat(mag.reshape(*mag.shape[:-1], -1, 32).max(-1), 32, -1)
    n, hd = max(lens), q.shape[-1]
    rel = 2 * (hd + 16) * 2.0 ** -24 * worst + 2.0 ** -20 + 8 * 8 * 2.0 ** -20 / 3 ** 0.5 + 8 * np.sqrt(n + 1) * 2.0 ** -24
    return ref, mag * rel + np.abs(ref) * 2.0 ** -24


def close(got, ref, lim):
    err = np.abs(got.float().cpu().numpy().astype(np.float64) - ref)
    assert np.all(err <= lim), (float(err.max()), float((err / np.maximum(lim, 1e-300)).max()))


def spread(rng, n, G, hd, scores):
    """Keys whose product with a query of 1 in dimension 0 is scores [n], and a little of the rest."""
    k = 0.01 * rng.standard_normal((n, G, hd))
    k[..., :32] = 0
    k[..., 0] = np.float16(np.asarray(scores) / 8)[:, None].astype(np.float64) * 8
    return k


def ones_first(rng, rows, H, hd):
    q = 0.1 * rng.standard_normal((rows, H, hd)).astype(np.float32)
    q[..., 0] = 1
    return q


@pytest.mark.parametrize("H,G,hd", [(32, 8, 64), (8, 4, 128), (8, 4, 256)])
@pytest.mark.parametrize("ql", [1, 6, 128])
@pytest.mark.parametrize("after", [1, 5, 20, 60])
def test_attention_pages_of_zero_values(H, G, hd, ql, after):
    """One key that stands out, then pages whose values are all 0 with scores 8
    to 12 powers of two below it: they weigh in the sum of every row."""
    rng = np.random.default_rng(after)
    n, seqs = 64 * (1 + after) + ql, 2
    pages, table, K, V = filled(rng, [n] * seqs, G, hd)
    for b in range(seqs):
        s = -np.log(2) * rng.uniform(8, 12, n)
        s[3] = 0
        v = rng.standard_normal((n, G, hd))
        v[64:64 * (1 + after)] = 0
        K[b], V[b] = store(pages, table, b, spread(rng, n, G, hd, s), v)
    q, start = ones_first(rng, seqs * ql, H, hd), ql * np.arange(seqs + 1)
    ref, lim = own_bound(q, K, V, [n] * seqs, start, 1.0)
    close(ops.kv4_attention(cuda(q), pages, i32(table), i32([n] * seqs), G, q_start=i32(start), scale=1.0), ref, lim)


@pytest.mark.parametrize("H,G,hd", [(32, 8, 64), (8, 4, 128), (8, 4, 256)])
@pytest.mark.parametrize("ql", [1, 6, 128])
@pytest.mark.parametrize("big_first", [True, False])
@pytest.mark.parametrize("low", [3e-6, 1e-3, 1.0, 100.0])
def test_attention_pages_of_unequal_values(H, G, hd, ql, big_first, low):
    """A page of large values that hardly weighs beside pages of small ones
    that carry the weight, before them and behind them."""
    rng = np.random.default_rng(int(low * 1e6) + big_first)
    n, seqs = 64 * 5 + ql, 2
    at = 0 if big_first else 192
    pages, table, K, V = filled(rng, [n] * seqs, G, hd)
    for b in range(seqs):
        s = rng.uniform(-2, 0, n)
        s[at:at + 64] -= 40
        v = low * rng.standard_normal((n, G, hd))
        v[at:at + 64] = 50000 * rng.uniform(-1, 1, (64, G, hd))
        K[b], V[b] = store(pages, table, b, spread(rng, n, G, hd, s), v)
    q, start = ones_first(rng, seqs * ql, H, hd), ql * np.arange(seqs + 1)
    ref, lim = own_bound(q, K, V, [n] * seqs, start, 1.0)
    close(ops.kv4_attention(cuda(q), pages, i32(table), i32([n] * seqs), G, q_start=i32(start), scale=1.0), ref, lim)


@pytest.mark.parametrize("H,G,hd", [(4, 2, 64), (8, 1, 128), (4, 1, 96), (2, 2, 256)])
@pytest.mark.parametrize("ql", [1, 5, 128])
@pytest.mark.parametrize("window", [0, 40])
def test_attention_blocks_and_rows_of_unequal_values(H, G, hd, ql, window):
    """Blocks of 32 dimensions 1e4 apart in size, held dimension by dimension,
    and rows 1e4 times larger than the others: outside the window, behind the
    query row, or with hardly any weight. None of them costs the rest."""
    rng = np.random.default_rng(hd + ql + window)
    lens = [150, 64, 39, 260]
    pages, table, K, V = filled(rng, lens, G, hd)
    start = ql * np.arange(len(lens) + 1)
    q = ones_first(rng, start[-1], H, hd)
    for kind in range(4):
        for b, n in enumerate(lens):
            s, v = rng.uniform(-2, 0, n), rng.standard_normal((n, G, hd))
            if kind == 0:
                v *= np.repeat(10.0 ** rng.uniform(-4, 0, (1, G, hd // 32)), 32, -1)
            elif kind == 1:  # a block each, of rows that hardly weigh
                for j in rng.integers(0, n, 5):
                    s[j] = -40
                    v[j, :, :32 * rng.integers(1, hd // 32 + 1)] *= 1e4
            elif kind == 2:  # hidden from every row, or from all but the last
                v[: max(0, n - ql - window + 1) if window else 0] *= 1e4
                v[n - ql + 1:] *= 1e4 if ql > 1 else 1
            else:
                v *= 10.0 ** rng.uniform(-4, 0, (n, 1, 1))
            K[b], V[b] = store(pages, table, b, spread(rng, n, G, hd, s), v)
        ref, lim = own_bound(q, K, V, lens, start, 1.0, window)
        got = ops.kv4_attention(cuda(q), pages, i32(table), i32(lens), G, q_start=i32(start), scale=1.0, window=window)
        close(got, ref, lim)


@pytest.mark.parametrize("H,G,hd,ql", [(8, 4, 64, 128), (8, 4, 256, 128), (8, 1, 128, 9), (4, 2, 64, 1)])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 60, 2 ** 40, 256, 255, 300])
def test_attention_windows_longer_than_the_cache(H, G, hd, ql, window):
    """As without one, also for more query rows than cached ones (256 and 300:
    longer than any sequence of the table, or just so)."""
    rng = np.random.default_rng(ql)
    lens = [100, 200, 3, 0] * 4
    pages, table, K, V = filled(rng, lens, G, hd)
    start = ql * np.arange(len(lens) + 1)
    q = cuda(rng.standard_normal((start[-1], H, hd)).astype(np.float32))
    args = (q, pages, i32(table), i32(lens), G)
    kw = dict(q_start=i32(start))
    assert torch.equal(ops.kv4_attention(*args, **kw, window=window), ops.kv4_attention(*args, **kw))
    ref, lim = own_bound(q.cpu().numpy(), K, V, lens, start, hd ** -0.5, min(window, 1000))
    close(ops.kv4_attention(*args, **kw, window=window), ref, lim)


@pytest.mark.parametrize("ql", [1, 128])
def test_attention_length_beyond_the_table_counts_as_its_end(ql):
    H, G, hd = 8, 4, 64
    rng = np.random.default_rng(2)
    pages, table, _, _ = filled(rng, [128, 128, 128, 128], G, hd)
    q, start = cuda(rng.standard_normal((4 * ql, H, hd)).astype(np.float32)), i32(ql * np.arange(5))
    at = i32(table[:, :2])
    want = ops.kv4_attention(q, pages, at, i32([128] * 4), G, q_start=start)
    assert torch.equal(want, ops.kv4_attention(q, pages, at, i32([129, 128, 5000, 2 ** 31 - 1]), G, q_start=start))


# ----------------------------------------------------------------- pages
@pytest.mark.parametrize("lens,add", [([300, 5], [0, 1]), ([257], [0]), ([2 ** 31 - 1, 0], [0, 0]), ([2 ** 31 - 1], [2 ** 31 - 1])])
def test_extend_refuses_lengths_beyond_the_table(lens, add):
    """A length that the table's row cannot hold is status 2 without new rows too."""
    table = i32(np.arange(4 * len(lens)).reshape(-1, 4))
    r = ops.pages_extend(i32(lens), i32(add), table, i32([90, 91, 92]), i32([3]), 8)
    assert int(r.status) == 2 and r.lens.tolist() == lens and int(r.n_free) == 3
    assert (r.slots == -1).all() and not r.q_start.any() and torch.equal(table, i32(np.arange(4 * len(lens)).reshape(-1, 4)))
    r = ops.pages_extend(i32([256]), i32([0]), table[:1], i32([90]), i32([1]), 8)
    assert int(r.status) == 0 and r.lens.tolist() == [256]


def test_extend_counts_below_zero_are_zero():
    r = ops.pages_extend(i32([-5, 70]), i32([2, -3]), i32([[-1, -1], [1, 0]]), i32([7, 8]), i32([2]), 4)
    assert int(r.status) == 0 and r.lens.tolist() == [2, 70] and int(r.n_free) == 1
    assert r.slots.tolist() == [8 * 64, 8 * 64 + 1, -1, -1] and r.q_start.tolist() == [0, 2, 2]


@pytest.mark.parametrize("page", [1 << 25, 1 << 26, (1 << 26) + 1, 2 ** 31 - 1, -1, -(2 ** 31)])
def test_extend_of_impossible_pages_names_no_slot(page):
    """page * 64 would pass 32 bits and name another page's rows."""
    add = i32([3, 2])
    r = ops.pages_extend(i32([5, 64]), add, i32([[page, -1], [0, -1]]), i32([4, page]), i32([2]), 6)
    assert int(r.status) == 0 and r.slots.tolist() == [-1] * 6
    r = ops.pages_extend(i32([5, 64]), add, i32([[(1 << 25) - 1, -1], [0, -1]]), i32([4, 3]), i32([2]), 6)
    last = 64 * ((1 << 25) - 1)
    assert r.slots.tolist() == [last + 5, last + 6, last + 7, 192, 193, -1]


# -------------------------------------------------------------- refusals
def test_attention_refuses_a_workspace_that_is_not_its_bytes():
    """One byte expanded, every other byte, or another type: the count of the
    elements says nothing of the memory behind them."""
    H, G, hd = 8, 2, 64
    pages, q = ops.kv4_pages(2, G, hd), torch.zeros(2, H, hd, device=DEV)
    ws = ops.kv4_workspace(H, G, hd)
    for bad in (ws[:1].expand(ws.numel()), torch.cat([ws, ws])[::2], ws.view(torch.float32), ws.view(torch.int8)):
        with pytest.raises(IfxError, match="InvalidArgument"):
            ops.kv4_attention(q, pages, i32([[0], [1]]), i32([1, 1]), G, workspace=bad)
    ops.kv4_attention(q, pages, i32([[0], [1]]), i32([1, 1]), G, workspace=ws)


def test_sample_refuses_one_draw_for_all_rows():
    z = torch.randn(4, 50, device=DEV)
    for u in (0.5, 1, np.float32(0.5), [0.1, 0.2, 0.3, 0.4]):
        with pytest.raises(IfxError, match="InvalidArgument"):
            ops.sample_rows(z, u)
    with pytest.raises(IfxError, match="Shape"):
        ops.sample_rows(z, torch.rand(1, device=DEV))


def test_sample_settings_that_are_nan():
    """NaN temperature: greedy; NaN top_p or min_p: off; NaN u: 0, and u beyond
    its range at its ends."""
    z, nan = torch.randn(6, 3000, device=DEV), float("nan")
    u = torch.rand(6, device=DEV)
    assert ops.sample_rows(z, u, nan, 5, 0.5)[0].tolist() == z.argmax(1).tolist()
    for got, want in (((u, 0.8, 40, nan, nan), (u, 0.8, 40)), ((u, 0.8, 0, nan, nan), (u, 0.8)),
                      ((u * nan, 0.8, 40), (u * 0, 0.8, 40)), ((u - 7, 0.8), (u * 0, 0.8)),
                      ((u + 7, 0.8, 0, 0.9), (u * 0 + 1 - 2 ** -24, 0.8, 0, 0.9))):
        a, b = ops.sample_rows(z, *got), ops.sample_rows(z, *want)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
