"""The batch whose cache is held in 4 bits (kv_batch(kv_bits=4)) and sampled
serving.

The reference keeps f32 rows (src/model/cache.rs:7-14); what this cache must
give is the model over the rows as they are quantised. A restatement of the
layer forward in 64 bits (forward.rs:215-440) over the file's dequantised
weights does that: a prompt attends to its own rows as computed, a decode
step to the Q4_0 rows. Logits are held to the bar of the other batch tests.
"""
import numpy as np
import pytest

import serve_rule as SR
from inferox_b200 import IfxError, Model, Sampler, synth
from inferox_b200.model import uniform
from inferox_b200.serving import Server
from oracle import refcpu as R

pytestmark = pytest.mark.gpu

ATOL, RTOL = 2e-2, 1e-2


def _close(g, r):
    return np.all(np.abs(g - r) <= ATOL + RTOL * np.abs(r))


class Ref:
    """Layer forward in 64 bits with a Q4_0 cache per sequence."""

    def __init__(self, g, compat=True):
        o = R.Model(g)
        c = self.c = o.config
        self.compat = compat

        D, F, hd = int(c.hidden_size), int(c.intermediate_size), int(c.head_dim)
        rows = {"attn_q": D, "attn_k": int(c.n_kv_heads) * hd, "attn_v": int(c.n_kv_heads) * hd, "attn_output": D,
                "ffn_gate": F, "ffn_up": F, "ffn_down": D, "token_embd": int(c.vocab_size), "output": int(c.vocab_size)}

        def t(name):
            kind = name.split(".")[-2]
            cols = F if kind == "ffn_down" else D
            x = R.dequantize(o.tensor_info(name)[0], o.tensor_bytes(name), rows.get(kind, 1) * cols).astype(np.float64)
            return x.reshape(rows[kind], cols) if kind in rows else x

        self.emb, self.norm = t("token_embd.weight"), t("output_norm.weight")
        self.head = t("output.weight") if o.has_output() else self.emb
        self.L = [{k: t(f"blk.{i}.{k}.weight") for k in ("attn_norm", "attn_q", "attn_k", "attn_v", "attn_output", "ffn_norm",
                                                         "ffn_gate", "ffn_up", "ffn_down")} for i in range(int(c.n_layers))]
        self.H, self.G, self.hd = int(c.n_heads), int(c.n_kv_heads), int(c.head_dim)

    def cache(self):
        return [[np.zeros((0, self.G, self.hd))] * 2 for _ in self.L]

    def rms(self, x, w):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.c.norm_eps) * w

    def rope(self, x, pos):
        i = np.arange(0, int(self.c.rope_dim), 2)
        ang = np.asarray(pos)[:, None] * (1.0 / self.c.rope_base ** (i / self.c.rope_dim))
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
        y = x.copy()
        a, b = x[..., i], x[..., i + 1]
        y[..., i], y[..., i + 1] = a * c - b * s, a * s + b * c
        return y

    def run(self, ids, cache, step):
        n, start = len(ids), len(cache[0][0])
        pos = np.arange(n) if self.compat else start + np.arange(n)
        if step and self.compat:
            pos = np.zeros(n)
        x = self.emb[np.asarray(ids)]
        for L, kv in zip(self.L, cache):
            h = self.rms(x, L["attn_norm"])
            q = self.rope((h @ L["attn_q"].T).reshape(n, self.H, self.hd), pos)
            k = self.rope((h @ L["attn_k"].T).reshape(n, self.G, self.hd), pos)
            v = (h @ L["attn_v"].T).reshape(n, self.G, self.hd)
            kv[0] = np.concatenate([kv[0], SR.values(*SR.quantise(k))])
            kv[1] = np.concatenate([kv[1], SR.values(*SR.quantise(v))])
            ks, vs = (kv[0], kv[1]) if step else (k, v)
            a = SR.attention(q, [ks], [vs], [len(ks)], [0, n], self.hd ** -0.5)[0]
            x = x + a.reshape(n, -1) @ L["attn_output"].T
            h = self.rms(x, L["ffn_norm"])
            g = h @ L["ffn_gate"].T
            x = x + (g / (1 + np.exp(-g)) * (h @ L["ffn_up"].T)) @ L["ffn_down"].T
        return self.rms(x[-1], self.norm) @ self.head.T


def _file(**kw):
    return synth.build(None, **(dict(vocab=2048, dim=512, n_layers=2, n_heads=8, n_kv_heads=2, ffn=1024, context=512,
                                     rope_base=500000.0, mix=1, seed=31) | kw))


@pytest.mark.parametrize("compat", [True, False])
@pytest.mark.parametrize("kw", [{}, dict(n_heads=4, n_kv_heads=1, seed=7)])  # 64- and 128-wide heads
def test_q4_batch_matches_the_quantised_model(kw, compat):
    g = _file(**kw)
    m, o = Model.from_bytes(g, rope_compat=compat), Ref(g, compat)
    V = int(m.config.vocab_size)
    lens = [60, 70, 130, 5]  # 1, 2, 3 and 1 pages; sequence 0 takes a page while decoding
    kb = m.kv_batch(len(lens), 256, pages=10, kv_bits=4)
    assert kb.pages() == (10, 10)
    caches, toks = [o.cache() for _ in lens], []
    for s, n in enumerate(lens):
        p = synth.prompt_ids(V, n, seed=70 + s)
        gl, rl = kb.prefill(s, p, True)[0], o.run(p, caches[s], False)
        assert _close(gl, rl), (s, float(np.max(np.abs(gl - rl))))
        toks.append(int(np.argmax(rl)))
    assert kb.pages() == (3, 10)
    for step in range(6):
        logits, amax = kb.decode_step(toks)
        for s in range(len(lens)):
            rl = o.run([toks[s]], caches[s], True)
            assert _close(logits[s], rl), (step, s, float(np.max(np.abs(logits[s] - rl))))
            assert int(amax[s]) == R.argmax(logits[s])
            toks[s] = int(np.argmax(rl))
    # some of them, out of order: rows keep the caller's order
    for seqs in ([3, 0], [2], [1, 3, 0]):
        logits, amax = kb.decode_step_seqs(seqs, [toks[s] for s in seqs])
        for i, s in enumerate(seqs):
            rl = o.run([toks[s]], caches[s], True)
            assert _close(logits[i], rl), (seqs, s, float(np.max(np.abs(logits[i] - rl))))
            assert int(amax[i]) == R.argmax(logits[i])
            toks[s] = int(np.argmax(rl))
    assert [kb.len(s) for s in range(4)] == [68, 77, 137, 13]
    assert kb.pages() == (10 - 2 - 2 - 3 - 1, 10)
    # a slot is handed to a new request, stale rows and all
    kb.reset(2)
    assert kb.pages() == (5, 10) and kb.len(2) == 0
    caches[2] = o.cache()
    p = synth.prompt_ids(V, 90, seed=99)
    assert _close(kb.prefill(2, p, True)[0], o.run(p, caches[2], False))
    logits, _ = kb.decode_step_seqs([2], [17])
    assert _close(logits[0], o.run([17], caches[2], True))


def test_q4_pool_runs_dry_and_refusals():
    m = Model.from_bytes(_file())
    kb = m.kv_batch(2, 512, pages=3, kv_bits=4)
    kb.prefill(0, synth.prompt_ids(2048, 64, seed=1), True)
    kb.prefill(1, synth.prompt_ids(2048, 100, seed=2), True)
    with pytest.raises(IfxError, match="OutOfMemory"):
        kb.decode_step([1, 2])  # sequence 0 needs a page
    assert kb.pages() == (0, 3) and [kb.len(s) for s in (0, 1)] == [64, 100]
    kb.decode_step_seqs([1], [5])
    with pytest.raises(IfxError, match="OutOfMemory"):
        kb.decode_greedy([1, 2], 30)
    with pytest.raises(IfxError, match="InvalidTensorIndex"):
        kb.prefill(0, np.arange(449), True)  # beyond max_seq
    with pytest.raises(IfxError, match="InvalidTensorIndex"):
        kb.prefill(0, [4000], True)
    kb.reset(1)
    kb.decode_step_seqs([0], [5])
    assert kb.pages() == (1, 3) and kb.len(0) == 65
    with pytest.raises(ValueError):
        m.kv_batch(2, 64, kv_bits=8)
    m48 = Model.from_bytes(synth.build("tiny", n_layers=1))
    with pytest.raises(IfxError, match="Unsupported"):  # 48-wide heads
        m48.kv_batch(2, 64, kv_bits=4)


def test_q4_greedy_loop_replays_the_steps():
    """The captured loop gives what the same steps give one by one."""
    m = Model.from_bytes(_file())
    runs = []
    for loop in (False, True):
        kb = m.kv_batch(3, 256, kv_bits=4)
        toks = []
        for s, n in enumerate((50, 61, 10)):
            toks.append(int(np.argmax(kb.prefill(s, synth.prompt_ids(2048, n, seed=s), True)[0])))
        if loop:
            out = [list(map(int, r)) for r in kb.decode_greedy(toks, 20)[0]]
        else:
            out = []
            for _ in range(20):
                logits, amax = kb.decode_step(toks)
                toks = [int(t) for t in amax]
                top2 = np.sort(logits, 1)[:, -2:]
                out.append((toks, (top2[:, 1] - top2[:, 0]).min()))
        runs.append(out)
    for i, ((want, margin), got) in enumerate(zip(*runs)):
        if margin < 1e-2:  # sums of the weight products vary in order: a near tie may part the two
            break
        assert want == got, i
    assert i >= 1


def test_long_prompt_beyond_the_f16_pages():
    """A sequence longer than the 64 pages of the f16 pool's table."""
    m = Model.from_bytes(_file(n_layers=1, context=8192))
    kb = m.kv_batch(1, 5000, kv_bits=4)
    logits = kb.prefill(0, synth.prompt_ids(2048, 4500, seed=3), True)
    logits, _ = kb.decode_step([int(np.argmax(logits))])
    assert kb.len(0) == 4501 and np.isfinite(logits).all() and logits.std() > 0


class Recorder:
    """A batch that keeps the logits every draw was made from."""

    def __init__(self, kb):
        self.kb, self.batch, self.max_seq, self.draws = kb, kb.batch, kb.max_seq, []

    def pages(self):
        return self.kb.pages()

    def prefill(self, *a):
        self.last = self.kb.prefill(*a)
        return self.last

    def decode_step_seqs(self, seqs, toks, want_logits=True):
        self.last, amax = self.kb.decode_step_seqs(seqs, toks)
        return None, amax

    def reset(self, s):
        self.kb.reset(s)

    def sample(self, samplers, u):
        toks, logp = self.kb.sample(samplers, u)
        self.draws.append((self.last.copy(), samplers, u, toks, logp))
        return toks, logp


@pytest.mark.parametrize("kv_bits,pages", [(16, 0), (16, 8), (4, 8)])
def test_sampled_serving(kv_bits, pages):
    m = Model.from_bytes(_file())
    kb = Recorder(m.kv_batch(3, 192, pages, kv_bits))
    srv = Server(kb)
    kinds = [Sampler(0.8, 40, 0.95), None, Sampler(1.2, 0, 0.9, 0.02), Sampler(1.0), None, Sampler(0.7, 0, 1.0, 0.1)]
    rids = [srv.submit(synth.prompt_ids(2048, 20 + 17 * i, seed=i), 12 + 3 * i, sampler=s, seed=100 + i)
            for i, s in enumerate(kinds)]
    got = srv.run()
    assert [len(got[r]) for r in rids] == [12 + 3 * i for i in range(6)]
    n = 0
    for logits, samplers, us, toks, logp in kb.draws:
        assert len(logits) == len(samplers)
        for z, s, u, t, lp in zip(logits, samplers, us, toks, logp):
            ok = SR.sample(z, np.float32(u), np.float32(s.temperature), s.top_k, np.float32(s.top_p), np.float32(s.min_p), 1e-9)
            assert int(t) in ok and abs(ok[int(t)] - lp) <= 2.0 ** -23 * abs(lp) + 4e-9
            n += s.temperature > 0
    assert n >= 12 + 18 + 21 + 27  # a preempted request draws again


def test_sampler_with_min_p_on_the_model():
    m = Model.from_bytes(_file())
    kv = m.kv_cache(64)
    z = m.prefill(synth.prompt_ids(2048, 9, seed=4), kv, last_row_only=True)[0]
    for seed in range(20):
        t = Sampler(1.0, 0, 1.0, 0.2).sample(m, seed, 3)
        assert t in SR.sample(z, np.float32(uniform(seed, 3)), 1.0, 0, 1.0, np.float32(0.2), 1e-9)
    # the same uniform numbers as the single-row sampler's
    for seed in range(20):
        a, b = Sampler(0.9, 50, 0.9).sample(m, seed, 5), Sampler(0.9, 50, 0.9, 1e-30).sample(m, seed, 5)
        near = SR.sample(z, np.float32(uniform(seed, 5)), np.float32(0.9), 50, np.float32(0.9), 0.0, 21 * 2.0 ** -24)
        assert a == b or {a, b} <= set(near)
    kb = m.kv_batch(2, 64)
    with pytest.raises(IfxError, match="InvalidArgument"):
        kb.sample([Sampler(1.0)], [0.5])  # nothing decoded yet
    kb.prefill(0, [1, 2, 3], True)
    with pytest.raises(IfxError, match="InvalidArgument"):
        kb.sample([Sampler(1.0)] * 2, [0.5, 0.5])
