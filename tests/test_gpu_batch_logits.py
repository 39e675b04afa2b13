"""What a batch's sampling draws from: the batch's own latest logits, whatever
other caches and batches of the model have done in between."""
import numpy as np
import pytest

from inferox_b200 import IfxError, Model, Sampler, synth

pytestmark = pytest.mark.gpu


def _file():
    return synth.build(None, vocab=2048, dim=512, n_layers=2, n_heads=8, n_kv_heads=2, ffn=1024, context=512,
                       rope_base=500000.0, mix=1, seed=31)


def _greedy(kb, n=1):
    return [int(t) for t in kb.sample([Sampler.greedy()] * n, [0.0] * n)[0]]


def _last(z):
    return int(len(z) - 1 - np.argmax(z[::-1]))


@pytest.mark.parametrize("kv_bits,pages", [(16, 0), (16, 8), (4, 8)])
@pytest.mark.parametrize("last_row", [True, False])
def test_prompt_rows_survive_other_caches(kv_bits, pages, last_row):
    m = Model.from_bytes(_file())
    a, b, kv = m.kv_batch(2, 128, pages, kv_bits), m.kv_batch(2, 128, pages, kv_bits), m.kv_cache(128)
    tops = {}
    for seed in range(12):  # prompts whose most likely tokens differ
        m2 = m.prefill(synth.prompt_ids(2048, 9 + seed, seed=seed), m.kv_cache(128), last_row_only=True)[0]
        tops.setdefault(_last(m2), seed)
    assert len(tops) >= 2
    (ta, sa), (tb, sb) = list(tops.items())[:2]
    za = a.prefill(0, synth.prompt_ids(2048, 9 + sa, seed=sa), last_row)[-1]
    assert _greedy(a) == [_last(za)]
    zb = b.prefill(1, synth.prompt_ids(2048, 9 + sb, seed=sb), last_row)[-1]
    assert _last(za) != _last(zb)
    assert _greedy(a) == [_last(za)] and _greedy(b) == [_last(zb)]
    m.prefill(synth.prompt_ids(2048, 9 + sb, seed=sb), kv, last_row_only=True)
    z = m.decode_step(_last(zb), kv)
    assert _greedy(a) == [_last(za)] and _greedy(b) == [_last(zb)]
    assert Sampler.greedy().sample(m) == _last(np.asarray(z).reshape(-1))  # the model's own latest logits


@pytest.mark.parametrize("kv_bits", [16, 4])
def test_refused_steps_leave_the_rows_before(kv_bits):
    m = Model.from_bytes(_file())
    kb = m.kv_batch(3, 192, 3, kv_bits)
    for s in range(2):
        kb.prefill(s, synth.prompt_ids(2048, 63, seed=s), True)
    with pytest.raises(IfxError, match="InvalidArgument"):
        kb.sample([Sampler.greedy()] * 2, [0.0] * 2)  # one prompt row
    logits, _ = kb.decode_step_seqs([1, 0], [3, 4])
    want = [_last(z) for z in logits]
    kb.prefill(2, [5, 6], True)
    last = _greedy(kb)
    with pytest.raises(IfxError, match="OutOfMemory"):
        kb.decode_step_seqs([0, 1, 2], [1, 2, 3])  # sequences 0 and 1 would need a page each
    with pytest.raises(IfxError, match="InvalidArgument"):
        kb.sample([Sampler.greedy()] * 3, [0.0] * 3)
    assert _greedy(kb) == last
    logits, _ = kb.decode_step_seqs([2], [want[0]])
    with pytest.raises(IfxError, match="OutOfMemory"):
        kb.decode_step_seqs([1, 0], [1, 2])
    with pytest.raises(IfxError, match="InvalidTensorIndex"):
        kb.decode_step_seqs([2], [9999])
    assert _greedy(kb) == [_last(logits[0])]
    with pytest.raises(IfxError, match="InvalidTensorIndex"):
        kb.prefill(2, [9999], True)
    with pytest.raises(IfxError, match="InvalidTensorIndex"):
        kb.prefill(2, np.arange(200), True)  # beyond max_seq
    assert _greedy(kb) == [_last(logits[0])]


def test_greedy_loop_leaves_its_last_rows():
    m = Model.from_bytes(_file())
    for kv_bits in (16, 4):
        kb = m.kv_batch(2, 192, 0, kv_bits)
        for s in range(2):
            kb.prefill(s, synth.prompt_ids(2048, 20 + s, seed=s), True)
        out, _ = kb.decode_greedy([7, 8], 5)
        assert _greedy(kb, 2) == [int(t) for t in out[-1]]


@pytest.mark.parametrize("kind", ["cache", "batch", "paged", "q4"])
def test_memory_is_zeroed_before_its_first_use(kind):
    """Work of the caller's on the default stream, which the zeroing of a new
    cache runs behind, while the model's own stream is free."""
    import torch
    m, ids = Model.from_bytes(_file()), synth.prompt_ids(2048, 40, seed=3)

    def run():
        if kind == "cache":
            kv = m.kv_cache(128)
            m.prefill(ids, kv, last_row_only=True)
            torch.cuda.synchronize()
            return kv, m.decode_step(9, kv)
        kb = m.kv_batch(2, 128, 8 if kind in ("paged", "q4") else 0, 4 if kind == "q4" else 16)
        kb.prefill(1, ids, True)
        token = kb.sample([Sampler(1.0, 20, 0.9)], [0.7])[0][0]
        torch.cuda.synchronize()
        return kb, kb.decode_step_seqs([1], [9])[0][0], token

    want = run()
    torch.cuda._sleep(int(4e8))  # about 0.2 s
    got = run()
    assert np.all(np.abs(got[1] - want[1]) <= 2e-2 + 1e-2 * np.abs(want[1])), float(np.abs(got[1] - want[1]).max())
    assert got[2:] == want[2:]
