"""A prompt for which the device has no memory left fails as OutOfMemory,
changes nothing, and the calls after it go on as if it had not been made."""
import gc

import numpy as np
import pytest
import torch

from inferox_b200 import IfxError, Model, synth

pytestmark = pytest.mark.gpu

V, N, SPARE = 32000, 2000, 64 << 20  # all logits of N rows: 256 MB


@pytest.fixture
def full_device():
    """Fills the device but for SPARE bytes while the fixture's call runs."""
    def run(call):
        torch.cuda.synchronize()
        gc.collect()
        torch.cuda.empty_cache()
        held = torch.empty(max(0, torch.cuda.mem_get_info()[0] - SPARE), dtype=torch.uint8, device="cuda")
        try:
            return call()
        finally:
            del held
            torch.cuda.empty_cache()
    return run


def _model():
    return Model.from_bytes(synth.build(None, vocab=V, dim=256, n_layers=1, n_heads=4, n_kv_heads=2, ffn=512, context=4096,
                                        rope_base=500000.0, mix=1, seed=5))


def check(kind, full_device):
    m, ids = _model(), synth.prompt_ids(V, N, seed=1)
    if kind == "cache":
        kv = m.kv_cache(4096)
        prompt = lambda ids, last: m.prefill(ids, kv, last_row_only=last)
        step, length = (lambda t: m.decode_step(t, kv)), (lambda: len(kv))
    else:
        kb = m.kv_batch(2, 4096, 80 if kind in ("paged", "q4") else 0, 4 if kind == "q4" else 16)
        prompt = lambda ids, last: kb.prefill(1, ids, last)
        step, length = (lambda t: kb.decode_step_seqs([1], [t])[0][0]), (lambda: kb.len(1))
    prompt(ids, True)  # the workspace of N rows is there
    assert length() == N
    pages = kb.pages() if kind in ("paged", "q4") else None
    with pytest.raises(IfxError, match="OutOfMemory"):
        full_device(lambda: prompt(ids, False))
    assert length() == N
    if kind == "q4":
        assert kb.pages() == pages
    got = step(17)
    if kind != "cache":  # the same step of a batch that never failed
        kb = m.kv_batch(2, 4096, 80 if kind in ("paged", "q4") else 0, 4 if kind == "q4" else 16)
        kb.prefill(1, ids, True)
        want = kb.decode_step_seqs([1], [17])[0][0]
    else:
        kv = m.kv_cache(4096)
        m.prefill(ids, kv, last_row_only=True)
        want = m.decode_step(17, kv)
    # sums of up to 512 weight products vary in order from run to run: 512 * 2^-24 of logits below 10, over four layers' sums
    assert np.all(np.abs(got - want) <= 4 * 512 * 2.0 ** -24 * 10), float(np.abs(got - want).max())


@pytest.mark.parametrize("kind", ["cache", "batch", "paged"])
def test_prompt_without_memory_changes_nothing(kind, full_device):
    check(kind, full_device)


def test_prompt_without_memory_gives_its_pages_back(full_device):
    """The cache in 4 bits: the tables on the device had taken the prompt's
    pages when the call failed. Every page of the pool is there afterwards."""
    check("q4", full_device)
    m, ids = _model(), synth.prompt_ids(V, N, seed=1)
    kb = m.kv_batch(3, 4096, 70, 4)
    for s in (0, 1):
        kb.prefill(s, ids[:100 + 800 * s], True)  # two pages and fifteen
    kb.prefill(2, ids, True)
    kb.reset(2)
    assert kb.pages() == (53, 70)
    for _ in range(3):
        with pytest.raises(IfxError, match="OutOfMemory"):
            full_device(lambda: kb.prefill(2, ids, False))
        assert kb.pages() == (53, 70) and [kb.len(s) for s in range(3)] == [100, 900, 0]
    kb.prefill(2, synth.prompt_ids(V, 53 * 64, seed=2), True)  # the last page
    assert kb.pages() == (0, 70)
    logits = kb.decode_step_seqs([0, 1], [5, 6])[0]
    kb = m.kv_batch(3, 4096, 70, 4)
    for s in (0, 1):
        kb.prefill(s, ids[:100 + 800 * s], True)
    want = kb.decode_step_seqs([0, 1], [5, 6])[0]
    assert np.all(np.abs(logits - want) <= 4 * 512 * 2.0 ** -24 * 10), float(np.abs(logits - want).max())
