"""The engine's 8-bit KV cache where a call ends early or a context grows long (see test_gpu_kv_q8.py)."""
import numpy as np
import pytest

from conftest import rel_l2
from test_gpu_kv_q8 import LOGIT_TOL, Reference, _q8

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_no_allocation_after_the_first_call():
    """Prompts, single steps and batches of any length work in what gg_finalize (and the first batched call)
    allocated."""
    from gemma_b200 import synth
    from gemma_b200.native import engine_from_tensors
    cfg, tens = _q8("mid", 5, sliding_window=300, swa_period=2)
    n = 40
    eng = engine_from_tensors(cfg, tens, max_seqs=n)
    prompt = [int(t) for t in synth.make_prompt(5, 1000, cfg.vocab_size)]
    eng.seen_add(prompt)  # (the buffer of token ids grows with the longest list)
    free = []
    for length in (1, 9, 100, 500, 1000):
        for s in range(n):
            eng.prefill(prompt[:length], 0, seq=s)
        eng.decode_batch(list(range(n)), [7] * n, [length] * n, 20, [(0.0, 0.9, 1.0)] * n, np.zeros((20, n)))
        torch.cuda.synchronize()
        free.append(torch.cuda.mem_get_info()[0])
    assert free == free[:1] * 5
    eng.close()


def test_a_failed_call_drops_the_tokens_it_replaced():
    """A prefill, a step or a batch that starts below the slot's length and fails has replaced some of the
    later tokens: the slot then ends where that call started, and goes on from there."""
    from gemma_b200 import synth
    from gemma_b200.native import GemmaB200Error, engine_from_tensors
    cfg, tens = _q8("tiny", 7)
    prompt = [int(t) for t in synth.make_prompt(7, 60, cfg.vocab_size)]
    eng, want = engine_from_tensors(cfg, tens, max_seqs=2), Reference(cfg, tens)
    eng.prefill(prompt, 0)
    want.tokens(prompt, 0)
    eng.selftest_fail()
    with pytest.raises(GemmaB200Error, match="timed out"):
        eng.prefill(prompt[:9], 41)
    with pytest.raises(GemmaB200Error, match="beyond the 41 tokens"):
        eng.step(5, 50)
    eng.prefill(prompt[:9], 41)
    lg = want.tokens(prompt[:9], 41)
    eng.sample_last(0)
    assert rel_l2(eng.logits(), lg) < LOGIT_TOL
    eng.prefill(prompt, 0, seq=1)
    eng.selftest_fail()
    with pytest.raises(GemmaB200Error, match="timed out"):
        eng.decode_batch([1, 0], [3, 4], [30, 50], 2, [(0.0, 0.9, 1.0)] * 2, np.zeros((2, 2)))
    for seq, n in ((0, 50), (1, 30)):
        with pytest.raises(GemmaB200Error, match=f"beyond the {n} tokens of slot {seq}"):
            eng.step(5, n + 1, seq=seq)
    eng.selftest_fail()
    with pytest.raises(GemmaB200Error, match="timed out"):
        eng.step(5, 47)
    with pytest.raises(GemmaB200Error, match="beyond the 47 tokens"):
        eng.step(5, 48)
    want.tokens([5], 47)  # (it may have raised its block's scale)
    eng.step(11, 47)
    assert rel_l2(eng.logits(), want.tokens([11], 47)) < LOGIT_TOL
    eng.close()


def test_attention_wait_that_runs_out_is_reported():
    """The prompt attention's own wait ends after its limit and sets the engine's error word; the engine goes on."""
    from gemma_b200 import synth
    from gemma_b200.native import GG_E_DEVICE, engine_from_tensors
    cfg, tens = _q8("tiny", 7)
    eng, want = engine_from_tensors(cfg, tens), Reference(cfg, tens)
    assert eng.selftest_wait(20_000_000) == GG_E_DEVICE
    assert "activation wait timed out" in eng.last_error() and "ring wait timed out" in eng.last_error()
    prompt = [int(t) for t in synth.make_prompt(7, 50, cfg.vocab_size)]
    eng.prefill(prompt, 0)
    eng.sample_last(0)
    assert rel_l2(eng.logits(), want.tokens(prompt, 0)) < LOGIT_TOL
    eng.close()
