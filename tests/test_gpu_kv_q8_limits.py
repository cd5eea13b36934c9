"""The engine's 8-bit KV cache where a call ends early or a context grows long (see test_gpu_kv_q8.py)."""
import numpy as np
import pytest

from test_gpu_kv_q8 import _q8

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
