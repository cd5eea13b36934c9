"""The 8-bit KV cache of the engine (GG_FLAG_KV_Q8, GemmaConfig.kv_dtype = "q8") against a plain
64-bit forward that quantises every block of 16 tokens as gg_kv8_append does (ops_reference).

The engine's own f32 roundings differ from the reference's as in test_gpu_parity.py, hence its
logit tolerance of 2e-3 relative L2. A value within those roundings (1e-5) of the middle between
two codes may be stored one code apart; at 1e-5 of a step's width per value that is one value in
1e4 moved by 1/64 of its block's largest, far inside the tolerance.
"""
import dataclasses

import numpy as np
import pytest

import ops_reference as ref
from conftest import rel_l2, synthetic

pytestmark = pytest.mark.gpu

LOGIT_TOL = 2e-3
B = 16


def dequant(dims, raw):
    K, M = int(dims[0]), int(dims[1])
    blocks = np.frombuffer(raw, np.uint8).reshape(M, K // 32, 34)
    d = blocks[:, :, :2].copy().view(np.float16).astype(np.float64)
    return (blocks[:, :, 2:].copy().view(np.int8).astype(np.float64) * d).reshape(M, K)


class Reference:
    """One conversation, 64 bits; tokens() appends rows as one call of the engine does."""

    def __init__(self, cfg, tens):
        self.c = cfg
        get = lambda n: np.frombuffer(tens[n][2], np.float32).astype(np.float64)  # noqa: E731
        self.embd = dequant(tens["token_embd.weight"][0], tens["token_embd.weight"][2])
        self.out_norm = get("output_norm.weight")
        self.layers = []
        for i in range(cfg.num_layers):
            w = {}
            for n in ("attn_q", "attn_k", "attn_v", "attn_output", "ffn_gate", "ffn_up", "ffn_down"):
                dims, _, raw = tens[f"blk.{i}.{n}.weight"]
                w[n] = dequant(dims, raw)
            for n in ("attn_norm", "ffn_norm", "attn_q_norm", "attn_k_norm", "post_attention_norm", "post_ffw_norm"):
                w[n] = get(f"blk.{i}.{n}.weight")
            nb = -(-cfg.context_length // B)
            w["codes"] = [np.zeros((nb, cfg.num_kv_heads, B, cfg.head_dim), np.uint8) for _ in range(2)]
            w["scale"] = [np.zeros((nb, cfg.num_kv_heads)) for _ in range(2)]
            self.layers.append(w)

    def norm(self, x, w):
        return x * w / np.sqrt((x * x).mean(-1, keepdims=True) + self.c.rms_norm_eps)

    def tokens(self, ids, p0):
        """Runs ids at positions p0..; returns the last one's logits."""
        c = self.c
        T, H, D, G = len(ids), c.num_q_heads, c.head_dim, c.num_q_heads // c.num_kv_heads
        pos = np.arange(p0, p0 + T)
        h = self.embd[list(ids)] * np.sqrt(np.float64(c.hidden_size))
        for i, w in enumerate(self.layers):
            local = (i % c.swa_period) < c.swa_period - 1
            freqs = np.float64(c.rope_theta_swa if local else c.rope_theta_global) ** (-2.0 * np.arange(D // 2) / D)
            x = self.norm(h, w["attn_norm"])
            q = self.norm((x @ w["attn_q"].T).reshape(T, H, D), w["attn_q_norm"])
            k = self.norm((x @ w["attn_k"].T).reshape(T, -1, D), w["attn_k_norm"])
            v = (x @ w["attn_v"].T).reshape(T, -1, D)
            q, k = (ref.rope(y, pos, freqs, "half", 1.0, False) for y in (q, k))
            for which, y in enumerate((k, v)):
                ref.append(w["codes"][which], w["scale"][which], y.astype(np.float32), list(pos), "int8")
            rows = [(ref.decode(w["codes"][j], "int8") * w["scale"][j][:, :, None, None]).transpose(0, 2, 1, 3).reshape(-1, c.num_kv_heads, D)
                    for j in range(2)]
            att = np.zeros((T, H, D))
            for t, p in enumerate(pos):
                lo = max(0, p - c.sliding_window + 1) if local and c.sliding_window else 0
                for j in range(H):
                    z = rows[0][lo:p + 1, j // G] @ q[t, j] / np.sqrt(D)
                    z = np.exp(z - z.max())
                    att[t, j] = z @ rows[1][lo:p + 1, j // G] / z.sum()
            h = h + self.norm(att.reshape(T, -1) @ w["attn_output"].T, w["post_attention_norm"])
            x = self.norm(h, w["ffn_norm"])
            g, u = x @ w["ffn_gate"].T, x @ w["ffn_up"].T
            t_ = np.clip(0.7978845608028654 * g * (1 + 0.044715 * g * g), -15, 15)
            h = h + self.norm((0.5 * g * (1 + np.tanh(t_)) * u) @ w["ffn_down"].T, w["post_ffw_norm"])
        return self.norm(h[-1], self.out_norm) @ self.embd.T


def _q8(shape, seed, **kw):
    cfg, tens = synthetic(shape, seed)
    return dataclasses.replace(cfg, kv_dtype="q8", **kw), tens


def near_argmax(logits, tok):
    return logits[tok] >= logits.max() - 4 * LOGIT_TOL * np.abs(logits).max()


@pytest.mark.parametrize("shape, seed, plen, window", [("small", 3, 41, 0), ("mid", 5, 530, 0), ("small", 9, 45, 16)])
def test_prefill_and_steps(shape, seed, plen, window):
    from gemma_b200 import synth
    from gemma_b200.native import engine_from_tensors
    extra = dict(sliding_window=window, rope_theta_swa=10000.0, swa_period=2) if window else {}
    cfg, tens = _q8(shape, seed, **extra)
    eng, want = engine_from_tensors(cfg, tens), Reference(cfg, tens)
    prompt = [int(t) for t in synth.make_prompt(seed, plen, cfg.vocab_size)]
    eng.prefill(prompt, 0)
    for c0 in range(0, plen, 512):  # the engine's prompt chunks
        lg = want.tokens(prompt[c0:c0 + 512], c0)
    tok = eng.sample_last(0)
    assert rel_l2(eng.logits(), lg) < LOGIT_TOL and near_argmax(lg, tok)
    pos = plen
    for _ in range(20):
        nxt = eng.step(tok, pos)
        lg = want.tokens([tok], pos)
        assert rel_l2(eng.logits(), lg) < LOGIT_TOL and near_argmax(lg, nxt)
        tok, pos = nxt, pos + 1
    for layer in (0, cfg.num_layers - 1):
        for which in (0, 1):
            w = want.layers[layer]
            for p in (0, plen - 1, pos - 1):
                row = eng.kv_row(layer, p, which)
                sc = w["scale"][which][p // B]
                ref_row = ref.decode(w["codes"][which][p // B, :, p % B], "int8") * sc[:, None]
                # equal codes, but for values at the middle of a step
                assert np.abs(row - ref_row.ravel()).max() <= sc.max()
                assert np.mean(row != ref_row.ravel()) < 0.05
    # chained decode gives the tokens of single steps (same batch of one, same kernels)
    eng.prefill(prompt, 0)
    first = eng.sample_last(0)
    chain = eng.decode(first, plen, 6)
    eng.prefill(prompt, 0)
    assert eng.sample_last(0) == first
    one, p = [], plen
    for _ in range(6):
        one.append(eng.step(one[-1] if one else first, p))
        p += 1
    assert list(chain) == one
    eng.close()


def test_batched_decode():
    from gemma_b200 import synth
    from gemma_b200.native import engine_from_tensors
    cfg, tens = _q8("small", 7)
    n, steps = 3, 18  # past the end of a block of 16
    prompts = [[int(t) for t in synth.make_prompt(80 + i, 15 + 9 * i, cfg.vocab_size)] for i in range(n)]
    eng = engine_from_tensors(cfg, tens, max_seqs=n + 1)
    slots = [2, 0, 3]
    first = []
    for s, p in zip(slots, prompts):
        eng.prefill(p, 0, seq=s)
        first.append(eng.sample_last(s))
    got = eng.decode_batch(slots, first, [len(p) for p in prompts], steps, [(0.0, 0.9, 1.0)] * n, np.zeros((steps, n)))
    for i, p in enumerate(prompts):
        want = Reference(cfg, tens)
        lg = want.tokens(p, 0)
        assert near_argmax(lg, first[i])
        tok = first[i]
        for k in range(steps):
            lg = want.tokens([tok], len(p) + k)
            assert near_argmax(lg, got[k, i]), (i, k)
            tok = int(got[k, i])
    eng.close()


def test_going_back_and_refusals():
    """A call may start below the slot's length (later tokens are dropped), not beyond it; reset
    starts over; gg_get_hidden and mixed flags are refused."""
    from gemma_b200 import synth
    from gemma_b200.native import GG_FLAG_SERIAL_PREFILL, GemmaB200Error, engine_from_tensors
    cfg, tens = _q8("tiny", 7)
    prompt = [int(t) for t in synth.make_prompt(7, 37, cfg.vocab_size)]
    eng, want = engine_from_tensors(cfg, tens), Reference(cfg, tens)
    with pytest.raises(GemmaB200Error, match="beyond the 0 tokens"):
        eng.prefill(prompt, 1)
    eng.prefill(prompt, 0)
    want.tokens(prompt, 0)
    with pytest.raises(GemmaB200Error, match="beyond the 37 tokens"):
        eng.step(5, 38)
    eng.prefill(prompt[:9], 21)
    lg = want.tokens(prompt[:9], 21)
    eng.sample_last(0)
    assert rel_l2(eng.logits(), lg) < LOGIT_TOL
    eng.step(11, 30)
    assert rel_l2(eng.logits(), want.tokens([11], 30)) < LOGIT_TOL
    with pytest.raises(GemmaB200Error, match="beyond the 31 tokens"):
        eng.decode_batch([0], [3], [33], 1, [(0.0, 0.9, 1.0)], np.zeros((1, 1)))
    with pytest.raises(GemmaB200Error, match="hidden"):
        eng.hidden()
    eng.reset_kv(0)
    with pytest.raises(GemmaB200Error, match="beyond the 0 tokens"):
        eng.step(5, 1)
    eng.prefill(prompt, 0)
    eng.sample_last(0)
    assert rel_l2(eng.logits(), Reference(cfg, tens).tokens(prompt, 0)) < LOGIT_TOL
    eng.close()
    with pytest.raises(GemmaB200Error, match="SERIAL_PREFILL"):
        engine_from_tensors(cfg, tens, flags=GG_FLAG_SERIAL_PREFILL)


def test_user_path():
    from gemma_b200.engine import create_gemma_engine
    eng = create_gemma_engine(model="synthetic:tiny", context_length=256, kv_dtype="q8", random=lambda: 0.3)
    out = []
    for text in ("hello", "and again"):
        eng.add_user_message(text)
        out.append(list(eng.generate(max_tokens=6, temperature=0.0, rep_penalty=1.0)))
    assert all(out) and eng.kv_position > 0
    eng.dispose()
