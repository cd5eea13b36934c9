"""Host side of the device-memory operators, without a GPU: refusals of the C entry points (every
check comes before the first CUDA call), layouts of the argument structures, RoPE frequencies."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest

import ops_reference as ref
from conftest import ROOT
from gemma_b200 import native
from gemma_b200.native import GGBlockPlan, GGKv8AppendCall, GGKv8AttentionCall, GGKv8Cache, GGRopeCall, GGRows

P = 4096  # stands for a device pointer: never read


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(native.LIB_PATH):
        import sys
        subprocess.check_call([sys.executable, os.path.join(ROOT, "webgpu-gemma_b200", "build.py")])
    return native.load()


def rows(**kw):
    return GGRows(**dict(dict(data=P, row_stride=1024, head_stride=256, heads=4, type=0), **kw))


def cache(**kw):
    return GGKv8Cache(**dict(dict(k_codes=P, v_codes=P, k_scale=P, v_scale=P, num_blocks=8, block_tokens=16,
                                  kv_heads=4, head_dim=256, code=0), **kw))


def attend(q=None, out=None, **kw):
    return GGKv8AttentionCall(**dict(dict(q=q or rows(), out=out or rows(), cu_rows=P, lens=P, table=P, table_stride=8, workspace=P,
                                          workspace_bytes=1 << 40, scale=0.1, seqs=2, rows=2, max_rows=1, max_len=128), **kw))


def append(lib, c, k, v, slots=P, n=3):
    call = GGKv8AppendCall(k, v, slots, n)
    return lib.gg_kv8_append(ctypes.byref(c), ctypes.byref(call), None)


def refused(lib, rc, *words):
    msg = lib.gg_last_error(None).decode()
    assert rc == native.GG_E_ARG, (rc, msg)
    for w in words:
        assert w in msg, msg


@pytest.mark.parametrize("kw, word", [
    (dict(k_codes=None), "null cache"), (dict(v_scale=P + 4), "16-byte"), (dict(block_tokens=48), "block_tokens 48"),
    (dict(block_tokens=8), "block_tokens"), (dict(head_dim=40), "head_dim 40"), (dict(head_dim=272), "head_dim"),
    (dict(head_dim=0), "head_dim"), (dict(kv_heads=0), "kv_heads"), (dict(num_blocks=0), "num_blocks"),
    (dict(num_blocks=1 << 27, block_tokens=16), "num_blocks"), (dict(code=2), "code 2")])
def test_cache_refused(lib, kw, word):
    c = cache(**kw)
    refused(lib, append(lib, c, rows(), rows()), "gg_kv8_append", word)
    refused(lib, lib.gg_kv8_attention(ctypes.byref(c), ctypes.byref(attend()), None), word)


@pytest.mark.parametrize("kw, word", [
    (dict(data=None), "k.data is null"), (dict(type=3), "k.type 3"), (dict(heads=3), "3"), (dict(heads=0), "heads"),
    (dict(data=P + 2), "aligned"), (dict(row_stride=-1024), "negative"), (dict(head_stride=255), "overlap"),
    (dict(row_stride=255), "overlap"), (dict(type=1), "different types")])
def test_append_rows_refused(lib, kw, word):
    c, v = cache(), rows()
    refused(lib, append(lib, c, rows(**kw), v), word)
    refused(lib, append(lib, c, v, v, n=-1), "rows")
    refused(lib, append(lib, c, v, v, slots=None), "null")
    refused(lib, lib.gg_kv8_append(ctypes.byref(c), None, None), "null")


@pytest.mark.parametrize("kw, qkw, okw, word", [
    (dict(table_stride=7), {}, {}, "table_stride 7"), (dict(seqs=-1), {}, {}, "seqs -1"), (dict(max_len=-1), {}, {}, "max_len"),
    (dict(lens=None), {}, {}, "null array"), ({}, dict(heads=6), dict(heads=6), "6 query heads over 4"), ({}, {}, dict(type=2), "another type"),
    ({}, dict(type=5), {}, "q.type 5"), ({}, dict(heads=4 * 1025), dict(heads=4 * 1025), "1024 query heads"), (dict(window=-1), {}, {}, "window"), (dict(scale=math.nan), {}, {}, "scale"),
    (dict(scale=math.inf), {}, {}, "scale"), (dict(seqs=1 << 20, rows=1 << 20, max_rows=1 << 20), {}, {}, "tiles")])
def test_attention_refused(lib, kw, qkw, okw, word):
    c, call = cache(), attend(rows(**qkw), rows(**okw), **kw)
    refused(lib, lib.gg_kv8_attention(ctypes.byref(c), ctypes.byref(call), None), word)


@pytest.mark.parametrize("n, max_rows", [(2, 1), (300, 300)])
def test_attention_workspace_refused(lib, n, max_rows):
    c, call = cache(), attend(max_len=128 * 16, table_stride=128, rows=n, max_rows=max_rows)
    need = ctypes.c_size_t()
    assert lib.gg_kv8_attention_workspace(ctypes.byref(c), ctypes.byref(call), ctypes.byref(need)) == 0
    assert need.value > 0
    for ws, size in ((P, need.value - 1), (None, need.value), (P + 8, need.value)):
        call.workspace, call.workspace_bytes = ws, size
        refused(lib, lib.gg_kv8_attention(ctypes.byref(c), ctypes.byref(call), None), "workspace")


@pytest.mark.parametrize("kw, word", [
    (dict(head_dim=0), "head_dim"), (dict(rot_dim=3), "rot_dim 3"), (dict(rot_dim=258), "rot_dim"), (dict(rot_dim=0), "rot_dim"),
    (dict(layout=2), "layout"), (dict(rows=-1), "rows"), (dict(positions=None), "null"), (dict(freqs=None), "null"),
    (dict(k_out=rows(data=None)), "null"), (dict(k_out=rows(heads=2)), "heads"), (dict(k_out=rows(type=1)), "another type"),
    (dict(q=rows(type=9)), "q.type 9")])
def test_rope_refused(lib, kw, word):
    call = GGRopeCall(**dict(dict(q=rows(), k=rows(), q_out=rows(), k_out=rows(), positions=P, freqs=P, mscale=1.0, rows=2, head_dim=256,
                                  rot_dim=256), **kw))
    refused(lib, lib.gg_rope(ctypes.byref(call), None), word)


PLAN = dict(old_len=P, new_len=P, table=P, table_stride=8, free_list=P, free_count=P, cu_rows=P, lens=2 * P, row_seq=P,
            positions=P, slots=P, free_count_out=P, status=P, seqs=2, max_blocks=8, block_tokens=16, free_capacity=4, rows=4)


@pytest.mark.parametrize("kw, word", [
    ({n: None}, "null") for n, t in GGBlockPlan._fields_ if t is ctypes.c_void_p] + [
    (dict(seqs=0), "seqs"), (dict(max_blocks=0), "max_blocks"), (dict(rows=-1), "rows"), (dict(free_capacity=-1), "free_capacity"),
    (dict(table_stride=7), "table_stride"), (dict(block_tokens=0), "block_tokens"), (dict(lens=P), "lens")])
def test_plan_refused(lib, kw, word):
    p = GGBlockPlan(**dict(PLAN, **kw))
    refused(lib, lib.gg_plan_blocks(ctypes.byref(p), None), "gg_plan_blocks", word)


def test_rows_of_nothing_are_fine(lib):
    """Zero rows: accepted, and nothing is launched (there is no GPU here)."""
    c, k = cache(), rows()
    assert append(lib, c, k, k, n=0) == 0
    call = GGRopeCall(q=k, q_out=k, positions=P, freqs=P, mscale=1.0, rows=0, head_dim=256, rot_dim=256)
    assert lib.gg_rope(ctypes.byref(call), None) == 0
    assert lib.gg_kv8_attention(ctypes.byref(c), ctypes.byref(attend(rows=0)), None) == 0


def freqs(lib, scaling, rot, theta=1e6, factor=8.0, trained=8192.0, low=1.0, high=4.0):
    f, m = np.zeros(max(rot // 2, 1)), ctypes.c_double()
    rc = lib.gg_rope_freqs(scaling, rot, theta, factor, trained, low, high, f.ctypes.data_as(ctypes.c_void_p), ctypes.byref(m))
    return rc, f, m.value


@pytest.mark.parametrize("rot", [2, 64, 96, 256])
def test_frequencies(lib, rot):
    i = np.arange(rot // 2)
    w = 1e6 ** (-2.0 * i / rot)
    rc, f, m = freqs(lib, native.GG_ROPE_NONE, rot)
    assert rc == 0 and m == 1.0
    np.testing.assert_allclose(f, w, rtol=1e-14)
    rc, f, m = freqs(lib, native.GG_ROPE_LINEAR, rot)
    assert rc == 0 and m == 1.0
    np.testing.assert_allclose(f, w / 8, rtol=1e-14)
    # bands: a turn of less than trained / high positions is kept, one of more than trained / low is stretched
    rc, f, m = freqs(lib, native.GG_ROPE_BANDS, rot)
    assert rc == 0 and m == 1.0
    for x, y in zip(f, w):
        turn = 2 * math.pi / y
        t = 1.0 if turn < 8192 / 4 else 0.0 if turn > 8192 / 1 else (8192 / turn - 1) / 3
        assert x == pytest.approx((1 - t) * y / 8 + t * y, rel=1e-13)
    # yarn: pairs that turn 32 times or more in the trained positions are kept, once or less stretched
    rc, f, m = freqs(lib, native.GG_ROPE_YARN, rot, trained=32768.0, low=1.0, high=32.0)
    assert rc == 0 and m == pytest.approx(0.1 * math.log(8.0) + 1, rel=1e-15)
    turns = 32768 * w / (2 * math.pi)
    pair = lambda n: rot * math.log(32768 / (n * 2 * math.pi)) / (2 * math.log(1e6))  # noqa: E731
    lo, hi = max(0, math.floor(pair(32))), min(rot - 1, math.ceil(pair(1)))
    for j, (x, y) in enumerate(zip(f, w)):
        t = 1.0 if j <= lo else 0.0 if j >= hi else 1 - (j - lo) / (hi - lo)
        assert x == pytest.approx(t * y + (1 - t) * y / 8, rel=1e-13)
    if rot >= 64:
        assert turns[0] > 32 and f[0] == pytest.approx(w[0]) and f[-1] == pytest.approx(w[-1] / 8)


@pytest.mark.parametrize("kw, word", [(dict(rot=3), "rot_dim"), (dict(rot=0), "rot_dim"), (dict(theta=1.0), "theta"), (dict(theta=math.nan), "theta"),
                                      (dict(factor=0.0), "factor"), (dict(low=4.0), "low < high"), (dict(trained=0.0), "trained")])
def test_frequencies_refused(lib, kw, word):
    rc, _, _ = freqs(lib, native.GG_ROPE_YARN, **dict(dict(rot=64), **kw))
    refused(lib, rc, word)
    assert freqs(lib, 7, 64)[0] == native.GG_E_ARG


def test_structures_match_the_header(tmp_path):
    structs = {"gg_rows": GGRows, "gg_block_plan": GGBlockPlan, "gg_kv8_cache": GGKv8Cache,
               "gg_rope_call": GGRopeCall, "gg_kv8_append_call": GGKv8AppendCall, "gg_kv8_attention_call": GGKv8AttentionCall}
    consts = ["GG_T_F32", "GG_T_BF16", "GG_T_F16", "GG_ROPE_HALF", "GG_ROPE_INTERLEAVED", "GG_ROPE_NONE", "GG_ROPE_LINEAR",
              "GG_ROPE_BANDS", "GG_ROPE_YARN", "GG_KV8_INT8", "GG_KV8_E4M3", "GG_PLAN_OK", "GG_PLAN_NO_BLOCKS", "GG_PLAN_TOO_LONG",
              "GG_PLAN_NO_ROWS", "GG_PLAN_BAD_LENGTH", "GG_PLAN_BAD_STACK"]
    lines = ["#include <stdio.h>", '#include "gemma_b200.h"', "int main(void) {"]
    for n, c in structs.items():
        lines.append(f'  printf("{n} %zu\\n", sizeof({n}));')
        lines += [f'  printf("{n}.{f} %zu\\n", offsetof({n}, {f}));' for f, _ in c._fields_]
    lines += [f'  printf("{c} %d\\n", (int)({c}));' for c in consts] + ["  return 0;", "}"]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines) + "\n")
    subprocess.check_call(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")])
    got = dict(ln.rsplit(" ", 1) for ln in subprocess.check_output([str(tmp_path / "layout")], text=True).splitlines())
    for n, c in structs.items():
        assert int(got[n]) == ctypes.sizeof(c), n
        for f, _ in c._fields_:
            assert int(got[f"{n}.{f}"]) == getattr(c, f).offset, (n, f)
    for c in consts:
        assert int(got[c]) == getattr(native, c), c
    # the packed forms that gemma_b200.ops hands over
    ops = pytest.importorskip("gemma_b200.ops")
    n = range(1, 100)
    for pack, c, count in ((ops._pack_plan, GGBlockPlan, 18), (ops._pack_rope, GGRopeCall, 28), (ops._pack_append, GGKv8AppendCall, 12),
                           (ops._pack_attend, GGKv8AttentionCall, 23)):
        raw = pack(*n[:count])
        assert len(raw) == ctypes.sizeof(c)
        flat = []
        for f, t in c._fields_:
            v = getattr(c.from_buffer_copy(raw), f)
            flat += [getattr(v, g) for g, _ in GGRows._fields_] if t is GGRows else [v]
        assert flat == list(n[:count]), c


def test_reference_codes():
    """The tests' own encoder: every e4m3 code survives a round trip, ties go to even, zero keeps its sign."""
    codes = np.array([c for c in range(256) if c & 127 != 127], np.uint8)
    assert np.array_equal(ref.encode(ref.decode(codes, "e4m3"), "e4m3"), codes)
    v = ref.E4M3[:127]
    mid = (v[1:] + v[:-1]) / 2
    assert np.all(ref.encode(mid, "e4m3") % 2 == 0)
    assert ref.decode(ref.encode(np.array([2.5, -3.5, 127.0]), "int8"), "int8").tolist() == [2.0, -4.0, 127.0]
    torch = pytest.importorskip("torch")
    x = np.random.default_rng(1).standard_normal(4096) * 60
    x = x[np.abs(x) <= 448].astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(ref.encode(x.astype(np.float64), "e4m3"), want)


def test_torch_wrappers_refuse_cpu_tensors(lib):
    torch = pytest.importorskip("torch")
    from gemma_b200 import ops
    z = torch.zeros(2, 1, 16, 32, dtype=torch.int8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.KV8Cache(z, z, torch.ones(2, 1), torch.ones(2, 1))
    with pytest.raises(ValueError, match="CUDA"):
        ops.rope(torch.zeros(2, 1, 32), None, torch.zeros(2, dtype=torch.int32), torch.zeros(16, dtype=torch.float64))
    with pytest.raises(ValueError, match="scaling"):
        ops.rope_frequencies(64, 1e4, "cubic", device="cpu")
    f, m = ops.rope_frequencies(64, 1e4, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,) and m == 1.0


def test_q8_cache_flag(lib):
    """GG_FLAG_KV_Q8 goes with neither the bf16 cache nor serial prefill (checked before any device)."""
    from gemma_b200 import config, synth
    cfg = synth.SHAPES["tiny"].config()
    cfg.kv_dtype = "q8"
    assert config.kv_flags(cfg) == config.GG_FLAG_KV_Q8 == 4
    for flags in (config.GG_FLAG_KV_BF16, native.GG_FLAG_SERIAL_PREFILL):
        h = ctypes.c_void_p()
        assert lib.gg_create(ctypes.byref(config.to_cconfig(cfg, flags=flags)), 0, ctypes.byref(h)) == native.GG_E_ARG
        assert b"GG_FLAG_KV_Q8" in lib.gg_last_error(None)
    cfg.kv_dtype = "q4"
    with pytest.raises(ValueError, match="q8"):
        config.kv_flags(cfg)
