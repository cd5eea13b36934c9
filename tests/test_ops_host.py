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
from gemma_b200.native import GGBlockPlan, GGKv8Batch, GGKv8Cache, GGRows

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


def batch(**kw):
    return GGKv8Batch(**dict(dict(cu_rows=P, lens=P, table=P, table_stride=8, seqs=2, rows=2, max_rows=1, max_len=128), **kw))


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
    k = rows()
    c = cache(**kw)
    refused(lib, lib.gg_kv8_append(ctypes.byref(c), ctypes.byref(k), ctypes.byref(k), P, 3, None), "gg_kv8_append", word)
    q, b = rows(), batch()
    refused(lib, lib.gg_kv8_attention(ctypes.byref(c), ctypes.byref(q), ctypes.byref(q), None, ctypes.byref(b), 0.1, 0, P, 1 << 30, None), word)


@pytest.mark.parametrize("kw, word", [
    (dict(data=None), "k.data is null"), (dict(type=3), "k.type 3"), (dict(heads=3), "3"), (dict(heads=0), "heads"),
    (dict(data=P + 2), "aligned"), (dict(row_stride=-1024), "negative"), (dict(head_stride=255), "overlap"),
    (dict(row_stride=255), "overlap"), (dict(type=1), "different types")])
def test_append_rows_refused(lib, kw, word):
    c, k, v = cache(), rows(**kw), rows()
    refused(lib, lib.gg_kv8_append(ctypes.byref(c), ctypes.byref(k), ctypes.byref(v), P, 3, None), word)
    refused(lib, lib.gg_kv8_append(ctypes.byref(c), ctypes.byref(v), ctypes.byref(v), P, -1, None), "rows")
    refused(lib, lib.gg_kv8_append(ctypes.byref(c), None, ctypes.byref(v), P, 3, None), "null")
    refused(lib, lib.gg_kv8_append(ctypes.byref(c), ctypes.byref(v), ctypes.byref(v), None, 3, None), "null")


@pytest.mark.parametrize("bkw, qkw, okw, window, scale, word", [
    (dict(table_stride=7), {}, {}, 0, 0.1, "table_stride 7"), (dict(seqs=-1), {}, {}, 0, 0.1, "seqs -1"),
    (dict(max_len=-1), {}, {}, 0, 0.1, "max_len"), (dict(lens=None), {}, {}, 0, 0.1, "null array"),
    ({}, dict(heads=6), dict(heads=6), 0, 0.1, "6 query heads over 4"), ({}, {}, dict(type=2), 0, 0.1, "another type"),
    ({}, {}, {}, -1, 0.1, "window"), ({}, {}, {}, 0, math.nan, "scale"), ({}, {}, {}, 0, math.inf, "scale"),
    (dict(seqs=1 << 20, rows=1 << 20, max_rows=1 << 20), {}, {}, 0, 0.1, "tiles")])
def test_attention_refused(lib, bkw, qkw, okw, window, scale, word):
    c, q, o, b = cache(), rows(**qkw), rows(**okw), batch(**bkw)
    refused(lib, lib.gg_kv8_attention(ctypes.byref(c), ctypes.byref(q), ctypes.byref(o), None, ctypes.byref(b), scale, window,
                                      P, 1 << 40, None), word)


def test_attention_workspace_refused(lib):
    c, q, b = cache(), rows(), batch(max_len=128 * 16, table_stride=128)
    need = ctypes.c_size_t()
    assert lib.gg_kv8_attention_workspace(ctypes.byref(c), ctypes.byref(q), ctypes.byref(b), 0, ctypes.byref(need)) == 0
    assert need.value > 0
    call = lambda ws, n: lib.gg_kv8_attention(ctypes.byref(c), ctypes.byref(q), ctypes.byref(q), None, ctypes.byref(b), 0.1, 0, ws, n, None)  # noqa: E731
    refused(lib, call(P, need.value - 1), "workspace")
    refused(lib, call(None, need.value), "workspace")
    refused(lib, call(P + 8, need.value), "workspace")


@pytest.mark.parametrize("kw, word", [
    (dict(head_dim=0), "head_dim"), (dict(rot=3), "rot_dim 3"), (dict(rot=258), "rot_dim"), (dict(rot=0), "rot_dim"),
    (dict(layout=2), "layout"), (dict(rows=-1), "rows"), (dict(pos=None), "null"), (dict(freqs=None), "null"),
    (dict(k_out=None), "null"), (dict(ko=dict(heads=2)), "heads"), (dict(ko=dict(type=1)), "another type")])
def test_rope_refused(lib, kw, word):
    q, k, ko = rows(), rows(), rows(**kw.get("ko", {}))
    k_out = ctypes.byref(ko) if kw.get("k_out", 1) else None
    refused(lib, lib.gg_rope(ctypes.byref(q), ctypes.byref(k), ctypes.byref(q), k_out, kw.get("rows", 2), kw.get("head_dim", 256),
                             kw.get("rot", 256), kw.get("layout", 0), kw.get("pos", P), kw.get("freqs", P), 1.0, 0, None), word)


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
    c, k, b = cache(), rows(), batch(rows=0)
    assert lib.gg_kv8_append(ctypes.byref(c), ctypes.byref(k), ctypes.byref(k), P, 0, None) == 0
    assert lib.gg_rope(ctypes.byref(k), None, ctypes.byref(k), None, 0, 256, 256, 0, P, P, 1.0, 0, None) == 0
    assert lib.gg_kv8_attention(ctypes.byref(c), ctypes.byref(k), ctypes.byref(k), None, ctypes.byref(b), 0.1, 0, None, 0, None) == 0


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
    structs = {"gg_rows": GGRows, "gg_block_plan": GGBlockPlan, "gg_kv8_cache": GGKv8Cache, "gg_kv8_batch": GGKv8Batch}
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
