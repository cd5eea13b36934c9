"""Sizes at the edge of what the operators take, on the host: refusals and workspaces, without a GPU."""
import ctypes
import math
import subprocess
import sys

import pytest

from conftest import ROOT
from gemma_b200 import native
from test_ops_host import attend, cache, freqs, lib, rows  # noqa: F401 (lib is a fixture)

HUGE = """
import ctypes, sys
sys.path[:0] = [{root!r} + "/webgpu-gemma_b200", {root!r} + "/tests"]
from gemma_b200 import native
from test_ops_host import attend, cache, rows
lib = native.load()
for seqs in (0, 1, 2):
    for max_rows in (1 << 21, 1 << 29, 1 << 30, (1 << 31) - 1):
        c, need = cache(kv_heads={kv}, head_dim=128), ctypes.c_size_t()
        call = attend(rows(heads={heads}), rows(heads={heads}), seqs=seqs, max_rows=max_rows)
        print(seqs * max_rows * {heads}, lib.gg_kv8_attention_workspace(ctypes.byref(c), ctypes.byref(call), ctypes.byref(need)),
              lib.gg_kv8_attention(ctypes.byref(c), ctypes.byref(call), None), lib.gg_last_error(None).decode(), flush=True)
"""


@pytest.mark.parametrize("kv, heads", [(1, 1024), (64, 65472), (8, 8)])
def test_attention_of_too_many_rows_refused(lib, kv, heads):  # noqa: F811
    """Refused, not computed with tile counts that have wrapped around (in a process of its own: an
    integer division by zero ends it)."""
    r = subprocess.run([sys.executable, "-c", HUGE.format(root=ROOT, kv=kv, heads=heads)], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stdout[-300:], r.stderr[-300:])
    lines = r.stdout.splitlines()
    assert len(lines) == 12
    for ln in lines:
        total, rc, rc2, *msg = ln.split(" ", 3)
        if int(total) >= 2 ** 31 - 1:
            assert (int(rc), int(rc2)) == (native.GG_E_ARG, native.GG_E_ARG) and "tiles" in msg[0]
        elif int(total) == 0:
            assert (int(rc), int(rc2)) == (0, 0)


@pytest.mark.parametrize("type_", [0, 1])
@pytest.mark.parametrize("kv, group, dim", [(1, 4, 256), (8, 4, 128), (2, 1, 64)])
def test_attention_workspace_grows_with_the_length(lib, type_, kv, group, dim):  # noqa: F811
    """A workspace for the longest context is enough for every shorter one (what holds one for many calls
    sizes it once)."""
    c, need = cache(kv_heads=kv, head_dim=dim, num_blocks=1 << 16), ctypes.c_size_t()
    for seqs, max_rows, window in ((1, 1, 0), (1, 500, 0), (3, 70, 0), (1, 40, 700), (64, 1, 0), (2, 9, 5000)):
        last = 0
        for max_len in list(range(0, 40000, 16)) + list(range(40000, 140000, 1000)):
            call = attend(rows(heads=kv * group, type=type_), seqs=seqs, rows=seqs * max_rows, max_rows=max_rows, max_len=max_len, window=window)
            assert lib.gg_kv8_attention_workspace(ctypes.byref(c), ctypes.byref(call), ctypes.byref(need)) == 0
            assert need.value >= last, (seqs, max_rows, window, max_len)
            last = need.value
        assert last > 0


def test_gradients_of_either_mode_are_refused():
    """A tensor that requires a gradient, and a dual tensor, whose requires_grad is False."""
    torch = pytest.importorskip("torch")
    from torch.autograd import forward_ad
    from gemma_b200 import ops
    x = torch.zeros(2, 1, 32)
    assert ops._rows("q", x, -1)[3] == 1  # (-1: where a CPU tensor is; the wrappers never come here with one)
    with pytest.raises(ValueError, match="gradient"):
        ops._rows("q", x.clone().requires_grad_(), -1)
    with torch.no_grad():
        ops._rows("q", x.clone().requires_grad_(), -1)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="tangent"):
            ops._rows("q", forward_ad.make_dual(x, torch.ones_like(x)), -1)
        ops._rows("q", x, -1)


@pytest.mark.parametrize("factor", [0.25, 0.5, 1.0, 1.0000001, 4.0])
def test_yarn_never_shrinks_the_rotation(lib, factor):  # noqa: F811
    """cos and sin are lengthened where a context is stretched, and left alone where it is not."""
    rc, f, m = freqs(lib, native.GG_ROPE_YARN, 64, factor=factor, trained=32768.0, low=1.0, high=32.0)
    assert rc == 0 and m == (pytest.approx(0.1 * math.log(factor) + 1, rel=1e-15) if factor > 1 else 1.0)
    assert f[0] == pytest.approx(1.0, rel=1e-15) and f[-1] == pytest.approx(1e6 ** (-62 / 64) / factor, rel=1e-13)


@pytest.mark.parametrize("at, name", [(7, "requests"), (8, "rows"), (9, "max_rows"), (10, "max_len"), (11, "window")])
@pytest.mark.parametrize("value", [1 << 31, (1 << 32) + 1, -(1 << 31) - 1, 1 << 70])
def test_sizes_beyond_32_bits_refused(lib, at, name, value):  # noqa: F811
    """Not cut to their low bits on the way into the library."""
    ops = pytest.importorskip("gemma_b200.ops")
    sizes = [8, 16, 1, 64, native.GG_KV8_INT8, 4, native.GG_T_F32, 1, 1, 1, 100, 0]
    assert ops._attend_bytes(*sizes) >= 0
    sizes[at] = value
    with pytest.raises(ValueError, match=f"{name} {value} does not fit"):
        ops._attend_bytes(*sizes)
