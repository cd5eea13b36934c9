"""Sizes at the edge of what the operators take, on the host: refusals and workspaces, without a GPU."""
import subprocess
import sys

import pytest

from conftest import ROOT
from gemma_b200 import native
from test_ops_host import lib  # noqa: F401 (a fixture)

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
        rows, rc, rc2, *msg = ln.split(" ", 3)
        if int(rows) >= 2 ** 31 - 1:
            assert (int(rc), int(rc2)) == (native.GG_E_ARG, native.GG_E_ARG) and "tiles" in msg[0]
        elif int(rows) == 0:
            assert (int(rc), int(rc2)) == (0, 0)
