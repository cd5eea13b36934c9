"""The device-memory operators at the limits of their calls: sizes that cut a batch short, lengths
beyond one tile or range, scales and slots at the edge of what a cache may hold. References and tolerances are
those of test_gpu_ops.py."""
import numpy as np
import pytest

from test_gpu_ops import check_attend, make_batch

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# ------------------------------------------------------------------------- batches cut short

@pytest.mark.parametrize("code, dtype, D, H, G, window, max_rows", [
    ("int8", "f32", 256, 1, 4, 512, 1), ("e4m3", "bf16", 128, 8, 4, 1024, 1), ("int8", "f16", 64, 2, 2, 1100, 5), ("int8", "f32", 64, 1, 1, 0, 2)])
def test_attend_window_of_cut_requests(code, dtype, D, H, G, window, max_rows):
    """max_rows below the rows of a request whose window is cut into parts: its keys end with the last row
    that is computed, and the requests behind it have their results."""
    rng = np.random.default_rng(D + window)
    rows, lens = [1500, 1, 40], [1900, 2600, 1300]
    a = make_batch(rng, rows, lens, 16, H, D, code)
    check_attend(rng, rows, lens, H * G, *a, code, dtype, window=window, max_rows=max_rows)
    assert a[0].workspace_bytes(torch.empty(1541, H * G, D, device="cuda"), 3, max_rows, 2600, window) > 0  # (the units are cut)
