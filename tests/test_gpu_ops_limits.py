"""The device-memory operators at the limits of their calls: sizes that cut a batch short, lengths
beyond one tile or range, scales and slots at the edge of what a cache may hold. References and tolerances are
those of test_gpu_ops.py."""
import math

import numpy as np
import pytest

import ops_reference as ref
from test_gpu_ops import DT, HALF_EPS, check_attend, dev, f64, make_batch, new_cache, raw

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


# ------------------------------------------------------------------------- scales of any size in a started block

def append_reference(raws, scales, x, slots, code):
    """ref.append for started blocks whose old scale is any positive number: one run, all in 64 bits."""
    B, top = raws.shape[2], ref.TOP[code]
    blk, first = slots[0] // B, min(s % B for s in slots)
    for h in range(raws.shape[1]):
        amax, old = np.abs(x[:, h]).max(), scales[blk, h]
        need = max(amax / top, 2.0 ** -60, old if first > 0 else 0.0)
        e = math.floor(math.log2(need))
        e += 2.0 ** e < need
        if e > 127:  # no f32 holds it
            scales[blk, h], raws[blk, h, [s % B for s in slots]] = math.nan, 0
            continue
        if first > 0 and old != 2.0 ** e:
            raws[blk, h, :first] = ref.encode(ref.decode(raws[blk, h, :first], code) * (old / 2.0 ** e), code)
        scales[blk, h] = 2.0 ** e
        for r, s in enumerate(slots):
            raws[blk, h, s % B] = ref.encode(x[r, h] * 2.0 ** -e, code)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("size", [0.001, 1.0, 300.0])
def test_append_to_scales_of_any_size(code, size):
    """An old scale that is no power of two, or below or above the range that the append itself writes: the
    new one is the next power of two that holds it and the new values, and earlier tokens keep their values
    (to half a step). The scales have few bits, so that code times scale is exact in f32."""
    olds = [1.5, 1.0, 0.75, 1.25, 3.0, 0.0234375, 2.0 ** -60, 1.5 * 2.0 ** -60, 2.0 ** -61, 2.0 ** -100, 2.0 ** -149, 3 * 2.0 ** -149,
            2.0 ** 122, 1.5 * 2.0 ** 122, 2.0 ** 125, 2.0 ** 127, 1.5 * 2.0 ** 126, 1.25 * 2.0 ** 127]
    H, D, B = len(olds), 32, 16
    rng = np.random.default_rng(5)
    c, raws, scales = new_cache(3, H, B, D, code, 6)
    for s, t in zip(scales, (c.k_scale, c.v_scale)):
        s[:] = olds
        t.copy_(dev(s, torch.float32))
        assert np.array_equal(f64(t), s)
    for start in (0, 5):
        k, v = ((rng.standard_normal((2, H, D)) * size).astype(np.float32) for _ in range(2))
        for i, x in enumerate((k, v)):
            append_reference(raws[i], scales[i], x.astype(np.float64), [B + start, B + start + 1], code)
        c.append(dev(k, torch.float32), dev(v, torch.float32), dev([B + start, B + start + 1]))
        for got, want in ((c.k_scale, scales[0]), (c.v_scale, scales[1])):
            assert np.array_equal(f64(got), want, equal_nan=True), start
        for got, want in ((c.k_codes, raws[0]), (c.v_codes, raws[1])):
            assert np.array_equal(raw(got), want), start
        for s, t in zip(scales, (c.k_scale, c.v_scale)):  # the second pass starts from these scales again
            s[:] = olds
            t.copy_(dev(s, torch.float32))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_keeps_earlier_values(code):
    """Old scales of 24 bits: the value of every earlier token is off by half a step of the new scale at most
    (and by the f32 product's 2^-24 of itself)."""
    H, D, B = 64, 32, 16
    rng = np.random.default_rng(8)
    c, raws, scales = new_cache(2, H, B, D, code, 2)
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.rand(2, H, device="cuda") * 2 + 0.01)
    before = [ref.decode(r[1], code) * f64(t)[1][:, None, None] for r, t in zip(raws, (c.k_scale, c.v_scale))]
    x = dev(rng.standard_normal((1, H, D)), torch.float32)
    c.append(x, x, dev([B + 9]))
    for b, codes, t, r in zip(before, (c.k_codes, c.v_codes), (c.k_scale, c.v_scale), raws):
        s = f64(t)[1][:, None, None]
        after = ref.decode(raw(codes)[1], code) * s
        step = s if code == "int8" else s * 2.0 ** (np.floor(np.log2(np.maximum(np.abs(b / s), 2.0 ** -6))) - 3)
        assert np.all(np.abs(after - b)[:, :9] <= (step / 2 + np.abs(b) * 2.0 ** -24)[:, :9])
        assert np.array_equal(raw(codes)[1][:, 10:], r[1][:, 10:])  # slots behind keep their codes


# ------------------------------------------------------------------------- skipped rows inside a block's run

def append_together(raws, scales, x, slots, code):
    """ref.append where skipped rows may stand between the rows of a block: the batch without them."""
    live = [r for r, s in enumerate(slots) if 0 <= s < raws.shape[0] * raws.shape[2]]
    ref.append(raws, scales, x[live], [slots[r] for r in live], code)


def gaps(rng, n, start, share, longest):
    """Slots start .. of consecutive tokens, some masked, now and then a longer stretch without a slot; rows
    with a slot stand fewer than 128 apart."""
    slots, since = [], 0
    for s in range(start, start + n):
        live = since > 60 or rng.random() >= share
        slots.append(s if live else int(rng.choice([-1, -9, 2 ** 31 - 1])))
        since = 0 if live else since + 1
        if rng.random() < 0.05:
            more = int(rng.integers(1, longest))
            slots += [-1] * min(more, 125 - since)
            since += min(more, 125 - since)
    return slots


@pytest.mark.parametrize("code, dtype", [("int8", "f32"), ("e4m3", "bf16"), ("int8", "f16")])
@pytest.mark.parametrize("H, D, B, nb", [(1, 256, 16, 60), (3, 80, 32, 40), (2, 64, 128, 20)])
def test_append_skipped_rows(code, dtype, H, D, B, nb):
    """Rows masked by -1 between rows of a block: one scale for all of them, whichever row of a CTA's tile or
    of a 32-row step they stand at. Then rows as far apart as the call allows."""
    rng = np.random.default_rng(B)
    c, raws, scales = new_cache(nb, H, B, D, code, B)
    batches = [[B + 5, -1, B + 6], [-1, B + 7, -1, -1, B + 9, -1], [-1] * 200 + [2 * B, -1, 2 * B + 2] + [-1] * 300,
               [3 * B] + [-1] * 126 + [3 * B + 1] + [-1] * 126 + [3 * B + 2], [3 * B + 3, -1, -1, 4 * B, -1, 4 * B + 1, 5 * B],
               [6 * B + 3, -1, 6 * B + 3, -1, 6 * B + 1]]
    batches += [gaps(rng, nb * B - 3, 3, share, 130) for share in (0.1, 0.5, 0.9)]
    for slots in batches:
        last = None  # neighbours with a slot stand fewer than 128 rows apart, or are of different blocks
        for r, s in enumerate(slots):
            if 0 <= s < nb * B:
                assert last is None or r - last[0] < 128 or last[1] // B != s // B
                last = r, s
        k, v = ((dev(rng.standard_normal((len(slots), H, D)) * 2.0 ** rng.uniform(-3, 3, (len(slots), H, 1)), torch.float32)).to(DT[dtype]) for _ in range(2))
        for i, x in enumerate((k, v)):
            append_together(raws[i], scales[i], f64(x), slots, code)
        c.append(k, v, dev(slots))
        for got, want in ((c.k_scale, scales[0]), (c.v_scale, scales[1])):
            assert np.array_equal(f64(got), want), slots[:20]
        for got, want in ((c.k_codes, raws[0]), (c.v_codes, raws[1])):
            assert np.array_equal(raw(got), want), slots[:20]


# ------------------------------------------------------------------------- every kernel in one process

def test_attend_raises_no_limit_twice():
    """All kernels of the attention (a process may use them all) raise their shared-memory limit on their first
    launch, and no later call does so again."""
    from torch.profiler import ProfilerActivity, profile
    rng = np.random.default_rng(3)
    lens, cu = [300], dev([0, 40])
    caches = [make_batch(rng, None, lens, 16, 1, D, code) for D in (64, 128, 256) for code in ("int8", "e4m3")]
    qs = {(heads, D, dtype): torch.randn(40, heads, D, device="cuda").to(DT[dtype]) for heads in (8, 16, 32) for D in (64, 128, 256) for dtype in ("f32", "bf16")}

    def every():
        for c, _, _, table in caches:
            for dtype in ("f32", "bf16"):
                for heads, max_rows in ((8, 1), (16, 1), (32, 1), (8, 40)):
                    c.attend(qs[heads, c.head_dim, dtype], cu, dev(lens), dev(table), max_rows=max_rows, max_len=300)
        torch.cuda.synchronize()

    every()
    with profile(activities=[ProfilerActivity.CPU, ProfilerActivity.CUDA]) as p:
        every()
    names = [e.name for e in p.events()]
    assert len({n for n in names if "gg_kv8_rows_kernel" in n or "gg_kv8_prompt_kernel" in n}) == 44
    assert sum(n.startswith("cudaLaunchKernel") for n in names) >= 48
    assert not [n for n in names if n.startswith("cudaFuncSetAttribute")]


# ------------------------------------------------------------------------- long sums

@pytest.mark.parametrize("D, H, n", [(64, 8, 40), (128, 4, 80), (256, 1, 300)])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_attend_sums_over_many_keys_of_a_warp(code, D, H, n):
    """Single f32 tokens of so many requests that none is cut: a warp sums 16384 keys. All values are positive and
    all weights alike, so a sum that is always rounded one way would be off by 1e-4. The requests share
    their pages. Tolerance as in check_attend."""
    from gemma_b200 import ops
    B, L, G = 128, 65536, 4
    g = torch.Generator(device="cuda").manual_seed(D)
    c = ops.KV8Cache.empty(L // B, B, H, D, code)
    for t, lo in ((c.k_codes, -127), (c.v_codes, 64)):
        t.copy_(torch.randint(lo, 128, t.shape, device="cuda", generator=g).float().to(t.dtype))
    c.k_scale.fill_(2.0 ** -20)
    table = torch.arange(L // B, dtype=torch.int32, device="cuda").repeat(n, 1)
    q = torch.randn(n, H * G, D, device="cuda", generator=g)
    out, lse = c.attend(q, torch.arange(n + 1, dtype=torch.int32, device="cuda"), torch.full((n,), L, dtype=torch.int32, device="cuda"), table,
                        max_rows=1, max_len=L, return_lse=True)
    for i, h in ((0, 0), (n - 1, H - 1)):
        k, v = (t[:, h].float().double().reshape(-1, D) for t in (c.k_codes, c.v_codes))
        z = q[i, h * G:(h + 1) * G].double() @ (k * 2.0 ** -20).T * D ** -0.5
        want = torch.softmax(z, -1) @ v  # the values are positive: also the sum of p |v|
        ds = (q[i, h * G:(h + 1) * G].double().abs() @ (k.abs() * 2.0 ** -20).T * D ** -0.5).amax(-1, keepdim=True) * (2.0 ** -21 + 2.0 ** -19) + 2.0 ** -22
        tol = (2 * (2 * ds + 2.0 ** -18) + 2.0 ** -24) * want
        got = out[i, h * G:(h + 1) * G].double()
        assert bool(((got - want).abs() <= tol).all()), ((got - want) / want).abs().max().item()
        assert bool(((lse[i, h * G:(h + 1) * G].double() - torch.logsumexp(z, -1)).abs() <= ds[:, 0] + 2.0 ** -20 + 2.0 ** -22 * 12).all())


@pytest.mark.parametrize("D, H", [(64, 8), (128, 8), (256, 4)])
@pytest.mark.parametrize("L", [4095, 4097, 16385])
def test_attend_sums_of_f32_prompts(D, H, L):
    """Many f32 rows, positive values and weights alike, between and behind the points where O goes to memory: off
    by no more than the bound the header gives (7e-6) and the output's rounding."""
    from gemma_b200 import ops
    B, n, rows = 64, 12, 40
    g = torch.Generator(device="cuda").manual_seed(D + L)
    c = ops.KV8Cache.empty(-(-L // B), B, H, D, "int8")
    for t, lo in ((c.k_codes, -127), (c.v_codes, 64)):
        t.copy_(torch.randint(lo, 128, t.shape, device="cuda", generator=g, dtype=torch.int32))
    c.k_scale.fill_(2.0 ** -20)
    table = torch.arange(c.num_blocks, dtype=torch.int32, device="cuda").repeat(n, 1)
    q = torch.randn(n * rows, 4 * H, D, device="cuda", generator=g)
    out = c.attend(q, torch.arange(n + 1, dtype=torch.int32, device="cuda") * rows, dev([L] * n), table, max_rows=rows, max_len=L)
    for h in (0, H - 1):
        k, v = (t[:, h].double().reshape(-1, D)[:L] for t in (c.k_codes, c.v_codes))
        want = torch.softmax(q[rows - 1, 4 * h:4 * h + 4].double() @ (k * 2.0 ** -20).T * D ** -0.5, -1) @ v
        assert bool(((out[rows - 1, 4 * h:4 * h + 4].double() - want).abs() <= (7e-6 + 2.0 ** -24) * want).all())


@pytest.mark.parametrize("rows, n, L", [(1, 300, 1 << 22), (128, 75, 1 << 22)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attend_sums_over_millions_of_keys(dtype, rows, n, L):
    """16-bit rows over contexts beyond 2^18 keys, more (request, head) units than the GPU holds: no sum may lose
    more than its rounding. Tolerance as in check_attend; all values are positive, the requests share their pages."""
    from gemma_b200 import ops
    B, D, G = 128, 16, 4 if rows == 1 else 2
    g = torch.Generator(device="cuda").manual_seed(L)
    c = ops.KV8Cache.empty(L // B, B, 1, D, "int8")
    for t, lo in ((c.k_codes, -127), (c.v_codes, 64)):
        t.copy_(torch.randint(lo, 128, t.shape, device="cuda", generator=g, dtype=torch.int32))
    c.k_scale.fill_(2.0 ** -20)
    table = torch.arange(L // B, dtype=torch.int32, device="cuda").repeat(n, 1)
    q = torch.randn(n * rows, G, D, device="cuda", generator=g).to(DT[dtype])
    out = c.attend(q, torch.arange(n + 1, dtype=torch.int32, device="cuda") * rows, torch.full((n,), L, dtype=torch.int32, device="cuda"), table,
                   max_rows=rows, max_len=L)
    k, v = (t.double().reshape(-1, D) for t in (c.k_codes, c.v_codes))
    for i in (rows - 1, n * rows - 1):  # rows that see all keys
        z = q[i].double() @ (k * 2.0 ** -20).T * D ** -0.5
        want = torch.softmax(z, -1) @ v
        ds = (q[i].double().abs() @ (k.abs() * 2.0 ** -20).T * D ** -0.5).amax(-1, keepdim=True) * (2.0 ** -21 + 2.0 ** -19) + 2.0 ** -22
        tol = (2 * (2 * ds + 2.0 ** -18) + 2 * 2.0 ** -11 + HALF_EPS[dtype]) * want
        assert bool(((out[i].double() - want).abs() <= tol).all()), ((out[i].double() - want) / want).abs().max().item()


# ------------------------------------------------------------------------- what autograd would follow

def test_rope_refuses_tangents_and_learned_frequencies():
    """Neither a dual tensor nor frequencies that require a gradient lose it silently."""
    from gemma_b200 import ops
    from torch.autograd import forward_ad
    x, pos = torch.randn(4, 2, 32, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda")
    f, _ = ops.rope_frequencies(32, 1e4)
    want = ops.rope(x, None, pos, f)[0]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for q, k, fr in ((dual, None, f), (x, dual, f), (x, None, forward_ad.make_dual(f, f))):
            with pytest.raises(ValueError, match="tangent"):
                ops.rope(q, k, pos, fr)
        assert torch.equal(ops.rope(x, None, pos, f)[0], want)
    learned = f.clone().requires_grad_()
    with pytest.raises(ValueError, match="freqs requires a gradient"):
        ops.rope(x, None, pos, learned)
    with torch.no_grad():
        assert torch.equal(ops.rope(x, None, pos, learned)[0], want)


# ------------------------------------------------------------------------- large keys, small queries

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows, lens", [([1, 1], [90, 700]), ([40], [300])])
def test_attend_large_keys_small_queries(dtype, rows, lens):
    """Scores of ordinary size from keys of 2^120, queries of 2^-100 and a scale of 2^-16: no step between them
    overflows."""
    rng = np.random.default_rng(2)
    c, raws, scales, table = make_batch(rng, rows, lens, 16, 1, 64, "int8")
    scales[0][:] = 2.0 ** 113
    c.k_scale.fill_(2.0 ** 113)
    q = (torch.randn(sum(rows), 4, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * 2.0 ** -40).to(DT[dtype])
    check_attend(rng, rows, lens, 4, c, raws, scales, table, "int8", dtype, q=q * 2.0 ** -60, scale=2.0 ** -16)


# ------------------------------------------------------------------------- block ids that no cache has

@pytest.mark.parametrize("n, chunk", [(3, 20), (700, 5), (5000, 2), (64, 100)])
def test_plan_of_impossible_block_ids(n, chunk):
    """Ids below 0, and so large that their slots pass 31 bits, from the table or from the free list: the rows
    there have no slot. (Wrapped around, they would be another request's.)"""
    from gemma_b200 import ops
    B = 16
    rng = np.random.default_rng(n)
    old = rng.integers(0, 40, n)
    new = old + chunk
    blocks = -(-int(new.max()) // B)
    held = -(-old // B)
    bad = np.array([-1, -2 ** 27, 2 ** 27, 2 ** 27 + 3, 2 ** 28 + 1, 2 ** 31 - 1, -2 ** 31])
    ids = np.where(rng.random(n * (blocks + 1)) < 0.3, rng.choice(bad, n * (blocks + 1)), rng.integers(0, 2 ** 27, n * (blocks + 1)))
    table = np.where(np.arange(blocks)[None] < held[:, None], ids[:n * blocks].reshape(n, blocks), -1)
    free = rng.permutation(ids)
    rows = n * chunk + 3
    t, fl = dev(table), dev(free)
    p = ops.plan_blocks(dev(old), dev(new), t, fl, dev([len(free)]), B, rows)
    assert int(p.status) == 0
    t = t.cpu().numpy().astype(np.int64)
    slots = [t[i, x // B] * B + x % B for i in range(n) for x in range(old[i], new[i])]
    want = [int(s) if 0 <= s < 2 ** 31 else -1 for s in slots] + [-1] * 3
    assert want.count(-1) > 3  # some rows stand in such a block
    assert p.slots.cpu().tolist() == want


def test_sizes_beyond_32_bits_refused():
    """As ValueError, before anything of that size is allocated or looked up."""
    from gemma_b200 import ops
    c = ops.KV8Cache.empty(4, 16, 1, 32)
    q, one, t = torch.zeros(1, 4, 32, device="cuda"), dev([1]), dev([[0, 1]])
    for kw in (dict(max_rows=(1 << 32) + 1, max_len=16), dict(max_rows=1, max_len=16, window=1 << 31), dict(max_rows=1, max_len=-(1 << 40))):
        with pytest.raises(ValueError, match="32 bits"):
            c.attend(q, dev([0, 1]), one, t, **kw)
    with pytest.raises(ValueError, match="32 bits"):
        c.workspace_bytes(q, 1 << 40, 1, 16)
    for rows, block in ((1 << 31, 16), (4, 1 << 33)):
        with pytest.raises(ValueError, match="32 bits"):
            ops.plan_blocks(one, one, t, dev([0]), dev([1]), block, rows)


# ------------------------------------------------------------------------- many keys to a CTA

LONG = [511, 512, 513, 1023, 1025, 4095, 4096, 4097, 8191, 8193, 16383, 16385]


def long_cache(D, H, B, code, g):
    """A cache with room for LONG[-1] tokens of one request, random codes and scales, blocks in random order."""
    from gemma_b200 import ops
    nb = -(-LONG[-1] // B) + 2
    c = ops.KV8Cache.empty(nb, B, H, D, code)
    for t in (c.k_codes, c.v_codes):
        t.copy_(torch.randint(-127, 128, t.shape, device="cuda", generator=g).float().to(t.dtype))
    c.k_scale.copy_(2.0 ** torch.randint(-7, -4, c.k_scale.shape, device="cuda", generator=g))
    c.v_scale.copy_(2.0 ** torch.randint(-9, -3, c.v_scale.shape, device="cuda", generator=g))
    return c, torch.randperm(nb, device="cuda", generator=g)[:-(-LONG[-1] // B)].int()


def check_long(c, row, lens, rows, q, out, lse, window, dtype):
    """The first and the last row of every request, in the first and the last key head, against softmax in 64
    bits; tolerances as in check_attend. All requests share the pages of `row`."""
    B, D, H = c.block_tokens, c.head_dim, c.kv_heads
    G, w = q.shape[1] // H, 0.0 if dtype == "f32" else 2 * 2.0 ** -11
    for h in {0, H - 1}:
        codes = [t.view(torch.int8)[row.long(), h].view(t.dtype).float().double() for t in (c.k_codes, c.v_codes)]
        ks, vs = (t[row.long(), h].double().repeat_interleave(B) for t in (c.k_scale, c.v_scale))
        k, v = codes[0].reshape(-1, D) * ks[:, None], codes[1].reshape(-1, D) * vs[:, None]
        for i, n in enumerate(lens):
            for r in {0, rows - 1}:
                p = n - rows + r
                lo = max(0, p - window + 1) if window else 0
                x = q[i * rows + r, h * G:(h + 1) * G].double()
                kk, vv = k[lo:p + 1], v[lo:p + 1]
                z = x @ kk.T * D ** -0.5
                pr = torch.softmax(z, -1)
                want, pv = pr @ vv, pr @ vv.abs()
                least = (pr * vs[lo:p + 1]).amax(-1, keepdim=True) * (vv.abs() / vs[lo:p + 1, None]).sum(0)
                ds = (x.abs() @ kk.abs().T).amax(-1, keepdim=True) * D ** -0.5 * (2.0 ** -21 + 2.0 ** -19) + 2.0 ** -22
                tol = (2 * (2 * ds + 2.0 ** -18) + w) * pv + HALF_EPS[dtype] * want.abs() + (2.0 ** -25 if dtype == "f16" else 0) + 2.0 ** -32 * least
                got = out[i * rows + r, h * G:(h + 1) * G].double()
                assert bool(((got - want).abs() <= tol).all()), (h, i, r, ((got - want).abs() / tol).max().item())
                ref_lse = torch.logsumexp(z, -1)
                err = (lse[i * rows + r, h * G:(h + 1) * G].double() - ref_lse).abs()
                assert bool((err <= ds[:, 0] + 2.0 ** -20 + 2.0 ** -22 * ref_lse.abs()).all()), (h, i, r)


def attend_long(c, row, lens, rows, q, window, odd):
    n = len(lens)
    table = row.repeat(n, 1)
    room = torch.full((n * rows * (q.shape[1] * c.head_dim + 3) + 1,), 7.0, device="cuda", dtype=q.dtype)
    width = q.shape[1] * c.head_dim + (3 if odd else 0)
    out = torch.as_strided(room, q.shape, (width, c.head_dim, 1), 1 if odd else 0)
    _, lse = c.attend(q, torch.arange(n + 1, dtype=torch.int32, device="cuda") * rows, dev(lens), table, max_rows=rows, max_len=max(lens),
                      window=window, out=out, return_lse=True)
    return out, lse


def ranges(c, q, n, rows, window):
    """Key ranges that a call with many rows is cut into: what its workspace holds beyond that of few rows."""
    few = c.workspace_bytes(q, n, 32 // (q.shape[1] // c.kv_heads), LONG[-1], window)
    more = c.workspace_bytes(q, n, rows, LONG[-1], window) - few
    each = q.shape[0] * q.shape[1] * (4 * c.head_dim + 8)
    assert more % each == 0
    return max(1, more // each)


@pytest.mark.parametrize("code, dtype", [("int8", "f32"), ("e4m3", "f32"), ("int8", "bf16"), ("e4m3", "f16")])
@pytest.mark.parametrize("D, H, B", [(64, 8, 32), (128, 8, 64), (256, 4, 16), (80, 8, 128)])
@pytest.mark.parametrize("window, odd", [(0, False), (0, True), (5000, False)])
def test_attend_prompts_over_many_tiles(code, dtype, D, H, B, window, odd):
    """So many tiles of query rows that no key range is cut: a CTA walks up to 257 tiles of 64 keys, through several
    batches of block ids, around its ring of scales, and adds f32 rows to memory every 4096 keys (at any
    alignment of the output)."""
    g = torch.Generator(device="cuda").manual_seed(D + B)
    c, row = long_cache(D, H, B, code, g)
    rows = 40
    q = torch.randn(len(LONG) * rows, 4 * H, D, device="cuda", generator=g).to(DT[dtype])
    assert ranges(c, q, len(LONG), rows, window) == 1
    out, lse = attend_long(c, row, LONG, rows, q, window, odd)
    check_long(c, row, LONG, rows, q, out, lse, window, dtype)


@pytest.mark.parametrize("code, dtype", [("int8", "f32"), ("e4m3", "bf16")])
@pytest.mark.parametrize("D, H, B", [(64, 8, 32), (128, 8, 64), (256, 4, 16)])
def test_attend_prompts_in_long_ranges(code, dtype, D, H, B):
    """Ranges of more than 4096 keys: f32 rows are added up in the workspace, then joined."""
    g = torch.Generator(device="cuda").manual_seed(D)
    c, row = long_cache(D, H, B, code, g)
    rows, lens = 40, [16385, 9000, 16384, 5000, 12289]
    q = torch.randn(len(lens) * rows, 4 * H, D, device="cuda", generator=g).to(DT[dtype])
    assert 2 <= ranges(c, q, len(lens), rows, 0) <= 3  # of 1025 steps of 16 keys
    out, lse = attend_long(c, row, lens, rows, q, 0, False)
    check_long(c, row, lens, rows, q, out, lse, 0, dtype)


@pytest.mark.parametrize("code, dtype", [("int8", "f32"), ("e4m3", "f32"), ("int8", "bf16"), ("e4m3", "f16")])
@pytest.mark.parametrize("D, H, B, n, rows", [(64, 8, 32, 48, 1), (128, 8, 64, 36, 2), (256, 4, 16, 72, 2), (80, 8, 128, 36, 7)])
@pytest.mark.parametrize("window", [0, 5000])
def test_attend_steps_over_many_batches(code, dtype, D, H, B, n, rows, window):
    """So many requests that none is cut far: a warp walks hundreds of steps, through several batches of block ids
    and scales."""
    g = torch.Generator(device="cuda").manual_seed(D + n)
    c, row = long_cache(D, H, B, code, g)
    lens = (LONG * 6)[:n]
    q = torch.randn(n * rows, 4 * H, D, device="cuda", generator=g).to(DT[dtype])
    out, lse = attend_long(c, row, lens, rows, q, window, rows == 2)
    check_long(c, row, lens, rows, q, out, lse, window, dtype)
