"""The device-memory operators (gemma_b200.ops) against plain restatements in 64 bits.

Integers, codes and scales must be equal. Floating results may differ by the kernels' own roundings,
counted from the arithmetic (eps/2 of a type: bf16 2^-8, f16 2^-11, f32 2^-24):

* rope: the angle's fraction of a turn is rounded to f32 (2^-25 of a turn at most, pi 2^-24 rad) and
  sincospi is good to 2 ulp, so c and s are off by less than 6 * 2^-24; with two products and a sum
  the result is off by at most 8 * 2^-24 mscale (|a| + |b|), plus the output's eps/2.
* attend: a score is off by ds <= S (2^-21 + 2^-19), S = scale max_j sum_d |q_d k_d|: queries enter as
  f16 hi + lo (2^-22 each) or exactly, and the sums of up to 256 products in f32 lose at most
  2^-19 S (16 steps of 16 products, each step rounded or cut at 2^-23). A weight is then off by
  2 ds + 2^-18 (exponent, running maximum), plus 2^-11 where f16 and bf16 calls round it to f16,
  in numerator and denominator alike: |out - ref| <= (2 (2 ds + 2^-18) + w) sum p |v| + eps/2 |ref|.
  Weights enter the second product as f16 of 2^7 w with w = 1 or more for the largest, so a weight
  below f16's normal numbers is off by half its smallest step, 2^-25 / 2^7 of the largest weight;
  w_j = p_j vs_j up to a common factor, hence the last term 2^-32 max_j (p_j vs_j) sum_j |code_j|.
"""
import math

import numpy as np
import pytest

import ops_reference as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_EPS = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def dev(x, dtype=torch.int32):
    return torch.tensor(np.asarray(x), dtype=dtype, device="cuda")


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


# ---------------------------------------------------------------------------------------- plan

def run_plan(old, new, table, free, count, B, rows, alias=False):
    from gemma_b200 import ops
    t, fl, fc = dev(table), dev(free), dev([count])
    out = None
    if alias:
        e = lambda n: torch.full((n,), -9, dtype=torch.int32, device="cuda")  # noqa: E731
        out = ops.BlockPlan(e(len(old) + 1), e(len(old)), e(rows), e(rows), e(rows), fc, e(1))
    p = ops.plan_blocks(dev(old), dev(new), t, fl, fc, B, rows, out=out)
    return {k: v.cpu().numpy() for k, v in p._asdict().items()}, t.cpu().numpy(), fl.cpu().numpy(), int(fc)


def check_plan(old, new, table, free, count, B, rows, alias=False):
    got, t, fl, fc = run_plan(old, new, table, free, count, B, rows, alias)
    want, wt, wfl = ref.plan(old, new, table, free, count, B, rows)
    for k, v in want.items():
        assert np.array_equal(got[k].reshape(-1), np.asarray(v).reshape(-1)), k
    assert np.array_equal(t, wt)
    top = want["free_count"]
    assert np.array_equal(fl[:top], wfl[:top])
    assert fc == (top if alias else count)
    return want["status"]


def make_plan(rng, n, B, hi, kinds, spare):
    old = rng.integers(0, hi, n)
    new = old.copy()
    for i in range(n):
        k = rng.choice(kinds)
        new[i] = {"step": old[i] + 1, "chunk": old[i] + rng.integers(1, 3 * B + 40), "end": 0, "back": max(0, old[i] - rng.integers(1, B + 3)), "idle": old[i]}[k]
    width = int(max(ref.blocks_of(max(a, b), B) for a, b in zip(old, new))) + 1
    held = [ref.blocks_of(int(a), B) for a in old]
    ids = rng.permutation(sum(held) + spare)
    table = np.full((n, width), -1)
    at = 0
    for i, x in enumerate(held):
        table[i, :x] = ids[at:at + x]
        at += x
    free = np.concatenate([ids[at:], np.full(at, -5)])
    return [int(x) for x in old], [int(x) for x in new], table, free, spare


@pytest.mark.parametrize("n, B, hi, kinds", [
    (1, 16, 40, ["step"]), (1, 128, 3, ["chunk"]), (64, 16, 700, ["step"]), (7, 32, 90, ["end", "back", "chunk", "idle", "step"]),
    (300, 16, 400, ["step", "chunk", "end", "back", "idle"]), (5000, 64, 300, ["step", "chunk", "end", "back"]),
    (4096, 16, 20, ["step", "end"]), (4097, 16, 20, ["chunk", "back"]), (33, 1, 9, ["chunk", "end", "step"]), (9000, 16, 40, ["step", "idle"])])
@pytest.mark.parametrize("alias", [False, True])
def test_plan(n, B, hi, kinds, alias):
    rng = np.random.default_rng(n * 131 + B)
    old, new, table, free, count = make_plan(rng, n, B, hi, kinds, 8 * n + 20 * n * (B == 1) * 5 + n * (44 // B + 4))
    rows = sum(max(0, b - a) for a, b in zip(old, new))
    assert check_plan(old, new, table, free, count, B, rows + 13, alias) == 0
    assert check_plan(old, new, table, free, count, B, rows, alias) == 0


def test_plan_failures_change_nothing():
    rng = np.random.default_rng(5)
    old, new, table, free, count = make_plan(rng, 50, 16, 200, ["chunk", "step", "back"], 400)
    rows = sum(max(0, b - a) for a, b in zip(old, new))
    give = sum(max(0, ref.blocks_of(a, 16) - ref.blocks_of(b, 16)) for a, b in zip(old, new))
    take = sum(max(0, ref.blocks_of(b, 16) - ref.blocks_of(a, 16)) for a, b in zip(old, new))
    assert take > give
    assert check_plan(old, new, table, free, take - give, 16, rows) == 0     # exactly enough
    assert check_plan(old, new, table, free, take - give - 1, 16, rows) == 1
    assert check_plan(old, new, table, free, count, 16, rows - 1) == 4
    assert check_plan(old, new, table, free, -1, 16, rows) == 16
    assert check_plan(old, new, table, free, len(free) + 1, 16, rows) == 16
    assert check_plan(old, new, table, free[:count + give - 1], count, 16, rows) == 16
    long = list(new)
    long[3] = table.shape[1] * 16 + 1
    assert check_plan(old, long, table, free, count, 16, rows + 100000, alias=True) == 2
    bad = list(new)
    bad[7] = -1
    assert check_plan(old, bad, table, free, count, 16, rows + 100) == 8
    worse = list(old)
    worse[0] = table.shape[1] * 16 + 1
    assert check_plan(worse, new, table, free, count, 16, rows + 100000) & 8
    huge = [2 ** 31 - 1] * 50
    assert check_plan(old, huge, table, free, count, 16, rows) & 6 == 6


# ---------------------------------------------------------------------------------------- rope

@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D, rot, H, K, n", [(256, 256, 4, 1, 5), (128, 64, 8, 2, 33), (80, 26, 3, 1, 1), (64, 2, 1, 1, 700), (96, 48, 16, 16, 130), (20, 20, 2, 0, 9)])
@pytest.mark.parametrize("inverse", [False, True])
def test_rope(dtype, layout, D, rot, H, K, n, inverse):
    from gemma_b200 import ops
    rng = np.random.default_rng(D * 7 + n)
    x = dev(rng.standard_normal((n, H + 2 * K, D)) * 3, torch.float32).to(DT[dtype])  # rows of a fused projection
    q, k = x[:, :H], (x[:, H:H + K] if K else None)
    pos = rng.integers(0, 5000, n)
    pos[rng.random(n) < 0.1] = -1
    if n > 4:
        pos[1], pos[2], pos[3] = 2 ** 31 - 1, 1000003, 0
    freqs, m = ops.rope_frequencies(rot, 1e6, "yarn", 4.0, 32768.0, 1.0, 32.0)
    before = x.clone()
    oq, ok = ops.rope(q, k, dev(pos), freqs, layout=layout, mscale=m, inverse=inverse)
    assert torch.equal(x, before)
    for got, src in ((oq, q), (ok, k)):
        if src is None:
            assert got is None
            continue
        v = f64(src)
        want = ref.rope(v, pos, f64(freqs), layout, m, inverse)
        h = rot // 2
        mag = np.zeros_like(v)
        a, b = (v[..., :h], v[..., h:rot]) if layout == "half" else (v[..., 0:rot:2], v[..., 1:rot:2])
        s = np.abs(a) + np.abs(b)
        if layout == "half":
            mag[..., :h], mag[..., h:rot] = s, s
        else:
            mag[..., 0:rot:2], mag[..., 1:rot:2] = s, s
        # at position p the angle itself is a f64 product: 2^-53 p more
        ang = np.abs(pos)[:, None, None] * 2.0 ** -52
        tol = (8 * 2.0 ** -24 + ang) * m * mag + HALF_EPS[dtype] * np.abs(want) + (2.0 ** -25 if dtype == "f16" else 0)
        assert np.all(np.abs(f64(got) - want) <= tol)
        assert np.array_equal(f64(got)[pos < 0], v[pos < 0])      # padding is copied
        assert np.array_equal(f64(got)[..., rot:], v[..., rot:])  # and so is the rest of the head


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("off, pad", [(0, 0), (1, 0), (3, 5), (8, 8)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rope_in_place_and_any_alignment(layout, off, pad, dtype):
    from gemma_b200 import ops
    n, H, D, rot = 37, 3, 64, 32
    base = torch.randn(n * (H * D + pad) + off, device="cuda").to(DT[dtype])
    x = torch.as_strided(base, (n, H, D), (H * D + pad, D, 1), off)
    keep, pos = base.clone(), torch.arange(n, dtype=torch.int32, device="cuda")
    freqs, _ = ops.rope_frequencies(rot, 1e4)
    want = ops.rope(x.contiguous(), None, pos, freqs, layout=layout)[0]
    got = ops.rope(x, None, pos, freqs, layout=layout, out=(x, None))[0]
    assert got.data_ptr() == x.data_ptr() and torch.equal(got, want)
    torch.as_strided(base, (n, H, D), (H * D + pad, D, 1), off).copy_(torch.as_strided(keep, (n, H, D), (H * D + pad, D, 1), off))
    assert torch.equal(base, keep)  # nothing between or behind the rows was written


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_gradient(layout):
    """The inverse call is the transpose of the forward call: against differences and the formula."""
    from gemma_b200 import ops
    n, H, D, rot = 11, 2, 48, 32
    freqs, m = ops.rope_frequencies(rot, 1e4, "yarn", 8.0, 64.0, 1.0, 8.0)
    pos = dev(np.arange(n) * 13)
    g = torch.Generator(device="cuda").manual_seed(3)
    x, dy, dx = (torch.randn(n, H, D, device="cuda", generator=g) for _ in range(3))
    turn = lambda v, inv=False: ops.rope(v, None, pos, freqs, layout=layout, mscale=m, inverse=inv)[0]  # noqa: E731
    h = 0.5  # the call is linear: a large step loses nothing
    along = (f64(turn(x + h * dx)) - f64(turn(x - h * dx))).ravel() @ f64(dy).ravel() / (2 * h)
    grad = f64(turn(dy, True))
    # sums of n H D products, each value off by at most 2^-20 of a sum of two normal values
    bound = 2.0 ** -20 * (np.abs(f64(dy)).sum() + np.abs(f64(dx)).sum()) * 8
    assert abs(grad.ravel() @ f64(dx).ravel() - along) <= bound
    want = ref.rope(f64(dy), f64(pos).astype(int), f64(freqs), layout, m, True)
    assert np.all(np.abs(grad - want) <= 2.0 ** -19 * m * np.abs(f64(dy)).max())
    back = f64(turn(turn(x), True))
    assert np.allclose(back[..., :rot], m * m * f64(x)[..., :rot], rtol=0, atol=2.0 ** -18 * m * m * 5)


def test_rope_refuses():
    from gemma_b200 import ops
    x, pos = torch.zeros(4, 2, 32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    f, _ = ops.rope_frequencies(32, 1e4)
    with pytest.raises(ValueError, match="gradient"):
        ops.rope(x.clone().requires_grad_(), None, pos, f)
    with pytest.raises(ValueError, match="contiguous"):
        ops.rope(x.transpose(1, 2), None, pos, f)
    with pytest.raises(ValueError, match="positions"):
        ops.rope(x, None, pos[:3], f)
    with pytest.raises(ValueError, match="int32"):
        ops.rope(x, None, pos.long(), f)
    with pytest.raises(ValueError, match="float64"):
        ops.rope(x, None, pos, f.float())
    with pytest.raises(ops.GemmaB200Error, match="rot_dim"):
        ops.rope(x, None, pos, ops.rope_frequencies(34, 1e4)[0])
    with pytest.raises(ValueError, match="differ"):
        ops.rope(x, x.half(), pos, f)


# ---------------------------------------------------------------------------------------- append

def new_cache(nb, H, B, D, code, seed):
    """(KV8Cache, raw codes and scales of K and V as numpy) filled with earlier tokens."""
    from gemma_b200 import ops
    rng = np.random.default_rng(seed)
    raws, scales = [], []
    for _ in range(2):
        x = np.clip(rng.standard_normal((nb, H, B, D)) * ref.TOP[code] / 4, -ref.TOP[code], ref.TOP[code])
        raws.append(ref.encode(x, code))
        scales.append(2.0 ** rng.integers(-9, -3, (nb, H)).astype(np.float64))
    t = [dev(r.view(np.int8), torch.int8) for r in raws]
    if code == "e4m3":
        t = [v.view(torch.float8_e4m3fn) for v in t]
    return ops.KV8Cache(*t, *(dev(s, torch.float32) for s in scales)), raws, scales


def raw(t):
    return t.view(torch.int8).cpu().numpy().view(np.uint8)


def check_append(c, raws, scales, k, v, slots, code):
    for i, x in enumerate((k, v)):
        ref.append(raws[i], scales[i], f64(x), list(slots), code)
    c.append(k, v, dev(slots))
    for got, want in ((c.k_scale, scales[0]), (c.v_scale, scales[1])):
        assert np.array_equal(f64(got), want, equal_nan=True)
    for got, want in ((c.k_codes, raws[0]), (c.v_codes, raws[1])):
        assert np.array_equal(raw(got), want)


def values(rng, n, H, D, dtype, spread=3.0):
    x = rng.standard_normal((n, H, D)) * 2.0 ** rng.uniform(-spread, spread, (n, H, 1))
    return dev(x, torch.float32).to(DT[dtype])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H, D, B", [(1, 256, 16), (3, 80, 32), (8, 128, 64), (2, 16, 128)])
def test_append_steps_and_prompts(code, dtype, H, D, B):
    """Single tokens one call after another, then a prompt over several blocks, then single tokens again."""
    rng = np.random.default_rng(D + B)
    c, raws, scales = new_cache(24, H, B, D, code, D)
    order = rng.permutation(24)
    slot = lambda s, p: int(order[8 * s + p // B]) * B + p % B  # noqa: E731 (three requests of 8 blocks)
    lens = [0, B - 2, 3 * B // 2]
    for _ in range(5):
        slots = [slot(s, lens[s]) for s in range(3)]
        check_append(c, raws, scales, values(rng, 3, H, D, dtype), values(rng, 3, H, D, dtype), slots, code)
        lens = [x + 1 for x in lens]
    slots = [slot(1, p) for p in range(lens[1], lens[1] + 2 * B + 5)] + [-1, -7] + [slot(2, p) for p in range(lens[2], 4 * B)]
    check_append(c, raws, scales, values(rng, len(slots), H, D, dtype), values(rng, len(slots), H, D, dtype), slots, code)
    lens[1] += 2 * B + 5
    for _ in range(3):
        check_append(c, raws, scales, values(rng, 1, H, D, dtype, 6), values(rng, 1, H, D, dtype, 6), [slot(1, lens[1])], code)
        lens[1] += 1


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_many_rows(code):
    """More rows than the kernel takes one to a CTA: tiles whose first row continues a block."""
    rng = np.random.default_rng(8)
    H, D, B, nb = 4, 32, 32, 400
    c, raws, scales = new_cache(nb, H, B, D, code, 1)
    slots = np.concatenate([np.arange(13, 7000), [-1] * 11, np.arange(8000, 12000)])
    k, v = values(rng, len(slots), H, D, "bf16"), values(rng, len(slots), H, D, "bf16")
    check_append(c, raws, scales, k, v, [int(s) for s in slots], code)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_odd_slots(code):
    """Slots outside the cache, the same slot twice, rows of a block in any order, rewritten slots."""
    rng = np.random.default_rng(2)
    H, D, B, nb = 2, 64, 16, 6
    c, raws, scales = new_cache(nb, H, B, D, code, 4)
    for slots in ([nb * B, 2 ** 31 - 1, -2 ** 31, 5], [20, 20, 20], [37, 36, 35, 36], [48, 49, 48], [90, 91, 92, 95], [64] * 40, [3, 4, 5], [4]):
        n = len(slots)
        check_append(c, raws, scales, values(rng, n, H, D, "f32"), values(rng, n, H, D, "f32"), slots, code)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("start", [0, 5])
def test_append_extremes(code, start):
    """Zeros, the smallest and largest values, values on the border of a scale, rounding ties."""
    H, D, B = 1, 32, 16
    top = ref.TOP[code]
    rows = [np.zeros(D), np.full(D, 1e-45), np.full(D, 2.0 ** -60 * top), np.full(D, np.nextafter(np.float32(2.0 ** -60 * top), np.float32(1))),
            np.full(D, top), np.full(D, np.nextafter(np.float32(top), np.float32(1e9))), np.arange(D) + 0.5, -(np.arange(D) * 2 + 1) / 2,
            np.full(D, 3.4e38), np.concatenate([np.full(D - 1, 1e-20), [1.0]])]
    for i, x in enumerate(rows):
        c, raws, scales = new_cache(4, H, B, D, code, i)
        k = dev(x.reshape(1, 1, D), torch.float32)
        check_append(c, raws, scales, k, -k, [2 * B + start], code)


def test_append_not_finite():
    """A NaN or infinity poisons its (block, head) until the block is started anew, and nothing else."""
    from gemma_b200 import ops  # noqa: F401
    rng = np.random.default_rng(3)
    H, D, B = 2, 32, 16
    for bad in (math.nan, math.inf, -math.inf):
        c, raws, scales = new_cache(3, H, B, D, "int8", 4)
        k, v = values(rng, 2, H, D, "f32"), values(rng, 2, H, D, "f32")
        k[1, 0, 7] = bad
        check_append(c, raws, scales, k, v, [B + 3, B + 4], "int8")
        assert torch.isnan(c.k_scale).cpu().numpy().tolist() == [[False, False], [True, False], [False, False]]
        check_append(c, raws, scales, values(rng, 1, H, D, "f32"), v[:1], [B + 5], "int8")
        assert bool(torch.isnan(c.k_scale[1, 0]))
        check_append(c, raws, scales, values(rng, 2, H, D, "f32"), v, [B, B + 1], "int8")
        assert not bool(torch.isnan(c.k_scale).any())


@pytest.mark.parametrize("dtype, off, pad", [("bf16", 1, 0), ("f32", 3, 1), ("f16", 8, 8), ("f32", 0, 4)])
def test_append_any_alignment(dtype, off, pad):
    rng = np.random.default_rng(off)
    H, D, B, n = 2, 48, 16, 40
    c, raws, scales = new_cache(8, H, B, D, "int8", 9)
    base = torch.randn(2, n * (H * (D + pad) + 5) + off, device="cuda").to(DT[dtype])
    k, v = (torch.as_strided(base[i], (n, H, D), (H * (D + pad) + 5, D + pad, 1), base[i].storage_offset() + off) for i in range(2))
    check_append(c, raws, scales, k, v, [int(x) for x in np.arange(7, 7 + n)], "int8")
    check_append(c, raws, scales, k[:0], v[:0], [], "int8")


# ---------------------------------------------------------------------------------------- attend

class Reader:
    def __init__(self, raws, scales, code, B):
        self.raws, self.scales, self.code, self.B = raws, scales, code, B
        self.blocks, self.heads = raws[0].shape[:2]

    def __call__(self, h, row, keys):
        ids, off = row[keys // self.B], keys % self.B
        k, v = (ref.decode(self.raws[i][ids, h, off], self.code) * self.scales[i][ids, h][:, None] for i in range(2))
        return k, v, self.scales[1][ids, h]


def make_batch(rng, rows, lens, B, H, D, code, width=None, spare=3):
    held = [ref.blocks_of(a, B) for a in lens]
    nb = sum(held) + spare
    c, raws, scales = new_cache(nb, H, B, D, code, int(rng.integers(1 << 30)))
    table = rng.integers(-3, nb + 3, (len(lens), max(held + [1]) + 1 if width is None else width))  # entries behind a request hold anything
    order, at = rng.permutation(nb), 0
    for i, x in enumerate(held):
        table[i, :x] = order[at:at + x]
        at += x
    if code == "e4m3":  # codes behind a request's last token hold anything, NaN among it
        for i, a in enumerate(lens):
            if a % B:
                for r in raws:
                    r[table[i, a // B], :, a % B:] = 0x7f
        for t, r in ((c.k_codes, raws[0]), (c.v_codes, raws[1])):
            t.view(torch.int8).copy_(dev(r.view(np.int8), torch.int8))
    return c, raws, scales, table


def check_attend(rng, rows, lens, heads, c, raws, scales, table, code, dtype, window=0, scale=None, q=None, max_rows=None, max_len=None, tail=3, qmul=2.0):
    from gemma_b200 import ops  # noqa: F401
    B, D = c.block_tokens, c.head_dim
    total = sum(rows)
    cu = np.concatenate([[0], np.cumsum(rows)]).astype(int)
    if q is None:
        q = (torch.randn(total + tail, heads, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(int(rng.integers(1 << 30)))) * qmul).to(DT[dtype])
    max_rows = max(rows) if max_rows is None else max_rows
    max_len = max(lens) if max_len is None else max_len
    out = torch.full_like(q, 7.0)
    sc = D ** -0.5 if scale is None else scale
    got, lse = c.attend(q, dev(cu), dev(lens), dev(table), max_rows=max_rows, max_len=max_len, scale=scale, window=window, out=out, return_lse=True)
    assert got.data_ptr() == out.data_ptr()
    want, wlse, pv, smax, least = ref.attend(f64(q), cu, lens, table, Reader(raws, scales, code, B), B, sc, window, max_rows, max_len)
    o, l = f64(out), f64(lse)
    written = ~np.isnan(wlse)
    assert np.all(o[~written] == 7.0)  # rows behind the batch stay as they were
    ds = smax * (2.0 ** -21 + 2.0 ** -19) + 2.0 ** -22
    w = 0 if dtype == "f32" else 2 * 2.0 ** -11
    tol = (2 * (2 * ds + 2.0 ** -18) + w)[..., None] * pv + HALF_EPS[dtype] * np.abs(want) + (2.0 ** -25 if dtype == "f16" else 0) + 2.0 ** -32 * least
    bad = written[..., None] & ~(np.abs(o - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], np.nanmax(np.abs(o - want) / tol))
    fin = written & np.isfinite(wlse)
    assert np.all(np.isneginf(l[written & ~fin]))
    assert np.all(np.abs(l[fin] - wlse[fin]) <= ds[fin] + 2.0 ** -20 + 2.0 ** -22 * np.abs(wlse[fin]))
    return out, lse


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D, H, G, B", [(256, 1, 4, 16), (128, 2, 4, 64), (64, 2, 2, 32), (80, 1, 3, 16), (16, 1, 1, 128), (192, 1, 8, 32), (112, 2, 16, 16)])
def test_attend_steps(code, dtype, D, H, G, B):
    rng = np.random.default_rng(D + B)
    lens = [1, 641, 0, 15, 16, 17, 130]
    a = make_batch(rng, [1] * 7, lens, B, H, D, code)
    check_attend(rng, [1] * 7, lens, H * G, *a, code, dtype)


@pytest.mark.parametrize("code, dtype", [("int8", "f32"), ("e4m3", "bf16"), ("int8", "f16")])
@pytest.mark.parametrize("window", [0, 1, 5, 16, 100])
@pytest.mark.parametrize("D, H, G", [(64, 2, 2), (128, 1, 5), (256, 1, 4)])
def test_attend_drafts(code, dtype, window, D, H, G):
    """A few rows per request, idle requests, more rows than tokens, windows inside and beyond a step."""
    rng = np.random.default_rng(window)
    rows, lens = [3, 0, 8, 1, 5, 2, 0], [3, 50, 333, 1, 64, 1, 0]
    a = make_batch(rng, rows, lens, 32, H, D, code)
    check_attend(rng, rows, lens, H * G, *a, code, dtype, window=window)


@pytest.mark.parametrize("code, dtype", [("int8", "f32"), ("e4m3", "bf16"), ("int8", "bf16"), ("e4m3", "f16"), ("int8", "f16"), ("e4m3", "f32")])
@pytest.mark.parametrize("rows, lens, window", [([33, 70], [33, 200], 0), ([129], [129], 0), ([64, 1, 0, 40], [300, 9, 30, 20], 0),
                                                ([100, 31], [401, 100], 48), ([257], [300], 7)])
@pytest.mark.parametrize("D, H, G, B", [(128, 1, 4, 64), (64, 2, 1, 16), (256, 1, 4, 16), (96, 1, 3, 32)])
def test_attend_prompts(code, dtype, rows, lens, window, D, H, G, B):
    rng = np.random.default_rng(sum(rows) + D)
    a = make_batch(rng, rows, lens, B, H, D, code)
    check_attend(rng, rows, lens, H * G, *a, code, dtype, window=window)


@pytest.mark.parametrize("code, dtype, D, rows, lens, window", [
    ("int8", "f32", 128, [40, 9], [5000, 2100], 0), ("e4m3", "bf16", 64, [33, 1], [3001, 9000], 0), ("int8", "f16", 256, [34], [2500], 0),
    ("int8", "bf16", 128, [70], [6000], 3000), ("e4m3", "f32", 256, [20, 3], [1100, 4500], 2000)])
def test_attend_long(code, dtype, D, rows, lens, window):
    """Keys over many tiles, several batches of block ids and, for few rows, many steps of a warp; several key ranges."""
    rng = np.random.default_rng(D + sum(lens))
    a = make_batch(rng, rows, lens, 16 if D == 256 else 64, 1, D, code)
    check_attend(rng, rows, lens, 4, *a, code, dtype, window=window)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_many_requests(dtype):
    """More requests than one pass of a CTA's prefix sums takes, many of them without rows or keys."""
    rng = np.random.default_rng(31)
    n = 1300
    rows = [int(x) for x in rng.choice([0, 1, 1, 2], n)]
    lens = [int(x) if x > 3 else int(rows[i] and x) for i, x in enumerate(rng.integers(0, 60, n))]
    a = make_batch(rng, rows, lens, 16, 1, 32, "int8")
    check_attend(rng, rows, lens, 3, *a, "int8", dtype)


@pytest.mark.parametrize("G, rows, lens", [(33, [1, 0, 2], [40, 0, 300]), (1000, [2, 1], [70, 9]), (1024, [1, 1], [1, 200])])
@pytest.mark.parametrize("code, dtype, D", [("int8", "f32", 64), ("e4m3", "bf16", 256), ("int8", "f16", 128)])
def test_attend_wide_groups(code, dtype, D, G, rows, lens):
    """More query heads to a key head than a tile has rows: tokens begin and end inside tiles."""
    rng = np.random.default_rng(G + D)
    a = make_batch(rng, rows, lens, 16, 1, D, code)
    check_attend(rng, rows, lens, G, *a, code, dtype)


def test_attend_bad_pages():
    """Block ids outside the cache hide their keys; a request with no valid block gives zeros."""
    rng = np.random.default_rng(1)
    rows, lens = [1, 2, 40], [100, 64, 90]
    c, raws, scales, table = make_batch(rng, rows, lens, 16, 1, 64, "int8")
    table[0, 2], table[0, 6] = -1, 10 ** 6
    table[1, :4] = [c.num_blocks, -5, 2 ** 31 - 1, -2 ** 31]
    table[2, 3] = -1
    for dtype in ("f32", "bf16"):
        check_attend(rng, rows, lens, 4, c, raws, scales, table, "int8", dtype)


def test_attend_limits_cut():
    """max_rows and max_len below the batch's own: rows behind are not written, keys behind not read."""
    rng = np.random.default_rng(6)
    rows, lens = [5, 2, 9], [80, 40, 60]
    a = make_batch(rng, rows, lens, 16, 2, 64, "int8")
    for dtype in ("f32", "f16"):
        check_attend(rng, rows, lens, 4, *a, "int8", dtype, max_rows=3, max_len=48)
        check_attend(rng, rows, lens, 4, *a, "int8", dtype, max_rows=40, max_len=96)
        check_attend(rng, rows, lens, 4, *a, "int8", dtype, max_rows=9, max_len=0)


@pytest.mark.parametrize("group, last", [(2, [2 ** 31 - 1]), (16, [])])
def test_attend_bad_cu_rows(group, last):
    """cu_rows that do not ascend, below zero and beyond the batch: no access outside of it, and the
    requests whose own two entries are right (rows 5 to 7 and 0 to 2) have their results."""
    rng = np.random.default_rng(group)
    lens = [40, 20, 30, 25, 9][:4 + len(last)]
    c, raws, scales, table = make_batch(rng, None, lens, 16, 1, 64, "int8")
    cu = [5, 8, -2 ** 31, 0, 3] + last
    guarded = torch.full((30, group, 64), 7.0, device="cuda")
    out, q = guarded[10:20], torch.randn(10, group, 64, device="cuda")
    c.attend(q, dev(cu), dev(lens), dev(table), max_rows=2 if last else 80, max_len=40, out=out)
    n = 2 if last else 3
    for first, i in ((5, 0), (0, 3)):
        want = c.attend(q[first:first + 3], dev([0, 3]), dev(lens[i:i + 1]), dev(table[i:i + 1]), max_rows=n, max_len=40)
        assert torch.equal(out[first:first + n], want[:n])
    assert bool((out[8:] == 7.0).all()) and bool((guarded[:10] == 7.0).all()) and bool((guarded[20:] == 7.0).all())
    if last:  # its rows are more than its tokens: they see nothing
        assert bool((out[3:5] == 0.0).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows, lens", [([1, 1], [700, 300]), ([40], [300])])
def test_attend_scales_far_apart(dtype, rows, lens):
    """Blocks whose scales differ by 2^40 share one running sum."""
    rng = np.random.default_rng(7)
    c, raws, scales, table = make_batch(rng, rows, lens, 16, 1, 64, "int8")
    for s, t in zip(scales, (c.k_scale, c.v_scale)):
        s[:] = 2.0 ** (rng.integers(-8, -4, s.shape) if s is scales[0] else rng.integers(-30, 10, s.shape))
        t.copy_(dev(s, torch.float32))
    check_attend(rng, rows, lens, 4, c, raws, scales, table, "int8", dtype)


@pytest.mark.parametrize("rows, lens", [([1, 1], [90, 300]), ([36], [300])])
def test_attend_large_and_zero_queries(rows, lens):
    """Queries of very different sizes in one tile: each row is scaled by itself."""
    rng = np.random.default_rng(9)
    a = make_batch(rng, rows, lens, 16, 2, 128, "int8")
    total = sum(rows)
    q = torch.randn(total, 4, 128, device="cuda")
    q *= (10.0 ** torch.linspace(-30, 1, total * 4, device="cuda")).reshape(total, 4, 1)
    q[0, 1] = 0
    check_attend(rng, rows, lens, 4, *a, "int8", "f32", q=q)
    check_attend(rng, rows, lens, 4, *a, "int8", "bf16", q=q.bfloat16())
    check_attend(rng, rows, lens, 4, *a, "int8", "f32", q=q, scale=-0.3)


@pytest.mark.parametrize("rows, lens", [([1, 2], [40, 70]), ([40, 2], [100, 40])])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attend_not_finite_stays_in_its_rows(rows, lens, dtype):
    """A NaN query gives NaN in its own row and head; a poisoned block in the rows that see it."""
    rng = np.random.default_rng(4)
    c, raws, scales, table = make_batch(rng, rows, lens, 16, 1, 64, "int8")
    q = torch.randn(sum(rows), 4, 64, device="cuda").to(DT[dtype])
    cu = dev(np.concatenate([[0], np.cumsum(rows)]))
    call = lambda x, **kw: c.attend(x, cu, dev(lens), dev(table), max_rows=max(rows), max_len=max(lens), **kw)  # noqa: E731
    clean = call(q)
    x = q.clone()
    x[1, 2, 5] = math.nan
    x[0, 0, 0] = math.inf
    got = call(x)
    bad = torch.isnan(got).all(-1)
    assert bad.nonzero().tolist() == [[0, 0], [1, 2]]
    assert torch.equal(got[~bad], clean[~bad])
    # the last block of request 1: seen by its last row only under a window that starts in it
    c.v_scale[int(table[1, (lens[1] - 1) // 16]), 0] = math.nan
    got = call(q)
    seen = torch.isnan(got).all(-1).all(-1)
    last = [r for r in range(rows[0], sum(rows)) if lens[1] - rows[1] + r - rows[0] >= (lens[1] - 1) // 16 * 16]
    assert seen.nonzero().flatten().tolist() == last
    keep = [r for r in range(sum(rows)) if r not in last]
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("rows, lens", [([1, 4], [90, 300]), ([36, 3], [300, 5])])
@pytest.mark.parametrize("dtype, off", [("f32", 1), ("bf16", 3), ("f16", 8)])
def test_attend_strided(rows, lens, dtype, off):
    """Queries inside a fused projection at odd offsets, output heads and rows apart."""
    rng = np.random.default_rng(off)
    H, G, D = 2, 2, 64
    c, raws, scales, table = make_batch(rng, rows, lens, 16, H, D, "e4m3")
    total = sum(rows)
    base = torch.randn(total * 500 + off, device="cuda").to(DT[dtype])
    q = torch.as_strided(base, (total, 4, D), (500, 65, 1), off)
    check_attend(rng, rows, lens, 4, c, raws, scales, table, "e4m3", dtype, q=q)
    want = c.attend(q, dev(np.concatenate([[0], np.cumsum(rows)])), dev(lens), dev(table), max_rows=max(rows), max_len=max(lens))
    room = torch.full((total * 431 + off,), 7.0, device="cuda").to(DT[dtype])
    out = torch.as_strided(room, (total, 4, D), (431, 71, 1), off)
    c.attend(q, dev(np.concatenate([[0], np.cumsum(rows)])), dev(lens), dev(table), max_rows=max(rows), max_len=max(lens), out=out)
    assert torch.equal(out, want)
    out.fill_(7.0)
    assert bool((room == 7.0).all())


def test_attend_refuses():
    rng = np.random.default_rng(1)
    c, _, _, table = make_batch(rng, [1], [30], 16, 2, 64, "int8")
    q, cu, lens, t = torch.zeros(1, 4, 64, device="cuda"), dev([0, 1]), dev([30]), dev(table)
    ok = dict(max_rows=1, max_len=30)
    c.attend(q, cu, lens, t, **ok)
    for bad, match in ((lambda: c.attend(q[..., :32], cu, lens, t, **ok), "head_dim"), (lambda: c.attend(q, cu[:1], lens, t, **ok), "cu_rows"),
                       (lambda: c.attend(q, cu, lens.long(), t, **ok), "int32"), (lambda: c.attend(q, cu, lens, t.t(), **ok), "table"),
                       (lambda: c.attend(q, cu, lens, t, max_rows=1, max_len=1000), "max_len"), (lambda: c.attend(q.double(), cu, lens, t, **ok), "float64"),
                       (lambda: c.attend(q, cu.cpu(), lens, t, **ok), "CUDA"), (lambda: c.attend(q.requires_grad_(), cu, lens, t, **ok), "gradient")):
        with pytest.raises(ValueError, match=match):
            bad()
    from gemma_b200 import ops
    q = q.detach()
    with pytest.raises(ops.GemmaB200Error, match="query heads"):
        c.attend(q[:, :3], cu, lens, t, **ok)
    with pytest.raises(ops.GemmaB200Error, match="workspace"):
        big = c.workspace_bytes(q, 1, 1, 5000)
        wide = torch.zeros(1, 400, dtype=torch.int32, device="cuda")
        c.attend(q, cu, lens, wide, max_rows=1, max_len=5000, workspace=torch.empty(big - 1, dtype=torch.uint8, device="cuda"))


# ------------------------------------------------------------------------- a run of them together

def serve(steps, code, dtype, capture=False):
    """A small serving loop through all four operators, checked against the references at every step."""
    from gemma_b200 import ops
    rng = np.random.default_rng(21)
    H, G, D, B, width, n, rows = 2, 2, 64, 16, 6, 4, 48
    c, raws, scales = new_cache(14, H, B, D, code, 2)
    reader = Reader(raws, scales, code, B)
    table, free, count = np.full((n, width), -1), np.arange(14), 14
    t, fl, fc = dev(table), dev(free), dev([count])
    freqs, m = ops.rope_frequencies(48, 1e4, "linear", 8.0)
    old = [0] * n
    x = torch.zeros(rows, H * G + 2 * H, D, device="cuda", dtype=DT[dtype])
    d_old, d_new = dev(old), dev(old)

    def step():
        p = ops.plan_blocks(d_old, d_new, t, fl, fc, B, rows)
        q, k = ops.rope(x[:, :H * G], x[:, H * G:H * G + H], p.positions, freqs, mscale=m)
        c.append(k, x[:, H * G + H:], p.slots)
        out = c.attend(q, p.cu_rows, p.lens, t, max_rows=rows, max_len=width * B)
        fc.copy_(p.free_count)
        return p, q, k, out

    graph = None
    for i, new in enumerate(steps):
        x.copy_(torch.randn(x.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)).to(x.dtype))
        d_old.copy_(dev(old))
        d_new.copy_(dev(new))
        if capture and graph is None:
            keep = [v.clone() for v in (t, fl, fc, c.k_codes.view(torch.int8), c.v_codes.view(torch.int8), c.k_scale, c.v_scale)]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                result = step()
            for a, b in zip((t, fl, fc, c.k_codes.view(torch.int8), c.v_codes.view(torch.int8), c.k_scale, c.v_scale), keep):
                a.copy_(b)
        if graph is not None:
            graph.replay()
            p, q, k, out = result
        else:
            p, q, k, out = step()
        want, table, free = ref.plan(old, new, table, free, count, B, rows)
        count = want["free_count"]
        for name in ("cu_rows", "lens", "row_seq", "positions", "slots"):
            assert np.array_equal(getattr(p, name).cpu().numpy(), want[name]), (i, name)
        assert int(p.status) == want["status"]
        for src, turned in ((x[:, :H * G], q), (x[:, H * G:H * G + H], k)):
            r = ref.rope(f64(src), want["positions"], f64(freqs), "half", m, False)
            assert np.all(np.abs(f64(turned) - r) <= 16 * HALF_EPS[dtype] * 8)
        for j, v in enumerate((k, x[:, H * G + H:])):
            ref.append(raws[j], scales[j], f64(v), list(want["slots"]), code)
        assert np.array_equal(raw(c.k_codes), raws[0]) and np.array_equal(raw(c.v_codes), raws[1])
        r, _, pv, smax, least = ref.attend(f64(q), want["cu_rows"], want["lens"], table, reader, B, D ** -0.5, 0, rows, width * B)
        live = want["cu_rows"][-1]
        tol = (2 * (smax * 2.0 ** -18 + 2.0 ** -17) + 2.0 ** -10 * (dtype != "f32"))[..., None] * pv + HALF_EPS[dtype] * np.abs(r) + 2.0 ** -32 * least
        assert np.all(np.abs(f64(out) - r)[:live] <= tol[:live]), i
        old = [int(v) for v in want["lens"]]
    return old


STEPS = [[20, 0, 3, 0], [21, 7, 4, 0], [22, 8, 5, 33], [23, 9, 0, 34], [20, 10, 1, 35], [21, 11, 40, 36], [60, 60, 60, 60], [22, 12, 41, 37], [0, 0, 0, 0], [5, 6, 7, 8]]


@pytest.mark.parametrize("code, dtype", [("int8", "f32"), ("e4m3", "bf16")])
@pytest.mark.parametrize("capture", [False, True])
def test_serving_steps(code, dtype, capture):
    """Prompts, single tokens, an ended request, a taken-back draft, a step that finds too few blocks
    (and changes nothing), eager and captured into one graph that is replayed for every step."""
    assert serve(STEPS, code, dtype, capture) == [5, 6, 7, 8]


def test_two_streams_at_once():
    """Two calls at the same time on two streams, each with its own workspace."""
    rng = np.random.default_rng(12)
    rows, lens = [1] * 3, [4000, 900, 2500]
    c, raws, scales, table = make_batch(rng, rows, lens, 16, 1, 128, "int8")
    cu, ln, tb = dev([0, 1, 2, 3]), dev(lens), dev(table)
    qs = [torch.randn(3, 4, 128, device="cuda") for _ in range(2)]
    want = [c.attend(q, cu, ln, tb, max_rows=1, max_len=4000) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(c.attend(qs[i], cu, ln, tb, max_rows=1, max_len=4000))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])  # and the result does not depend on the order of its parts


@pytest.mark.parametrize("D, dtype", [(64, "bf16"), (128, "f32")])
def test_two_streams_of_prompts_at_once(D, dtype):
    """Two calls with many rows at the same time: their CTAs take turns on the SMs' tensor memory."""
    rng = np.random.default_rng(D)
    rows, lens = [300, 90], [900, 400]
    c, raws, scales, table = make_batch(rng, rows, lens, 16, 2, D, "int8")
    cu, ln, tb = dev([0, 300, 390]), dev(lens), dev(table)
    qs = [torch.randn(390, 8, D, device="cuda").to(DT[dtype]) for _ in range(2)]
    want = [c.attend(q, cu, ln, tb, max_rows=300, max_len=900) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(c.attend(qs[i], cu, ln, tb, max_rows=300, max_len=900))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])
