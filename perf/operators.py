"""Cases and plain forms of the serving operators around a paged 8-bit key/value cache.

Four operators, in the order a serving step runs them:

* ``plan``    block tables, the slot of every new row and its position, from request lengths;
* ``rope``    rotary positions on the new queries and keys (and the gradient's way back);
* ``append``  new key and value rows quantised into the cache, a power-of-two scale per block and head;
* ``attend``  attention of ragged query rows over the cached rows of their sequence.

``run`` computes them with elementary torch operations, or (``own``) through ``gemma_b200.ops``.
"""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
MIN_EXP = -60  # the smallest scale exponent of a block

_ops = None


def ops():
    """gemma_b200.ops, imported on the first call that needs it."""
    global _ops
    if _ops is None:
        sys.path.insert(0, os.path.join(ROOT, "webgpu-gemma_b200"))
        from gemma_b200 import ops as module
        _ops = module
    return _ops


# --------------------------------------------------------------------------------------- cases

def listed():
    return [
        # One decode step of 64 conversations (the batched-decode benchmark's shape): each grows by one token.
        dict(name="plan_step_64", op="plan", seqs=64, block=16, len_lo=1, len_hi=2047, chunk=1, prompts=0.0, ends=0.0,
             backs=0.0, rows=64, shape_seed=1),
        # A scheduler's step over 1000 requests: decodes, prompt chunks, finished requests, rejected drafts.
        dict(name="plan_mixed_1000", op="plan", seqs=1000, block=32, len_lo=0, len_hi=4096, chunk=512, prompts=0.1,
             ends=0.05, backs=0.05, rows=32768, shape_seed=2),
        # One decode step of 64 conversations of the 1B model: 4 query heads and 1 key head of 256, f32.
        dict(name="rope_step_64", op="rope", rows=64, heads=4, kv_heads=1, head_dim=256, rot=256, layout="half",
             scaling="linear", factor=8.0, theta=1e6, pos_hi=2048, dtype="f32", back=False),
        # A long prompt in bf16 whose context was stretched four times.
        dict(name="rope_prompt_8192", op="rope", rows=8192, heads=32, kv_heads=8, head_dim=128, rot=128, layout="half",
             scaling="yarn", factor=4.0, theta=1e6, pos_hi=131072, dtype="bf16", back=False),
        # The gradient of a training batch with interleaved pairs on half of each head, an odd number of rows.
        dict(name="rope_back_2047", op="rope", rows=2047, heads=16, kv_heads=16, head_dim=96, rot=48,
             layout="interleaved", scaling="none", factor=1.0, theta=1e4, pos_hi=2047, dtype="f16", back=True),
        # The 64 new rows of a decode step, each into a block that holds earlier tokens.
        dict(name="append_step_64", op="append", seqs=64, rows_lo=1, rows_hi=1, len_lo=0, len_hi=2047, kv_heads=1,
             head_dim=256, block=16, code="int8", dtype="f32", pad=0, shape_seed=3),
        # Prompt chunks of several requests and a few padded rows, 8 key heads of 128.
        dict(name="append_prompt_8192", op="append", seqs=9, rows_lo=100, rows_hi=1700, len_lo=0, len_hi=1000,
             kv_heads=8, head_dim=128, block=64, code="e4m3", dtype="bf16", pad=37, shape_seed=4),
        # One conversation of the 1B model in the middle of its benchmark: the smallest step, latency counts.
        dict(name="attend_step_1", op="attend", seqs=1, rows_lo=1, rows_hi=1, len_lo=641, len_hi=641, heads=4,
             kv_heads=1, head_dim=256, block=16, code="int8", dtype="f32", window=0, empty=0, shape_seed=5),
        # 64 conversations of very different lengths in one decode step of the 1B model.
        dict(name="attend_step_64", op="attend", seqs=64, rows_lo=1, rows_hi=1, len_lo=100, len_hi=8192, heads=4,
             kv_heads=1, head_dim=256, block=16, code="int8", dtype="f32", window=0, empty=0, shape_seed=6),
        # Four conversations over very long contexts, 8 key heads shared by 4 query heads each.
        dict(name="attend_long_4", op="attend", seqs=4, rows_lo=1, rows_hi=1, len_lo=100000, len_hi=131072, heads=32,
             kv_heads=8, head_dim=128, block=64, code="e4m3", dtype="bf16", window=0, empty=0, shape_seed=7),
        # Drafts of 1 to 8 tokens checked under a sliding window, some requests idle.
        dict(name="attend_drafts_16", op="attend", seqs=16, rows_lo=1, rows_hi=8, len_lo=9, len_hi=2000, heads=16,
             kv_heads=8, head_dim=64, block=32, code="int8", dtype="f16", window=512, empty=3, shape_seed=8),
        # Prompt chunks of two requests behind their earlier turns.
        dict(name="attend_prompt_2", op="attend", seqs=2, rows_lo=1531, rows_hi=2048, len_lo=4000, len_hi=8192,
             heads=32, kv_heads=8, head_dim=128, block=64, code="int8", dtype="bf16", window=0, empty=0, shape_seed=9),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "rope", "append", "attend", "attend"])
    top = [work(c) for c in listed() if c["op"] == op]
    top = {k: max(w[k] for w in top) for k in ("bytes", "flops")}
    while True:
        c = _draw_plan(rng) if op == "plan" else _draw_rope(rng) if op == "rope" else \
            _draw_append(rng) if op == "append" else _draw_attend(rng)
        w = work(c)
        if w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"] and _padded(c) <= 1 << 30:
            return c


def _padded(c):
    """What the plain form of attend spreads out: a score for each pair of padded rows and keys, a value for each cached number."""
    if c["op"] != "attend":
        return 0
    return c["seqs"] * c["len_hi"] * max(c["heads"] * c["rows_hi"], 2 * c["kv_heads"] * c["head_dim"])


def _draw_plan(rng):
    n = _log(rng, 1, 1000)
    decode = rng.random() < 0.4
    chunk = 1 if decode else _log(rng, 2, 512)
    prompts = 0.0 if decode else rng.uniform(0.02, 0.4)
    rows = n if decode else min(32768, n * chunk)
    return dict(op="plan", seqs=n, block=rng.choice([16, 32, 64, 128]), len_lo=rng.choice([0, 1]), len_hi=_log(rng, 40, 8000),
                chunk=chunk, prompts=prompts, ends=0.0 if decode else rng.uniform(0, 0.1),
                backs=0.0 if decode else rng.uniform(0, 0.1), rows=rows, shape_seed=rng.randrange(1 << 30))


def _draw_rope(rng):
    d = rng.choice([64, 80, 96, 128, 192, 256])
    kv = rng.choice([1, 2, 4, 8])
    return dict(op="rope", rows=_log(rng, 1, 8192), heads=kv * rng.choice([1, 2, 3, 4, 8]), kv_heads=kv, head_dim=d,
                rot=rng.choice([d, d, d // 2, 2 * (d // 6)]), layout=rng.choice(["half", "interleaved"]),
                scaling=rng.choice(["none", "linear", "bands", "yarn"]), factor=rng.choice([2.0, 4.0, 8.0]),
                theta=rng.choice([1e4, 1e6]), pos_hi=_log(rng, 500, 1000000), dtype=rng.choice(["f32", "bf16", "f16"]),
                back=rng.random() < 0.3)


def _draw_append(rng):
    step = rng.random() < 0.5
    hi = 1 if step else _log(rng, 2, 1700)
    return dict(op="append", seqs=_log(rng, 1, 200 if step else 16), rows_lo=1, rows_hi=hi, len_lo=0,
                len_hi=_log(rng, 10, 2000), kv_heads=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 80, 96, 128, 256]),
                block=rng.choice([16, 32, 64, 128]), code=rng.choice(["int8", "e4m3"]), dtype=rng.choice(["f32", "bf16", "f16"]),
                pad=rng.choice([0, 0, 5]), shape_seed=rng.randrange(1 << 30))


def _draw_attend(rng):
    kv = rng.choice([1, 2, 4, 8])
    kind = rng.choice(["step", "step", "drafts", "prompt"])
    rows_hi = 1 if kind == "step" else _log(rng, 2, 16) if kind == "drafts" else _log(rng, 30, 2048)
    n = _log(rng, 1, 128) if kind != "prompt" else _log(rng, 1, 8)
    hi = max(rows_hi + 1, _log(rng, 30, 131072 if kind == "step" else 16384))
    return dict(op="attend", seqs=n, rows_lo=1 if kind != "prompt" else max(1, rows_hi // 2), rows_hi=rows_hi,
                len_lo=rows_hi + (hi - rows_hi) // rng.choice([2, 8, 100]), len_hi=hi, heads=kv * rng.choice([1, 2, 4, 4, 8]),
                kv_heads=kv, head_dim=rng.choice([64, 80, 96, 128, 128, 256, 256]), block=rng.choice([16, 32, 64, 128]),
                code=rng.choice(["int8", "e4m3"]), dtype=rng.choice(["f32", "bf16", "f16"]),
                window=rng.choice([0, 0, 0, 100, 512]), empty=rng.choice([0, 0, 1]) if n > 1 else 0,
                shape_seed=rng.randrange(1 << 30))


# ------------------------------------------------------------------------- lengths, work, inputs

def _ceil(a, b):
    return -(-a // b)


def _plan_lengths(case):
    """(old, new) length of every request: a property of the case."""
    r = random.Random(case["shape_seed"])
    old, new, rows = [], [], 0
    for _ in range(case["seqs"]):
        a = r.randint(case["len_lo"], case["len_hi"])
        x = r.random()
        if x < case["prompts"]:
            b = a + r.randint(1, case["chunk"])
        elif x < case["prompts"] + case["ends"]:
            b = 0
        elif x < case["prompts"] + case["ends"] + case["backs"]:
            b = max(0, a - r.randint(1, 8))
        else:
            b = a + 1
        if b > a and rows + b - a > case["rows"]:
            b = a
        rows += max(0, b - a)
        old.append(a)
        new.append(b)
    return old, new


def _row_lengths(case):
    """(new rows, length with them) of every request: a property of the case."""
    r = random.Random(case["shape_seed"])
    rows, lens = [], []
    for i in range(case["seqs"]):
        n = r.randint(case["rows_lo"], case["rows_hi"])
        a = r.randint(case["len_lo"], case["len_hi"])
        if case["op"] == "append":
            a += n
        elif i < case["empty"]:
            n, a = 0, (0 if i % 2 else a)
        rows.append(n)
        lens.append(max(a, n))
    return rows, lens


def work(case):
    op = case["op"]
    if op == "plan":
        old, new = _plan_lengths(case)
        rows = sum(max(0, b - a) for a, b in zip(old, new))
        blocks = sum(abs(_ceil(b, case["block"]) - _ceil(a, case["block"])) for a, b in zip(old, new))
        # lengths in; cumulative rows and lengths out; three words for each row of the padded batch; a block moved is read and written
        return {"bytes": 4.0 * (2 * len(old) + 2 * len(old) + 3 * case["rows"] + 2 * blocks), "flops": float(rows)}
    if op == "rope":
        n = case["rows"] * (case["heads"] + case["kv_heads"])
        return {"bytes": float(2 * n * case["head_dim"] * BYTES[case["dtype"]] + 4 * case["rows"] + 4 * case["rot"]),
                "flops": 3.0 * n * case["rot"]}
    rows, lens = _row_lengths(case)
    H, D = case["kv_heads"], case["head_dim"]
    if op == "append":
        n = sum(rows) * H * D * 2
        return {"bytes": float(n * BYTES[case["dtype"]] + n + 4 * sum(rows)), "flops": 3.0 * n}
    W, keys, pairs = case["window"], 0, 0
    for n, a in zip(rows, lens):
        first = a - n  # position of the first row
        if n:
            keys += a - (max(0, first - W + 1) if W else 0)
            if not W:
                pairs += n * first + n * (n + 1) // 2
            else:
                pairs += sum(min(W, p + 1) for p in range(first, a))
    b = 2 * keys * H * D + 2 * 4 * _ceil(keys, case["block"]) * H + 2 * sum(rows) * case["heads"] * D * BYTES[case["dtype"]]
    return {"bytes": float(b), "flops": 4.0 * pairs * case["heads"] * D}


def _exponent(amax, code):
    """Smallest e >= MIN_EXP with amax <= 127 * 2^e (int8) or 448 * 2^e (e4m3), in 32 bits without a rounding."""
    m, x = torch.frexp(amax)
    e = x - 7 + (m > 127 / 128).int() if code == "int8" else x - 9 + (m > 448 / 512).int()
    return torch.where(amax > 0, e, torch.full_like(e, MIN_EXP)).clamp(min=MIN_EXP)


def _encode(x, code):
    """Values already divided by their scale -> codes."""
    return x.round().to(torch.int8) if code == "int8" else x.to(torch.float8_e4m3fn)


def _pow2(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)


def _filled(num_blocks, H, B, D, code, g):
    """A cache's codes and scales as earlier calls left them: [block][head][token][dim]."""
    codes = torch.empty(num_blocks, H, B, D, dtype=torch.int8 if code == "int8" else torch.float8_e4m3fn, device="cuda")
    scale = torch.empty(num_blocks, H, dtype=torch.float32, device="cuda")
    step = max(1, (1 << 26) // (H * B * D))
    for b in range(0, num_blocks, step):
        n = min(step, num_blocks - b)
        x = torch.randn(n, H, B, D, device="cuda", generator=g)
        x *= torch.exp2(torch.rand(n, H, 1, 1, device="cuda", generator=g) * 2 - 1)
        e = _exponent(x.abs().amax((2, 3)), code)
        codes[b:b + n] = _encode(x * _pow2(-e)[:, :, None, None], code)
        scale[b:b + n] = _pow2(e)
    return codes, scale


def _table(lens, block, num_blocks, g):
    """Block table [request][block] of blocks handed out in random order; -1 where a request has none."""
    width = max(1, max(_ceil(a, block) for a in lens))
    order = torch.randperm(num_blocks, device="cuda", generator=g).int()
    has = torch.tensor([_ceil(a, block) for a in lens], device="cuda")
    mask = torch.arange(width, device="cuda")[None, :] < has[:, None]
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    table[mask] = order[:sum(_ceil(a, block) for a in lens)]
    return table


def _frequencies(case):
    """Radians per position of each rotated pair, in 64 bits, and the factor on cos and sin."""
    r, f = case["rot"], case["factor"]
    i = torch.arange(r // 2, dtype=torch.float64)
    w = case["theta"] ** (-2 * i / r)
    if case["scaling"] == "linear":
        return w / f, 1.0
    if case["scaling"] == "bands":  # slow pairs / f, fast pairs kept, a ramp between wavelengths 8192/1 and 8192/4
        t = ((8192 * w / (2 * math.pi) - 1) / 3).clamp(0, 1)
        return w * (t + (1 - t) / f), 1.0
    if case["scaling"] == "yarn":  # pairs between 32 and 1 turns in the 32768 trained positions are ramped
        def pair(turns):
            return r * math.log(32768 / (turns * 2 * math.pi)) / (2 * math.log(case["theta"]))
        lo, hi = max(0, math.floor(pair(32))), min(r - 1, math.ceil(pair(1)))
        t = 1 - ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return w * (t + (1 - t) / f), 0.1 * math.log(f) + 1
    return w, 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], dict(case)
    i32 = dict(dtype=torch.int32, device="cuda")
    if op == "plan":
        old, new = _plan_lengths(case)
        B = case["block"]
        width = max(_ceil(max(a, b), B) for a, b in zip(old, new)) + 1
        held = [_ceil(a, B) for a in old]
        spare = sum(max(0, _ceil(b, B) - _ceil(a, B)) for a, b in zip(old, new)) + 100
        order = torch.randperm(sum(held) + spare, device="cuda", generator=g).int()
        s["table"] = torch.full((len(old), width), -1, **i32)
        s["table"][torch.arange(width, device="cuda")[None, :] < torch.tensor(held, device="cuda")[:, None]] = order[:sum(held)]
        s["free"] = torch.cat([order[sum(held):], torch.full((sum(held),), -1, **i32)])
        s["free_count"] = torch.tensor([spare], **i32)
        s["old"], s["new"] = torch.tensor(old, **i32), torch.tensor(new, **i32)
        return s
    dt = DTYPES[case["dtype"]]
    if op == "rope":
        # rows of a fused projection: queries, keys and values side by side
        H, K, D = case["heads"], case["kv_heads"], case["head_dim"]
        x = torch.randn(case["rows"], H + 2 * K, D, device="cuda", generator=g).to(dt)
        s["q"], s["k"] = x[:, :H], x[:, H:H + K]
        s["positions"] = torch.randint(0, case["pos_hi"], (case["rows"],), device="cuda", generator=g).int()
        f, m = _frequencies(case)
        s["freqs"], s["mscale"] = f.cuda(), m
        return s
    rows, lens = _row_lengths(case)
    B, H, D = case["block"], case["kv_heads"], case["head_dim"]
    num_blocks = sum(_ceil(a, B) for a in lens) + 4
    s["kc"], s["ks"] = _filled(num_blocks, H, B, D, case["code"], g)
    s["vc"], s["vs"] = _filled(num_blocks, H, B, D, case["code"], g)
    s["table"] = _table(lens, B, num_blocks, g)
    total = sum(rows)
    if op == "append":
        x = torch.randn(total + case["pad"], 2 * H, D, device="cuda", generator=g)
        x *= torch.exp2(torch.rand(total + case["pad"], 2 * H, 1, device="cuda", generator=g) * 3 - 1)
        x = x.to(dt)
        s["k"], s["v"] = x[:, :H], x[:, H:]
        seq = [i for i, n in enumerate(rows) for _ in range(n)]
        pos = torch.tensor([lens[i] - n + j for i, n in enumerate(rows) for j in range(n)], dtype=torch.int64, device="cuda")
        slot = s["table"][torch.tensor(seq, device="cuda"), pos // B] * B + pos % B
        s["slots"] = torch.cat([slot.int(), torch.full((case["pad"],), -1, **i32)])
    else:
        s["q"] = (torch.randn(total, case["heads"], D, device="cuda", generator=g) * 2).to(dt)
        s["cu_rows"] = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], **i32)
        s["lens"] = torch.tensor(lens, **i32)
        s["scale"], s["max_rows"], s["max_len"] = D ** -0.5, max(rows), max(lens)
    if own:  # the handle that a serving program makes once for its cache
        s["cache"] = ops().KV8Cache(s["kc"], s["vc"], s["ks"], s["vs"])
    return s


# ------------------------------------------------------------------------------- one pass

def run(s):
    op = s["op"]
    if own:
        m = ops()
        if op == "plan":
            p = m.plan_blocks(s["old"], s["new"], s["table"], s["free"], s["free_count"], s["block"], s["rows"])
            return {"cu_rows": p.cu_rows, "lens": p.lens, "seq": p.row_seq, "pos": p.positions, "slots": p.slots,
                    "free_count": p.free_count, "status": p.status, "table": s["table"], "free": s["free"]}
        if op == "rope":
            q, k = m.rope(s["q"], s["k"], s["positions"], s["freqs"], layout=s["layout"], mscale=s["mscale"], inverse=s["back"])
            return {"q": q, "k": k}
        if op == "append":
            s["cache"].append(s["k"], s["v"], s["slots"])
            return {"kc": s["kc"], "vc": s["vc"], "ks": s["ks"], "vs": s["vs"]}
        out, lse = s["cache"].attend(s["q"], s["cu_rows"], s["lens"], s["table"], max_rows=s["max_rows"], max_len=s["max_len"],
                                     scale=s["scale"], window=s["window"], return_lse=True)
        return {"out": out, "lse": lse}
    return _plan(s) if op == "plan" else _rope(s) if op == "rope" else _append(s) if op == "append" else _attend(s)


def _plan(s):
    B, rows, table, free = s["block"], s["rows"], s["table"], s["free"]
    old, new, count = s["old"].long(), s["new"].long(), s["free_count"].long()
    n, width = table.shape
    dev = table.device
    hold, want = (old + B - 1) // B, (new + B - 1) // B
    take, give = (want - hold).clamp(min=0), (hold - want).clamp(min=0)
    grow = (new - old).clamp(min=0)
    status = (take.sum() > count[0] + give.sum()).long() + 2 * (want > width).any().long() + 4 * (grow.sum() > rows).long() \
        + 8 * ((old < 0) | (new < 0) | (hold > width)).any().long()
    ok = status == 0
    b = torch.arange(width, device=dev)[None, :]
    # given back, request by request in block order, on top of the stack
    given = ok & (b >= want[:, None]) & (b < hold[:, None])
    at = count + (give.cumsum(0) - give)[:, None] + b - want[:, None]
    list_ = torch.cat([free, free.new_zeros(1)]).scatter(0, torch.where(given, at, free.numel()).reshape(-1), table.reshape(-1))[:-1]
    # taken from the top, request by request in block order
    taken = ok & (b >= hold[:, None]) & (b < want[:, None])
    at = count + give.sum() - 1 - ((take.cumsum(0) - take)[:, None] + b - hold[:, None])
    table2 = torch.where(taken, list_[at.clamp(0, free.numel() - 1)], table)
    cu = torch.cat([grow.new_zeros(1), grow.cumsum(0)]) * ok
    r = torch.arange(rows, device=dev)
    seq = torch.searchsorted(cu[1:].contiguous(), r, right=True)
    live = r < cu[-1]
    i = seq.clamp(max=n - 1)
    pos = old[i] + r - cu[i]
    slot = table2[i, (pos // B).clamp(0, width - 1)].long() * B + pos % B
    return {"cu_rows": cu.int(), "lens": torch.where(ok, new, old).int(), "seq": torch.where(live, seq, -1).int(),
            "pos": torch.where(live, pos, -1).int(), "slots": torch.where(live, slot, -1).int(),
            "free_count": (count + (give.sum() - take.sum()) * ok).int(), "status": status.int().reshape(1), "table": table2, "free": list_}


def _rope(s):
    r, half = s["rot"], s["rot"] // 2
    angle = s["positions"].double()[:, None] * s["freqs"][None, :]
    c = (angle.cos() * s["mscale"]).float()[:, None, :]
    d = (angle.sin() * (-s["mscale"] if s["back"] else s["mscale"])).float()[:, None, :]

    def turn(x):
        y = x.float()
        a, b = (y[..., :half], y[..., half:r]) if s["layout"] == "half" else (y[..., 0:r:2], y[..., 1:r:2])
        u, v = a * c - b * d, b * c + a * d
        first = torch.cat([u, v], -1) if s["layout"] == "half" else torch.stack([u, v], -1).flatten(-2)
        return torch.cat([first, y[..., r:]], -1).to(x.dtype)

    return {"q": turn(s["q"]), "k": turn(s["k"])}


def _append(s):
    B, H, D, code, slots = s["block"], s["kv_heads"], s["head_dim"], s["code"], s["slots"].long()
    nb = s["kc"].shape[0]
    block = torch.where(slots >= 0, slots // B, nb)  # padded rows go to a block of their own behind the cache
    off = torch.where(slots >= 0, slots % B, 0)
    first = torch.full((nb + 1,), B, device=slots.device).scatter_reduce(0, block, off, "amin")[:nb]  # B: not touched
    token = torch.arange(B, device=slots.device)

    def put(x, codes, scale):
        x = x.float()
        amax = torch.zeros(nb + 1, H, device=x.device).scatter_reduce(0, block[:, None].expand(-1, H), x.abs().amax(-1), "amax")[:nb]
        e = _exponent(amax, code)
        old = _exponent(scale * (127 if code == "int8" else 448), code)
        e = torch.where(((first > 0) & (first < B))[:, None], torch.maximum(e, old), e)
        e = torch.where((first < B)[:, None], e, old)
        earlier = (token[None, :] < first[:, None]) & (first < B)[:, None]
        scaled = _encode(codes.float() * _pow2(old - e)[:, :, None, None], code)
        raw = torch.int8
        codes2 = torch.where(earlier[:, None, :, None], scaled.view(raw), codes.view(raw))
        codes2 = torch.cat([codes2, codes2.new_zeros(1, H, B, D)])
        inv = torch.cat([_pow2(-e), torch.ones(1, H, device=x.device)])
        codes2[block, :, off] = _encode(x * inv[block][..., None], code).view(raw)
        return codes2[:nb].view(codes.dtype), _pow2(e)

    (kc, ks), (vc, vs) = put(s["k"], s["kc"], s["ks"]), put(s["v"], s["vc"], s["vs"])
    return {"kc": kc, "vc": vc, "ks": ks, "vs": vs}


def _attend(s):
    B, H, D, G = s["block"], s["kv_heads"], s["head_dim"], s["heads"] // s["kv_heads"]
    table, cu, lens, q = s["table"], s["cu_rows"].long(), s["lens"].long(), s["q"]
    n, R, L = table.shape[0], s["max_rows"], s["max_len"]
    dev, total = q.device, q.shape[0]
    blocks = table[:, :_ceil(L, B)].clamp(min=0).long()

    def cached(codes, scale):  # [request][head][key][dim] in 32 bits
        x = codes.view(torch.int8)[blocks].view(codes.dtype).float() * scale[blocks][..., None, None]
        return x.transpose(1, 2).reshape(n, H, -1, D)[:, :, :L]

    rows = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + torch.arange(R, device=dev)[None, :]).clamp(max=total - 1)  # padded rows [request][row]
    x = q[at].float().reshape(n, R, H, G, D).permute(0, 2, 3, 1, 4).reshape(n, H, G * R, D)
    k, v = cached(s["kc"], s["ks"]), cached(s["vc"], s["vs"])
    score = (x @ k.transpose(-1, -2)).mul_(s["scale"]).reshape(n, H, G, R, L)
    pos = (lens - rows)[:, None] + torch.arange(R, device=dev)[None, :]
    key = torch.arange(L, device=dev)[None, None, :]
    seen = (key <= pos[..., None]) & (key < lens[:, None, None])
    if s["window"]:
        seen &= key > pos[..., None] - s["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(top > -math.inf, top, 0.0)).exp_()
    del score
    sum_ = p.sum(-1, keepdim=True)
    # key rows behind a request's end hold anything: a weight of zero would not remove an infinity or a NaN
    v = torch.where((key[0] < lens[:, None])[:, None, :, None], v, 0.0)
    o = (p.reshape(n, H, G * R, L) @ v).reshape(n, H, G, R, D) / torch.where(sum_ > 0, sum_, 1.0)
    lse = (top + sum_.log()).squeeze(-1)
    seq = torch.searchsorted(cu[1:].contiguous(), torch.arange(total, device=dev), right=True).clamp(max=n - 1)
    row = torch.arange(total, device=dev) - cu[seq]
    pick = lambda y: y.permute(0, 3, 1, 2, *range(4, y.dim()))[seq, row].flatten(1, 2)  # noqa: E731
    return {"out": pick(o).to(q.dtype), "lse": pick(lse)}


# ------------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "plan":
        return None
    if op == "rope":
        w = s["freqs"].double()
        out = {}
        for name in ("q", "k"):
            x = s[name].double()
            z = x[..., :case["rot"]]
            z = torch.complex(*((z[..., :w.numel()], z[..., w.numel():]) if case["layout"] == "half" else (z[..., ::2], z[..., 1::2])))
            phase = s["positions"].double()[:, None, None] * w
            z = z * torch.polar(torch.full_like(phase, s["mscale"]), -phase if case["back"] else phase)
            x = x.clone()
            if case["layout"] == "half":
                x[..., :w.numel()], x[..., w.numel():case["rot"]] = z.real, z.imag
            else:
                x[..., :case["rot"]:2], x[..., 1:case["rot"]:2] = z.real, z.imag
            out[name] = x
        return out
    if op == "append":
        return _exact_append(case, s)
    if _case_cost(case) > 3e12:
        return None
    return _exact_attend(case, s)


def _case_cost(case):
    rows, lens = _row_lengths(case)
    return 4.0 * sum(n * a for n, a in zip(rows, lens)) * case["heads"] * case["head_dim"]


def _exact_append(case, s):
    """Scales and codes from the definition, the codes as 64-bit values before their scale."""
    B, whole = case["block"], case["code"] == "int8"
    top = 127.0 if whole else 448.0
    held = {}
    for r, at in enumerate(s["slots"].tolist()):
        if at >= 0:
            held.setdefault(at // B, []).append((at % B, r))
    ids = torch.tensor(list(held), device=s["slots"].device)
    first = torch.tensor([min(o for o, _ in v) for v in held.values()], device=ids.device)
    block = torch.tensor([i for i, v in enumerate(held.values()) for _ in v], device=ids.device)
    off = torch.tensor([o for v in held.values() for o, _ in v], device=ids.device)
    row = torch.tensor([r for v in held.values() for _, r in v], device=ids.device)

    def nearest(x):
        if whole:
            return torch.round(x)
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(x / step) * step

    result = {}
    for name in ("k", "v"):
        x, codes = s[name].double()[row], s[name + "c"].view(torch.int8).clone()
        before = s[name + "s"].double()[ids]
        new = torch.stack([s[name].double()[[r for _, r in v]].abs().amax((0, 2)) for v in held.values()])
        need = torch.where((first > 0)[:, None], torch.maximum(new / top, before), new / top).clamp(min=2.0 ** MIN_EXP)
        e = torch.floor(torch.log2(need))
        e = e + (torch.exp2(e) < need)
        scale = torch.exp2(e - (torch.exp2(e - 1) >= need).to(e))
        old = codes[ids].view(s[name + "c"].dtype).double()
        earlier = torch.arange(B, device=ids.device)[None, :] < first[:, None]
        old = torch.where(earlier[:, None, :, None], nearest(old * (before / scale)[..., None, None]), old)
        old[block, :, off] = nearest(x / scale[block][..., None])
        values = codes.view(s[name + "c"].dtype).double()
        values[ids] = old
        scales = s[name + "s"].double().clone()
        scales[ids] = scale
        result[name + "c"], result[name + "s"] = values, scales
    return result


def _exact_attend(case, s):
    B, H, D, G = case["block"], case["kv_heads"], case["head_dim"], case["heads"] // case["kv_heads"]
    rows, lens = _row_lengths(case)
    total = sum(rows)
    dev = s["q"].device
    out = torch.zeros(total, H * G, D, dtype=torch.float64, device=dev)
    lse = torch.full((total, H * G), -math.inf, dtype=torch.float64, device=dev)
    r0 = 0
    for i, (n, a) in enumerate(zip(rows, lens)):
        if not n or not a:
            r0 += n
            continue
        ids = s["table"][i, :_ceil(a, B)].long()
        pos = torch.arange(a - n, a, device=dev)
        key = torch.arange(a, device=dev)
        hide = key[None, :] > pos[:, None]
        if case["window"]:
            hide |= key[None, :] <= pos[:, None] - case["window"]
        for h in range(H):
            k, v = ((s[c].view(torch.int8)[ids, h].view(s[c].dtype).double() * s[t][ids, h].double()[:, None, None]).reshape(-1, D)[:a]
                    for c, t in (("kc", "ks"), ("vc", "vs")))
            for j in range(G):
                z = s["q"][r0:r0 + n, h * G + j].double() @ k.T * s["scale"]
                z = z.masked_fill(hide, -math.inf)
                lse[r0:r0 + n, h * G + j] = torch.logsumexp(z, -1)
                out[r0:r0 + n, h * G + j] = torch.softmax(z, -1) @ v
        r0 += n
    return {"out": out, "lse": lse}
