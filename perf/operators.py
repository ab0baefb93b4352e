"""Performance cases of the serving and rotary operators: page tables, rotary positions, the 4-bit key/value cache.

A case names an operation and its sizes.  `prepare` makes what a program holds before the call, `run` is one pass, in a plain
form of elementary torch operations or through the package's public functions (`own`), `exact` the same from the definition
in 64 bits, `work` counts what a pass cannot do without.  Operations:

  extend    pages for new tokens of a batch of requests: block table, slots, positions (`cache_extend`)
  release   the pages of finished requests back on the free list (`cache_release`)
  rotary    rotary positions with one or several axes, on query and key heads, forward or backward
  store     new keys and values into a paged 4-bit cache, and all of it read back as bf16 (`cache_append_q4`, `cache_read_q4`:
            a chunk of a prompt, whose attention follows over what the cache now holds)
  decode    one query per sequence against a paged 4-bit cache (`attention_decode_q4`)

The 4-bit cache: groups of 32 channels of a token and head share a scale; channel values are n - 8 times it, n in 0 .. 15.
A page holds, for each key/value head, [page][D/2] bytes (channel 2j in the low half of byte j) and then [page][D/32] scale codes.
A code c stands for the 16-bit float with the bits c << 7, divided by 8; the largest written is 222, and 255 stands for NaN.
The scale of a group is the smallest with 7.5 * scale >= max |x|, and n - 8 is x / scale rounded to the nearest, ties to even.
"""
import importlib
import itertools
import math
import random

import torch

own = False

BF16, F32 = "bf16", "f32"
_DTYPE = {BF16: torch.bfloat16, F32: torch.float32}
_TOP_CODE = 222


def _package():
    return importlib.import_module("pku-aiprogramming_b200")


def listed():
    return [
        # one decode step of a full batch: a token for each request, a page now and then
        dict(name="extend_step", op="extend", B=64, page=64, max_pages=128, shortest=17, longest=8000, least=1, most=1, room=1.0, lens=3),
        # prompts admitted together, in pages of 16 rows, the pool too small for the last of them
        dict(name="extend_prompts", op="extend", B=256, page=16, max_pages=512, shortest=0, longest=4096, least=1, most=2048, room=0.9, lens=5),
        # a large batch of which half has finished
        dict(name="release", op="release", B=512, page=16, max_pages=512, shortest=1, longest=8192, done=0.5, lens=7),
        # queries and keys of one decode step, grouped heads, positions far into a long context
        dict(name="rotary_step", op="rotary", dtype=BF16, layout="packed", B=1, S=64, H=32, Hkv=8, D=128, R=128, axes=1, pairing="halves",
             far=1000000, back=False),
        # a packed batch of text, images and video: time, height and width, q and k as slices of one projection
        dict(name="rotary_media", op="rotary", dtype=BF16, layout="fused", B=1, S=16384, H=32, Hkv=8, D=128, R=128, axes=3, pairing="halves",
             far=32768, back=False),
        # training in the reference's own element type: gradients of an image model's heads, rows and columns, half of the channels
        dict(name="rotary_grad", op="rotary", dtype=F32, layout="dense", B=2, S=2048, H=8, Hkv=8, D=64, R=32, axes=2, pairing="neighbours",
             far=4096, back=True),
        # one token for each of many young sequences
        dict(name="store_step", op="store", dtype=BF16, B=64, Hkv=8, D=128, page=64, shortest=1, longest=48, least=1, most=1, lens=9),
        # chunks of prompts behind what the cache holds
        dict(name="store_chunk", op="store", dtype=BF16, B=8, Hkv=8, D=128, page=64, shortest=0, longest=8192, least=1024, most=4096, lens=11),
        # serving: one sequence, grouped heads, a length between two powers of two; bound by latency
        dict(name="decode_single", op="decode", B=1, H=32, Hkv=8, D=128, page=64, shortest=5001, longest=5001, lens=13),
        # serving: a full batch of long sequences, each at a length of its own; bound by the cache's bytes
        dict(name="decode_batch", op="decode", B=64, H=32, Hkv=8, D=128, page=64, shortest=4096, longest=8192, lens=15),
        # one query head per key/value head, head dim 64, small pages, some sequences just begun or empty
        dict(name="decode_d64", op="decode", B=48, H=16, Hkv=16, D=64, page=16, shortest=0, longest=4096, lens=17),
        # two very long sequences, sixteen query heads per key/value head
        dict(name="decode_long", op="decode", B=2, H=32, Hkv=2, D=128, page=128, shortest=120001, longest=131072, lens=19),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["extend", "release", "rotary", "rotary", "store", "store", "decode", "decode", "decode"])
    page = rng.choice([16, 32, 48, 64, 128])
    D = rng.choice([64, 128])
    seed = rng.randrange(1, 1 << 16)
    if op in ("extend", "release"):
        B = _log_int(rng, 1, 512)
        longest = _log_int(rng, 16, 8192)
        most = 1 if rng.random() < 0.5 else min(2048, _log_int(rng, 1, max(2, 400000 // B)))
        c = dict(op=op, B=B, page=page, max_pages=(longest + most + page - 1) // page + rng.randrange(4), shortest=rng.choice([0, 1, longest // 2]),
                 longest=longest, lens=seed)
        c.update(dict(done=rng.choice([0.05, 0.5, 1.0])) if op == "release" else dict(least=rng.choice([0, 1]) if B > 8 else 1, most=most, room=rng.choice([0.5, 1.0, 1.0])))
        return c
    if op == "rotary":
        layout = rng.choice(["packed", "fused", "dense"])
        D = rng.choice([64, 80, 96, 128, 256])
        R = rng.choice([D, D, D // 2, D // 4])
        Hkv = rng.choice([1, 2, 4, 8])
        H = min(32, Hkv * rng.choice([1, 2, 4, 8]))
        B = rng.randrange(1, 5) if layout == "dense" else 1
        S = _log_int(rng, 1, 16384)
        while B * S * (H + Hkv) * D > 40e6:
            S = max(1, S // 2)
        return dict(op=op, dtype=rng.choice([BF16, BF16, F32]), layout=layout, B=B, S=S, H=H, Hkv=Hkv, D=D, R=R, axes=rng.choice([1, 1, 2, 3]),
                    pairing=rng.choice(["halves", "neighbours"]), far=_log_int(rng, 64, 1000000), back=rng.random() < 0.5)
    if op == "store":
        B, Hkv = _log_int(rng, 1, 64), rng.choice([1, 2, 4, 8, 16])
        most = 1 if rng.random() < 0.4 else _log_int(rng, 1, 4096)
        longest = _log_int(rng, 1, 8192)
        while B > 1 and B * Hkv * D * (longest + most) > 50e6:
            B //= 2
        return dict(op=op, dtype=rng.choice([BF16, BF16, F32]), B=B, Hkv=Hkv, D=D, page=page, shortest=rng.choice([0, longest // 2]), longest=longest,
                    least=rng.choice([0, 1]) if B > 8 else 1, most=most, lens=seed)
    Hkv = rng.choice([1, 2, 4, 8, 16])
    H = Hkv * rng.choice([1, 2, 4, 5, 8, 16])
    B, longest = _log_int(rng, 1, 64), _log_int(rng, 1, 65536)
    while B > 1 and B * Hkv * D * longest > 250e6:
        B //= 2
    while longest > 1 and B * H * longest > 12e6:
        longest //= 2
    return dict(op=op, B=B, H=H, Hkv=Hkv, D=D, page=page, shortest=rng.choice([0 if B > 4 else 1, (longest + 1) // 2, longest]), longest=longest, lens=seed)


# ---- the sizes of a case: part of the case, not of its data

def _lengths(c):
    """(tokens a request holds, tokens it gets) of each request."""
    rng = random.Random(c["lens"])
    old = [rng.randint(c["shortest"], c["longest"]) for _ in range(c["B"])]
    new = [rng.randint(c.get("least", 0), c.get("most", 0)) for _ in range(c["B"])]
    return old, new


def _cols(n, page):
    return (n + page - 1) // page


def _done(c):
    rng = random.Random(c["lens"] + 1)
    return [rng.random() < c["done"] for _ in range(c["B"])]


def _served(c):
    """(tokens, pages) that an `extend` case hands out, and the pages on its free list."""
    old, new = _lengths(c)
    need = [_cols(o + n, c["page"]) - _cols(o, c["page"]) for o, n in zip(old, new)]
    free = max(1, int(sum(need) * c["room"]))
    n = sum(pages <= free for pages in itertools.accumulate(need))
    return sum(new[:n]), sum(need[:n]), free


# ---- the cache's number format

def _scales(codes):
    """What scale codes stand for, in 32 bits."""
    return (codes.to(torch.int16) << 7).view(torch.float16).float() / 8


def _quantised(x):
    """x [..., D] -> (bytes [..., D/2], codes [..., D/32])."""
    g = x.unflatten(-1, (-1, 32)).double()
    top = g.abs().amax(-1)
    every = _scales(torch.arange(_TOP_CODE + 1, device=x.device, dtype=torch.uint8)).double()
    code = torch.searchsorted(every * 7.5, top.contiguous()).clamp_max(_TOP_CODE)
    scale = every[code].unsqueeze(-1)
    n = torch.where(scale > 0, (g / scale).round(), 0.0).clamp(-8, 7) + 8
    bad = torch.isnan(top)
    n = torch.where(bad.unsqueeze(-1), 8.0, n).to(torch.uint8).flatten(-2)
    return n[..., 0::2] | (n[..., 1::2] << 4), torch.where(bad, 255, code).to(torch.uint8)


def _halves(cache, page, D):
    """The bytes [pages, Hkv, page, D/2] and codes [pages, Hkv, page, D/32] of a cache, as views."""
    at = page * D // 2
    return cache[..., :at].unflatten(-1, (page, D // 2)), cache[..., at:].unflatten(-1, (page, D // 32))


def _write(cache, page, D, slots, x):
    """Rows x [T, Hkv, D] into the cache at `slots` [T]."""
    data, codes = _quantised(x)
    into, scales = _halves(cache, page, D)
    into[slots // page, :, slots % page] = data
    scales[slots // page, :, slots % page] = codes


def _read(cache, page, D, slots):
    """The values in 32 bits, [*slots.shape, Hkv, D], of the rows at `slots`."""
    data, codes = _halves(cache, page, D)
    data, codes = data[slots // page, :, slots % page], codes[slots // page, :, slots % page]
    n = torch.stack((data & 15, data >> 4), -1).flatten(-2).float() - 8
    return (n.unflatten(-1, (-1, 32)) * _scales(codes).unsqueeze(-1)).flatten(-2)


# ---- prepare

def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _table(c, lens, g, more=0):
    """A block table over pages in the order in which a pool hands them out, entries behind a row's pages 0, and the pool's size."""
    per = [_cols(n, c["page"]) for n in lens]
    width = c.get("max_pages") or max(1, max(per))
    order = torch.randperm(sum(per) + more, generator=g, device="cuda").to(torch.int32)
    col = torch.arange(width, device="cuda").expand(len(per), width)
    n = torch.tensor(per, device="cuda").unsqueeze(1)
    table = torch.zeros((len(per), width), dtype=torch.int32, device="cuda")
    table[col < n] = order[:sum(per)]
    return table, order[sum(per):].contiguous(), sum(per) + more


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op = c["op"]
    dt = _DTYPE[c.get("dtype", BF16)]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=dt)

    s = {"case": c}
    if op in ("extend", "release"):
        old, new = _lengths(c)
        if op == "extend":
            free = _served(c)[2]
            s["table"], s["free"], _ = _table(c, old, g, free + 61)   # (the list is longer than what is on it)
            s.update(lens=_ints(old), new=_ints(new), n_free=_ints([free]), tokens=max(1, sum(new)))
        else:
            s["table"], s["free"], total = _table(c, old, g, 64)
            s["free"] = torch.cat((s["free"], torch.zeros(total, dtype=torch.int32, device="cuda")))
            s.update(lens=_ints(old), n_free=_ints([64]), done=torch.tensor(_done(c), device="cuda"))
        return s
    if op == "rotary":
        B, S, H, Hkv, D, R, A = (c[k] for k in ("B", "S", "H", "Hkv", "D", "R", "axes"))
        if c["layout"] == "dense":
            s.update(q=normal(B, H, S, D), k=normal(B, Hkv, S, D))
            where = (B, S)
        else:
            if c["layout"] == "fused":   # the keys and queries of one projection's rows, the values behind them
                rows = normal(S, H + 2 * Hkv, D)
                s.update(q=rows[:, :H], k=rows[:, H:H + Hkv])
            else:
                s.update(q=normal(S, H, D), k=normal(S, Hkv, D))
            where = (S,)
        s["positions"] = torch.randint(0, c["far"], (A,) + where, generator=g, device="cuda", dtype=torch.int32)
        i = torch.arange(R // 2, device="cuda")
        s["inv_freq"] = 10000.0 ** (-i.double() / (R // 2))
        s["axes"] = (i * A // (R // 2)).to(torch.int32) if A > 1 else None
        return s
    D, Hkv, page = c["D"], c["Hkv"], c["page"]
    old, new = _lengths(c)
    lens = [a + b for a, b in zip(old, new)]
    table, _, pages = _table(c, lens, g)
    shape = (max(1, pages), Hkv, page * D * 17 // 32)
    s.update(table=table, k_cache=torch.zeros(shape, dtype=torch.uint8, device="cuda"), v_cache=torch.zeros(shape, dtype=torch.uint8, device="cuda"))
    for b in range(c["B"]):   # what the cache holds of each sequence
        at = torch.arange(old[b], device="cuda")
        slots = table[b, at // page].long() * page + at % page
        for name in ("k_cache", "v_cache"):
            _write(s[name], page, D, slots, normal(old[b], Hkv, D))
    if op == "store":
        tokens = sum(new)
        at = torch.cat([torch.arange(a, n, device="cuda") for a, n in zip(old, lens)])
        row = torch.cat([torch.full((n,), b, device="cuda") for b, n in enumerate(new)])
        s.update(k=normal(tokens, Hkv, D), v=normal(tokens, Hkv, D), slots=(table[row, at // page] * page + at % page).to(torch.int32),
                 cu=_ints([sum(lens[:i]) for i in range(len(lens) + 1)]), total=sum(lens))
        return s
    s.update(q=normal(c["B"], c["H"], 1, D), lens=_ints(lens), longest=max(1, max(lens)))
    return s


# ---- the plain forms

def _extend(s):
    page, tokens, table = s["case"]["page"], s["tokens"], s["table"]
    B, width = table.shape
    old, new, free = s["lens"].long(), s["new"].long(), s["free"].long()
    n_free = s["n_free"].long().clamp(0, free.numel())
    fits = (old >= 0) & (new >= 0) & (old + new <= width * page)
    n = torch.where(fits, new, 0)
    have = (old + page - 1) // page
    need = torch.where(fits, (old + n + page - 1) // page - have, 0)
    ok = fits & (n.cumsum(0) <= tokens) & (need.cumsum(0) <= n_free)
    n, need = torch.where(ok, n, 0), torch.where(ok, need, 0)
    cu = torch.cat((n.new_zeros(1), n.cumsum(0)))
    before = need.cumsum(0) - need
    j = torch.arange(width, device=table.device) - have.unsqueeze(1)
    taken = (n_free - 1 - before.unsqueeze(1) - j).clamp(0, free.numel() - 1)
    table.copy_(torch.where((j >= 0) & (j < need.unsqueeze(1)), free[taken], table.long()))
    t = torch.arange(tokens, device=table.device)
    b = torch.searchsorted(cu[1:], t, right=True).clamp_max(B - 1)
    pos = old[b] + t - cu[b]
    at = table[b, (pos // page).clamp(0, width - 1)].long()
    there = t < cu[B]
    slots = torch.where(there & (at >= 0), at * page + pos % page, -1)
    return {"table": table, "lens": (old + n).int(), "n_free": (n_free - need.sum()).int(), "cu": cu.int(), "slots": slots.int(),
            "positions": torch.where(there, pos, 0).int()}


def _release(s):
    page, table, free = s["case"]["page"], s["table"], s["free"]
    width = table.shape[1]
    lens = s["lens"].long()
    n_free = s["n_free"].long().clamp(0, free.numel())
    count = torch.where(s["done"], (lens + page - 1) // page, 0)
    j = torch.arange(width, device=table.device)
    to = n_free + (count.cumsum(0) - count).unsqueeze(1) + j
    here = (j < count.unsqueeze(1)) & (to < free.numel())
    spare = torch.cat((free, free.new_zeros(1)))
    spare[torch.where(here, to, free.numel())] = table
    free.copy_(spare[:-1])
    return {"free": free, "lens": torch.where(s["done"], 0, lens).int(), "n_free": (n_free + count.sum()).clamp_max(free.numel()).int()}


def _rotated(x, cos, sin, R, halves, back):
    """x [..., D] by the angles' cosines and sines [..., R/2], in 32 bits, rounded once."""
    y = x.float()
    if halves:
        a, b = y[..., :R // 2], y[..., R // 2:R]
    else:
        a, b = y[..., 0:R:2], y[..., 1:R:2]
    sin = -sin if back else sin
    first, second = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat((first, second), -1) if halves else torch.stack((first, second), -1).flatten(-2)
    return torch.cat((turned, y[..., R:]), -1).to(x.dtype)


def _rotary(s):
    c = s["case"]
    pos = s["positions"].double()
    per_pair = pos[s["axes"].long()] if s["axes"] is not None else pos.expand((c["R"] // 2,) + pos.shape[1:])
    angle = per_pair.movedim(0, -1) * s["inv_freq"]   # far positions: 64 bits
    angle = angle.unsqueeze(1 if c["layout"] == "dense" else -2)
    cos, sin = angle.cos().float(), angle.sin().float()
    halves = c["pairing"] == "halves"
    return _rotated(s["q"], cos, sin, c["R"], halves, c["back"]), _rotated(s["k"], cos, sin, c["R"], halves, c["back"])


def _store(s):
    c = s["case"]
    page, D, table, cu = c["page"], c["D"], s["table"], s["cu"].long()
    slots = s["slots"].long()
    _write(s["k_cache"], page, D, slots, s["k"])
    _write(s["v_cache"], page, D, slots, s["v"])
    t = torch.arange(s["total"], device=cu.device)
    b = torch.searchsorted(cu[1:], t, right=True)
    at = t - cu[b]
    rows = table[b, at // page].long() * page + at % page
    return _read(s["k_cache"], page, D, rows).bfloat16(), _read(s["v_cache"], page, D, rows).bfloat16()


def _decode(s):
    c = s["case"]
    page, D, Hkv, table = c["page"], c["D"], c["Hkv"], s["table"]
    at = torch.arange(s["longest"], device=table.device)
    rows = table[:, at // page].long() * page + at % page
    there = at < s["lens"].unsqueeze(1)
    q = s["q"].float().view(c["B"], Hkv, -1, D)
    k = _read(s["k_cache"], page, D, rows)
    scores = torch.einsum("bhgd,blhd->bhgl", q, k) * D ** -0.5
    scores = scores.masked_fill(~there[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = (scores - top).exp()
    total = p.sum(-1, keepdim=True)
    v = _read(s["v_cache"], page, D, rows).masked_fill(~there[..., None, None], 0.0)
    out = torch.einsum("bhgl,blhd->bhgd", p, v) / torch.where(total == 0, 1.0, total)
    return out.reshape(s["q"].shape).to(s["q"].dtype), (top + total.log()).reshape(c["B"], c["H"], 1)


def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"extend": _extend, "release": _release, "rotary": _rotary, "store": _store, "decode": _decode}[op](s)
    tt = _package()
    if op == "extend":
        step = tt.cache_extend(s["table"], s["lens"], s["new"], s["free"], s["n_free"], c["page"], s["tokens"])
        return {"table": s["table"], "lens": step.seq_lens, "n_free": step.n_free, "cu": step.cu_new, "slots": step.slots, "positions": step.positions}
    if op == "release":
        lens, n_free = tt.cache_release(s["table"], s["lens"], s["done"], s["free"], s["n_free"], c["page"])
        return {"free": s["free"], "lens": lens, "n_free": n_free}
    if op == "rotary":
        call = tt.rotary_backward if c["back"] else tt.rotary_forward
        return call(s["q"], s["k"], s["positions"], s["inv_freq"], axes=s["axes"], interleaved=c["pairing"] == "neighbours")
    if op == "store":
        tt.cache_append_q4(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"])
        return tt.cache_read_q4(s["k_cache"], s["v_cache"], s["table"], s["cu"], s["total"], c["page"])
    return tt.attention_decode_q4(s["q"], s["k_cache"], s["v_cache"], block_table=s["table"], seq_lens=s["lens"], max_len=s["longest"])


# ---- 64 bits

def _value(byte_rows, code_rows):
    """Values of cache rows in 64 bits: byte_rows [..., D/2], code_rows [..., D/32]."""
    low, high = byte_rows % 16, byte_rows // 16
    n = torch.empty(byte_rows.shape[:-1] + (2 * byte_rows.shape[-1],), dtype=torch.float64, device=byte_rows.device)
    n[..., 0::2], n[..., 1::2] = low.double(), high.double()
    e, m = (code_rows // 8).double(), (code_rows % 8).double()
    # exponent 0 has no leading one; the 8 of the mantissa's steps and the division by 8 are in the power of two
    scale = torch.where(e > 0, (8 + m) * torch.exp2(e - 21), m * 2.0 ** -20)
    return (n - 8) * scale.repeat_interleave(32, -1)


def _nearest(x):
    """What 4 bits keep of x [..., D], in 64 bits: step by step up the scales, by the definition."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1)
    e = torch.floor(torch.log2(top / 7.5 + 1e-300)).clamp(-17, 9)   # (8 + m) 2^(e - 3), m of 0 .. 7, from the binade below on
    scale = torch.full_like(top, 896.0)
    for up in (2, 1, 0, -1):
        for m in range(7, -1, -1):
            s = (8 + m) * torch.exp2(e + up - 3)
            s = torch.where(e + up < -17, m * 2.0 ** -20, s)
            scale = torch.where((7.5 * s >= top) & (s < scale), s, scale)
    scale = torch.where(top == 0, 0.0, scale).unsqueeze(-1)
    n = torch.where(scale > 0, g / scale, 0.0)
    low = n.floor()
    n = torch.where((n - low > 0.5) | ((n - low == 0.5) & (low % 2 != 0)), low + 1, low).clamp(-8, 7)
    return (n * scale).flatten(-2)


def exact(c, seed):
    op = c["op"]
    if op in ("extend", "release"):
        return None
    s = prepare(c, seed)
    if op == "rotary":
        half, sign = c["R"] // 2, -1.0 if c["back"] else 1.0
        which = s["axes"].tolist() if s["axes"] is not None else [0] * half
        got = []
        for x in (s["q"], s["k"]):
            y = x.double().clone()
            for i in range(half):
                a = s["positions"][which[i]].double() * s["inv_freq"][i]
                a = a[:, None] if c["layout"] == "dense" else a[:, None].expand(-1, x.shape[1])
                at, to = (i, i + half) if c["pairing"] == "halves" else (2 * i, 2 * i + 1)
                u, w = x[..., at].double(), x[..., to].double()
                y[..., at] = u * a.cos() - sign * w * a.sin()
                y[..., to] = w * a.cos() + sign * u * a.sin()
            got.append(y)
        return tuple(got)
    page, D, Hkv, table = c["page"], c["D"], c["Hkv"], s["table"].tolist()

    def sequence(cache, b, n):
        """Keys 0 .. n of sequence b, [n, Hkv, D], page by page."""
        pages = cache[torch.tensor(table[b][:_cols(n, page)], dtype=torch.long, device="cuda")]
        data = pages[:, :, :page * D // 2].reshape(-1, Hkv, page, D // 2).transpose(1, 2).reshape(-1, Hkv, D // 2)
        code = pages[:, :, page * D // 2:].reshape(-1, Hkv, page, D // 32).transpose(1, 2).reshape(-1, Hkv, D // 32)
        return _value(data[:n], code[:n])

    old, new = _lengths(c)
    if op == "store":
        got, first = ([], []), [sum(new[:b]) for b in range(c["B"])]
        for b in range(c["B"]):
            for into, cache, x in zip(got, (s["k_cache"], s["v_cache"]), (s["k"], s["v"])):
                into += [sequence(cache, b, old[b]), _nearest(x[first[b]:first[b] + new[b]])]
        return tuple(torch.cat(x) for x in got)
    out, lse = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), torch.full((c["B"], c["H"], 1), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(c["B"]):
        if old[b]:
            k, v = sequence(s["k_cache"], b, old[b]), sequence(s["v_cache"], b, old[b])
            q = s["q"][b, :, 0].double().reshape(Hkv, -1, D)
            scores = torch.matmul(q, k.permute(1, 2, 0)) / math.sqrt(D)
            lse[b, :, 0] = torch.logsumexp(scores, -1).reshape(-1)
            out[b, :, 0] = torch.matmul(torch.softmax(scores, -1), v.transpose(0, 1)).reshape(-1, D)
    return out, lse


def work(c):
    """Bytes: every input read once, every output written once.  Operations: two per multiply-add of the attention's products,
    six per rotated pair, and a few per value where there is no product."""
    op = c["op"]
    size = 4 if c.get("dtype", BF16) == F32 else 2
    if op == "extend":
        tokens, pages, _ = _served(c)
        # lengths in and out, cumulative counts, a page's entry read and written, a slot and a position per token
        return {"bytes": 16 * c["B"] + 8 * pages + 8 * max(1, sum(_lengths(c)[1])), "flops": 4.0 * (c["B"] + tokens)}
    if op == "release":
        pages = sum(_cols(n, c["page"]) for n, d in zip(_lengths(c)[0], _done(c)) if d)
        return {"bytes": 9 * c["B"] + 8 * pages, "flops": 2.0 * (c["B"] + pages)}
    if op == "rotary":
        rows = c["B"] * c["S"]
        return {"bytes": rows * (2 * (c["H"] + c["Hkv"]) * c["D"] * size + 4 * c["axes"]), "flops": 3.0 * rows * (c["H"] + c["Hkv"]) * c["R"]}
    D, Hkv = c["D"], c["Hkv"]
    row = D * 17 // 32
    old, new = _lengths(c)
    held, fresh = sum(old), sum(new)
    if op == "store":
        # new rows in and their codes out, the whole cache's codes in (the new ones are at hand) and its values out
        return {"bytes": 2 * Hkv * (fresh * (D * size + row) + held * row + (held + fresh) * 2 * D), "flops": 2.0 * Hkv * D * (4 * fresh + held + fresh)}
    entries = sum(_cols(n, c["page"]) for n in old)
    return {"bytes": 2 * held * Hkv * row + c["B"] * c["H"] * (4 * D + 4) + 4 * entries, "flops": 4.0 * held * c["H"] * D}
