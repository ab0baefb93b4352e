"""Performance cases of the operators between a projection and its attention: norms of heads with rotary positions, appending to a
paged cache with the rotation on the way, and the 8-bit key/value cache with the attention that reads it.

A case names an operation and its sizes.  `prepare` makes what a program holds before the call, `run` is one pass, in a plain
form of elementary torch operations or through the package's public functions (`own`), `exact` the same from the definition
in 64 bits, `work` counts what a pass cannot do without.  Operations:

  norm      query and key heads divided by their root mean square, times a weight per channel, and turned by their positions
            (`norm_rotary_forward`), or the gradients of the heads and of the weights (`norm_rotary_backward`)
  append    a step's queries and keys turned (and normed, where there are weights), the keys and values into the slots of a paged
            16-bit cache (`cache_append_rotary`)
  store     new keys and values into a paged 8-bit cache, and all of it read back as bf16 (`cache_append_q8`, `cache_read_q8`: a chunk of
            a prompt, whose attention follows over what the cache now holds)
  decode    one query per sequence against a paged 8-bit cache (`attention_decode_q8`)

The 8-bit cache: values are 8-bit floats (e4m3) times a power of two that 16 tokens of a head share, those in the rows 16 j .. 16 j + 15
of a page.  A page holds, for each key/value head, [page][D] codes and then [page/16] bytes c, each for 2^(c - 64), up to a
multiple of 32 bytes.  Exponents are -40 .. 40: the smallest with 448 * 2^e >= every finite |x| of the block.  Tokens that come to a
block later raise its exponent where they have to, and what it holds is rounded to the new one; a call that brings a block's row 0
begins it anew.
"""
import importlib
import math
import random

import torch

own = False

BF16, F32 = "bf16", "f32"
_DTYPE = {BF16: torch.bfloat16, F32: torch.float32}
_LOW, _HIGH, _BIAS, _TOP = -40, 40, 64, 448.0


def _package():
    return importlib.import_module("pku-aiprogramming_b200")


def listed():
    return [
        # queries and keys of one decode step, grouped heads; bound by latency
        dict(name="norm_step", op="norm", dtype=BF16, weights=BF16, layout="packed", B=1, S=64, H=32, Hkv=8, D=128, R=128, axes=1, pairing="halves",
             far=1000000, back=False),
        # a packed batch of text, images and video: time, height and width, q and k as slices of one projection
        dict(name="norm_media", op="norm", dtype=BF16, weights=F32, layout="fused", B=1, S=16384, H=32, Hkv=8, D=128, R=128, axes=3, pairing="halves",
             far=32768, back=False),
        # training: gradients of the same heads and of weights kept in 32 bits
        dict(name="norm_grad", op="norm", dtype=BF16, weights=F32, layout="packed", B=1, S=8192, H=32, Hkv=8, D=128, R=128, axes=1, pairing="halves",
             far=8192, back=True),
        # training in the reference's own element type: an image model's heads, rows and columns, half of the channels, an odd length
        dict(name="norm_grad_f32", op="norm", dtype=F32, weights=F32, layout="dense", B=2, S=2047, H=8, Hkv=8, D=64, R=32, axes=2, pairing="neighbours",
             far=4096, back=True),
        # one decode step of a full batch with normed heads: a token for each request, anywhere in its page
        dict(name="append_step", op="append", dtype=BF16, weights=BF16, B=64, H=32, Hkv=8, D=128, R=128, pairing="halves", page=64, shortest=1, longest=1000,
             least=1, most=1, lens=9),
        # prompts of many lengths admitted together, pages of 16 rows, half of the channels turned, no norm
        dict(name="append_prompts", op="append", dtype=BF16, weights="", B=16, H=32, Hkv=8, D=128, R=64, pairing="halves", page=16, shortest=0, longest=512,
             least=1, most=2048, lens=11),
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
    op = rng.choice(["norm", "norm", "norm", "append", "append", "store", "store", "decode", "decode", "decode"])
    page = rng.choice([16, 32, 48, 64, 128])
    seed = rng.randrange(1, 1 << 16)
    dtype = rng.choice([BF16, BF16, F32])
    if op in ("norm", "append"):
        D = rng.choice([64, 80, 96, 128, 256] if op == "norm" else [64, 128, 128])
        R = rng.choice([D, D, D // 2, D // 4])
        Hkv = rng.choice([1, 2, 4, 8])
        H = min(32, Hkv * rng.choice([1, 2, 4, 8]))
        c = dict(op=op, dtype=dtype, weights=rng.choice([dtype, F32] if op == "norm" else [dtype, F32, ""]), H=H, Hkv=Hkv, D=D, R=R,
                 pairing=rng.choice(["halves", "neighbours"]))
        if op == "norm":
            layout = rng.choice(["packed", "fused", "dense"])
            B = rng.randrange(1, 5) if layout == "dense" else 1
            S = _log_int(rng, 1, 16384)
            back = rng.random() < 0.5
            while B * S * (H + Hkv) * D > (40e6 if not back else 27e6):
                S = max(1, S // 2)
            c.update(layout=layout, B=B, S=S, axes=rng.choice([1, 1, 2, 3]), far=_log_int(rng, 64, 1000000), back=back)
            return c
        B, longest = _log_int(rng, 1, 64), _log_int(rng, 1, 2000)
        most = 1 if rng.random() < 0.4 else _log_int(rng, 1, 2048)
        while B > 1 and B * Hkv * D * (longest + most) > 60e6:
            B //= 2
        while most > 1 and B * (H + 2 * Hkv) * D * most > 60e6:
            most //= 2
        c.update(B=B, page=page, shortest=rng.choice([0, longest // 2]), longest=longest, least=rng.choice([0, 1]) if B > 8 else 1, most=most, lens=seed)
        return c
    D = rng.choice([64, 128])
    if op == "store":
        B, Hkv = _log_int(rng, 1, 64), rng.choice([1, 2, 4, 8, 16])
        most = 1 if rng.random() < 0.4 else _log_int(rng, 1, 4096)
        longest = _log_int(rng, 1, 8192)
        while B > 1 and B * Hkv * D * (longest + most) > 50e6:
            B //= 2
        return dict(op=op, dtype=dtype, B=B, Hkv=Hkv, D=D, page=page, shortest=rng.choice([0, longest // 2]), longest=longest,
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
    return old, new if sum(new) or "most" not in c else [1] * c["B"]


def _cols(n, page):
    return (n + page - 1) // page


# ---- the cache's number format

def _power(e):
    """2^e in 32 bits, e whole numbers of -126 .. 127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent(top):
    """The smallest e with 448 * 2^e >= top, within the format's range; top in 32 bits, finite."""
    m, e = torch.frexp(top)   # m of 0.5 .. 1; 448 is 0.875 * 2^9
    return torch.where(top > 0, e - 9 + (m > 0.875), _LOW).clamp(_LOW, _HIGH)


def _codes(x, e):
    """x in 32 bits as bytes, times 2^-e; e broadcastable."""
    return (x * _power(-e)).clamp(-_TOP, _TOP).to(torch.float8_e4m3fn).view(torch.uint8)


def _row_bytes(page, D):
    return page * D + (page // 16 + 31) // 32 * 32


def _halves(cache, page, D):
    """The codes [pages, Hkv, page / 16, 16, D] and exponents' bytes [pages, Hkv, page / 16] of a cache, as views."""
    at = page * D
    return cache[..., :at].unflatten(-1, (page // 16, 16, D)), cache[..., at:at + page // 16]


def _write(cache, page, D, slots, x):
    """Rows x [T, Hkv, D] into the cache at `slots` [T]."""
    into, powers = _halves(cache, page, D)
    x = x.float()
    block, which = torch.unique(slots // 16, return_inverse=True)
    p, j = block // (page // 16), block % (page // 16)
    size = x.abs()
    size = torch.where(size < math.inf, size, 0.0).amax(-1)
    top = size.new_zeros((len(block), size.shape[1])).scatter_reduce_(0, which[:, None].expand_as(size), size, "amax")
    fresh = torch.zeros(len(block), dtype=torch.int32, device=x.device).scatter_reduce_(0, which, (slots % 16 == 0).int(), "amax") > 0
    was = torch.where(fresh[:, None], _LOW, (powers[p, :, j].int() - _BIAS).clamp(_LOW, _HIGH))
    e = torch.maximum(was, _exponent(top))
    held = into[p, :, j]
    moved = _codes(held.view(torch.float8_e4m3fn).float(), (e - was)[..., None, None])
    into[p, :, j] = torch.where(fresh[:, None, None, None], held, moved)
    powers[p, :, j] = (e + _BIAS).to(torch.uint8)
    into[slots // page, :, slots % page // 16, slots % 16] = _codes(x, e[which][..., None])


def _read(cache, page, D, slots):
    """The values in 32 bits, [*slots.shape, Hkv, D], of the rows at `slots`."""
    codes, powers = _halves(cache, page, D)
    p, j = slots // page, slots % page // 16
    return codes[p, :, j, slots % 16].view(torch.float8_e4m3fn).float() * _power(powers[p, :, j].int() - _BIAS).unsqueeze(-1)


# ---- prepare

def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _table(c, lens, g):
    """A block table over pages in the order in which a pool hands them out, entries behind a row's pages 0, and the pool's size."""
    per = [_cols(n, c["page"]) for n in lens]
    width = max(1, max(per))
    order = torch.randperm(sum(per), generator=g, device="cuda").to(torch.int32)
    col = torch.arange(width, device="cuda").expand(len(per), width)
    n = torch.tensor(per, device="cuda").unsqueeze(1)
    table = torch.zeros((len(per), width), dtype=torch.int32, device="cuda")
    table[col < n] = order
    return table, max(1, sum(per))


def _frequencies(s, R, axes):
    i = torch.arange(R // 2, device="cuda")
    s["inv_freq"] = 10000.0 ** (-i.double() / (R // 2))
    s["axes"] = (i * axes // (R // 2)).to(torch.int32) if axes > 1 else None


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, D, Hkv = c["op"], c["D"], c["Hkv"]
    dt = _DTYPE[c.get("dtype", BF16)]

    def normal(*shape, type=dt):
        return torch.randn(shape, generator=g, device="cuda", dtype=type)

    def tokens(n):   # rows of a projection: some tokens are larger than others
        return (normal(n, Hkv, D) * (0.5 * normal(n, 1, 1, type=torch.float32)).exp()).to(dt)

    s = {"case": c, "q_weight": None, "k_weight": None}
    if c.get("weights"):
        s.update({name: (1 + 0.2 * normal(D, type=torch.float32)).to(_DTYPE[c["weights"]]) for name in ("q_weight", "k_weight")})
    if op == "norm":
        B, S, H, A = (c[k] for k in ("B", "S", "H", "axes"))
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
        if c["back"]:
            s.update(dq=normal(*s["q"].shape), dk=normal(*s["k"].shape))
        s["positions"] = torch.randint(0, c["far"], (A,) + where, generator=g, device="cuda", dtype=torch.int32)
        _frequencies(s, c["R"], A)
        return s
    page = c["page"]
    old, new = _lengths(c)
    lens = [a + b for a, b in zip(old, new)]
    table, pages = _table(c, lens, g)
    s["table"] = table
    if op != "decode":
        at = torch.cat([torch.arange(a, n, device="cuda") for a, n in zip(old, lens)])
        row = torch.cat([torch.full((n,), b, device="cuda") for b, n in enumerate(new)])
        s["slots"] = (table[row, at // page] * page + at % page).to(torch.int32)
    if op == "append":
        rows = normal(sum(new), c["H"] + 2 * Hkv, D)   # one projection's rows
        s.update(q=rows[:, :c["H"]], k=rows[:, c["H"]:c["H"] + Hkv], v=rows[:, c["H"] + Hkv:], positions=at.to(torch.int32))
        _frequencies(s, c["R"], 1)
        s.update(k_pool=normal(pages, Hkv, page, D, type=torch.bfloat16), v_pool=normal(pages, Hkv, page, D, type=torch.bfloat16))
        return s
    shape = (pages, Hkv, _row_bytes(page, D))
    s.update(k_cache=torch.zeros(shape, dtype=torch.uint8, device="cuda"), v_cache=torch.zeros(shape, dtype=torch.uint8, device="cuda"))
    for b in range(c["B"]):   # what the cache holds of each sequence
        if old[b]:
            there = torch.arange(old[b], device="cuda")
            slots = table[b, there // page].long() * page + there % page
            for name in ("k_cache", "v_cache"):
                _write(s[name], page, D, slots, tokens(old[b]))
    if op == "store":
        s.update(k=tokens(sum(new)), v=tokens(sum(new)), cu=_ints([sum(lens[:i]) for i in range(len(lens) + 1)]), total=sum(lens))
        return s
    s.update(q=normal(c["B"], c["H"], 1, D), lens=_ints(lens), longest=max(1, max(lens)))
    return s


# ---- the plain forms

_EPS = 1e-6


def _angles(s, dense):
    """Cosines and sines [..., R/2] that broadcast over heads, in 32 bits of 64."""
    half = s["case"]["R"] // 2
    pos = s["positions"].double()
    pos = pos if pos.dim() > 1 else pos[None]
    per_pair = pos[s["axes"].long()] if s["axes"] is not None else pos.expand((half,) + pos.shape[1:])
    angle = (per_pair.movedim(0, -1) * s["inv_freq"]).unsqueeze(1 if dense else -2)   # far positions: 64 bits
    return angle.cos().float(), angle.sin().float()


def _turned(y, cos, sin, R, halves):
    """y [..., D] in 32 bits by the angles' cosines and sines."""
    if halves:
        a, b = y[..., :R // 2], y[..., R // 2:R]
    else:
        a, b = y[..., 0:R:2], y[..., 1:R:2]
    first, second = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat((first, second), -1) if halves else torch.stack((first, second), -1).flatten(-2)
    return torch.cat((turned, y[..., R:]), -1)


def _normed(x, weight):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * weight.float()


def _norm(s):
    c = s["case"]
    dense, halves = c["layout"] == "dense", c["pairing"] == "halves"
    cos, sin = _angles(s, dense)

    def forward(x, weight):
        return _turned(_normed(x, weight), cos, sin, c["R"], halves).to(x.dtype)

    def backward(dz, x, weight):
        g, y = _turned(dz.float(), cos, -sin, c["R"], halves), x.float()
        r = torch.rsqrt((y * y).mean(-1, keepdim=True) + _EPS)
        unit = y * r
        dw = (g * unit).flatten(0, -2).sum(0)
        g = g * weight.float()
        return (r * (g - unit * (g * unit).mean(-1, keepdim=True))).to(x.dtype), dw.to(weight.dtype)

    if not c["back"]:
        return forward(s["q"], s["q_weight"]), forward(s["k"], s["k_weight"])
    (dq, dwq), (dk, dwk) = backward(s["dq"], s["q"], s["q_weight"]), backward(s["dk"], s["k"], s["k_weight"])
    return dq, dk, dwq, dwk


def _append(s):
    c = s["case"]
    cos, sin = _angles(s, False)

    def one(x, weight):
        y = x.float() if weight is None else _normed(x, weight)
        return _turned(y, cos, sin, c["R"], c["pairing"] == "halves").bfloat16()

    p, r = s["slots"].long() // c["page"], s["slots"].long() % c["page"]
    s["k_pool"][p, :, r] = one(s["k"], s["k_weight"])
    s["v_pool"][p, :, r] = s["v"].bfloat16()
    return {"q": one(s["q"], s["q_weight"]), "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


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
        return {"norm": _norm, "append": _append, "store": _store, "decode": _decode}[op](s)
    tt = _package()
    if op == "norm":
        how = dict(axes=s["axes"], interleaved=c["pairing"] == "neighbours", eps=_EPS)
        if not c["back"]:
            return tt.norm_rotary_forward(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["inv_freq"], **how)
        return tt.norm_rotary_backward(s["dq"], s["dk"], s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["inv_freq"], **how)
    if op == "append":
        q = tt.cache_append_rotary(s["q"], s["k"], s["v"], s["slots"], s["positions"], s["inv_freq"], s["k_pool"], s["v_pool"],
                                   interleaved=c["pairing"] == "neighbours", q_weight=s["q_weight"], k_weight=s["k_weight"], eps=_EPS)
        return {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}
    if op == "store":
        tt.cache_append_q8(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"])
        return tt.cache_read_q8(s["k_cache"], s["v_cache"], s["table"], s["cu"], s["total"], c["page"])
    return tt.attention_decode_q8(s["q"], s["k_cache"], s["v_cache"], block_table=s["table"], seq_lens=s["lens"], max_len=s["longest"])


# ---- 64 bits

def _value(codes, powers):
    """Values of cache rows in 64 bits: codes [..., D], powers [...], one for each row."""
    n = codes.long()
    sign, e, m = 1 - 2 * (n // 128), n // 8 % 16, n % 8
    v = sign * torch.where(e > 0, (8 + m) * torch.exp2((e - 10).double()), m * 2.0 ** -9)
    return v * torch.exp2(powers.double() - _BIAS).unsqueeze(-1)


def _nearest(x, e):
    """x in 64 bits to the nearest of the 8-bit floats times 2^e, ties to the even one."""
    y = x.abs() * torch.exp2(-e)
    step = torch.exp2((torch.floor(torch.log2(y.clamp_min(2.0 ** -30))) - 3).clamp(-9, 5))
    n = y / step
    low = n.floor()
    n = torch.where((n - low > 0.5) | ((n - low == 0.5) & (low % 2 != 0)), low + 1, low)
    return torch.sign(x) * (n * step).clamp_max(_TOP) * torch.exp2(e)


def _unit(x):
    """x in 64 bits over its root mean square."""
    return x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + _EPS)


def exact(c, seed):
    op = c["op"]
    s = prepare(c, seed)
    D, Hkv = c["D"], c["Hkv"]
    if op in ("norm", "append"):
        half, dense = c["R"] // 2, c.get("layout") == "dense"
        which = s["axes"].tolist() if s["axes"] is not None else [0] * half
        pos = s["positions"] if s["positions"].dim() > 1 else s["positions"][None]

        def rotated(x, sign):
            y = x.clone()
            for i in range(half):
                a = pos[which[i]].double() * s["inv_freq"][i]
                a = a[:, None] if dense else a[:, None].expand(-1, x.shape[1])
                at, to = (i, i + half) if c["pairing"] == "halves" else (2 * i, 2 * i + 1)
                y[..., at] = x[..., at] * a.cos() - sign * x[..., to] * a.sin()
                y[..., to] = x[..., to] * a.cos() + sign * x[..., at] * a.sin()
            return y

        def forward(x, w):
            return rotated(x.double() if w is None else _unit(x.double()) * w.double(), 1.0)

        if op == "append":
            k_pool, v_pool, k, v = s["k_pool"].double(), s["v_pool"].double(), forward(s["k"], s["k_weight"]), s["v"].double()
            slots = s["slots"].long()
            for h in range(Hkv):
                k_pool[slots // c["page"], h, slots % c["page"]] = k[:, h]
                v_pool[slots // c["page"], h, slots % c["page"]] = v[:, h]
            return {"q": forward(s["q"], s["q_weight"]), "k_pool": k_pool, "v_pool": v_pool}
        if not c["back"]:
            return forward(s["q"], s["q_weight"]), forward(s["k"], s["k_weight"])
        found = []
        for dz, x, w in ((s["dq"], s["q"], s["q_weight"]), (s["dk"], s["k"], s["k_weight"])):
            y, g = x.double(), rotated(dz.double(), -1.0)
            mean = y.square().sum(-1, keepdim=True) / D + _EPS
            dw = (g * _unit(y)).reshape(-1, D).sum(0)
            g = g * w.double()
            found.append((g / mean.sqrt() - y * (g * y).sum(-1, keepdim=True) / (D * mean * mean.sqrt()), dw))
        return found[0][0], found[1][0], found[0][1], found[1][1]
    page, table = c["page"], s["table"].tolist()

    def sequence(cache, b, n):
        """Codes [Hkv, blocks, 16, D] and exponents' bytes [Hkv, blocks] of the blocks that hold sequence b's n tokens, page by page."""
        pages = cache[torch.tensor(table[b][:_cols(n, page)], dtype=torch.long, device="cuda")].transpose(0, 1)
        blocks = _cols(n, 16)
        codes = pages[..., :page * D].reshape(Hkv, -1, 16, D)[:, :blocks]
        return codes, pages[..., page * D:page * D + page // 16].reshape(Hkv, -1)[:, :blocks]

    def values(cache, b, n):
        """Tokens 0 .. n of sequence b, [n, Hkv, D]."""
        if n == 0:
            return torch.zeros((0, Hkv, D), dtype=torch.float64, device="cuda")
        codes, powers = sequence(cache, b, n)
        return _value(codes, powers[..., None].expand(codes.shape[:3])).flatten(1, 2)[:, :n].transpose(0, 1)

    old, new = _lengths(c)
    if op == "store":
        got, first = ([], []), [sum(new[:b]) for b in range(c["B"])]
        for b in range(c["B"]):
            n, total = old[b], old[b] + new[b]
            for into, cache, x in zip(got, (s["k_cache"], s["v_cache"]), (s["k"], s["v"])):
                held = values(cache, b, n)
                fresh = x[first[b]:first[b] + new[b]].double()
                whole = n // 16 * 16   # tokens of blocks that are full or keep what they have
                if new[b] == 0:
                    into.append(held)
                    continue
                tail = torch.cat((held[whole:], fresh))
                blocks = _cols(total - whole, 16)
                padded = torch.zeros((blocks * 16, Hkv, D), dtype=torch.float64, device="cuda")
                padded[:total - whole] = tail
                size = padded.abs()
                size[:n - whole] = 0   # what a block held has its say by its exponent
                top = size.view(blocks, 16, Hkv, D).amax((1, 3))
                e = torch.full_like(top, float(_HIGH))
                for up in range(_HIGH - 1, _LOW - 1, -1):
                    e = torch.where(_TOP * 2.0 ** up >= top, float(up), e)
                if n > whole:
                    e[0] = torch.maximum(e[0], sequence(cache, b, n)[1][:, -1].double() - _BIAS)
                into += [held[:whole], _nearest(padded, e.repeat_interleave(16, 0).unsqueeze(-1))[:total - whole]]
        return tuple(torch.cat(x) for x in got)
    out, lse = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), torch.full((c["B"], c["H"], 1), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(c["B"]):
        if old[b]:
            k, v = values(s["k_cache"], b, old[b]), values(s["v_cache"], b, old[b])
            q = s["q"][b, :, 0].double().reshape(Hkv, -1, D)
            scores = torch.matmul(q, k.permute(1, 2, 0)) / math.sqrt(D)
            lse[b, :, 0] = torch.logsumexp(scores, -1).reshape(-1)
            out[b, :, 0] = torch.matmul(torch.softmax(scores, -1), v.transpose(0, 1)).reshape(-1, D)
    return out, lse


def work(c):
    """Bytes: every input read once, every output written once.  Operations: two per multiply-add of the attention's products, and
    of the others six per rotated pair and four (eight in the gradient) per normed value."""
    op = c["op"]
    size = 4 if c.get("dtype", BF16) == F32 else 2
    D, Hkv = c["D"], c["Hkv"]
    if op == "norm":
        rows, heads = c["B"] * c["S"], c["H"] + c["Hkv"]
        values, weights = rows * heads * D, 2 * D * (4 if c["weights"] == F32 else 2)
        times = 3 if c["back"] else 2
        return {"bytes": times * values * size + 4 * rows * c["axes"] + weights * (times - 1), "flops": 3.0 * rows * heads * c["R"] + 4.0 * (times - 1) * values}
    old, new = _lengths(c)
    held, fresh = sum(old), sum(new)
    if op == "append":
        values = (c["H"] + 2 * Hkv) * D
        normed = (c["H"] + Hkv) * D if c["weights"] else 0
        return {"bytes": fresh * (values * (size + 2) + 8), "flops": fresh * (3.0 * (c["H"] + Hkv) * c["R"] + 4.0 * normed)}
    row = D + 1 / 16
    if op == "store":
        # new rows in and their codes out, the whole cache's codes in (the new ones are at hand) and its values out
        return {"bytes": 2 * Hkv * (fresh * (D * size + row) + held * row + (held + fresh) * 2 * D), "flops": 2.0 * Hkv * D * (4 * fresh + held + fresh)}
    entries = sum(_cols(n, c["page"]) for n in old)
    return {"bytes": 2 * held * Hkv * row + c["B"] * c["H"] * (4 * D + 4) + 4 * entries, "flops": 4.0 * held * c["H"] * D}
