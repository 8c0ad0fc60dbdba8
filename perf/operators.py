"""Timed operators of the 8-bit block cache, and what they compute in plain torch.

The cache holds the keys and values of `page` consecutive tokens of one head in 8 bits (whole numbers -127 .. 127, or
e4m3 floats) with one fp32 scale for each page, head and side; a table names the pages of every sequence.

    write   append_blocks, then read_blocks: new tokens are quantised into the pages (a page that was begun before keeps
            one scale: its tokens are re-quantised where the new ones need a larger one), and the values that the cache now
            stands for are read back
    read    read_blocks: a run of tokens of every sequence as dense rows, for re-encoding or for another cache
    decode  decode_blocks: attention of one new token of every sequence over its pages
    attend  attend_blocks: causal attention of the last tokens of every sequence (a prompt's chunk, drafted tokens)

Keys, values and queries are seeded Gaussians with a lognormal(0, 0.5) scale per channel, the distribution of the
benchmark configurations of this repository; pages lie in random physical order.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
STORE = {"i8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


def _case(name, kind, B, Hq, Hkv, dh, ctx, new, page, store, src, out, uneven, first):
    return dict(name=name, kind=kind, B=B, Hq=Hq, Hkv=Hkv, dh=dh, ctx=ctx, new=new, page=page, store=store, src=src, out=out,
                uneven=uneven, first=first)


def listed():
    return [
        # one decode step's new token: a few short sequences of a 1B-class head shape (the smallest call: latency), and
        # the 16 x 8K batch; the page that the token fell into is read back
        _case("write_step_b3_2k_dh64", "write", 3, 32, 8, 64, 2049, 1, 16, "i8", "f32", "f32", True, False),
        _case("write_step_b16_8k", "write", 16, 32, 8, 128, 8192, 1, 64, "e4m3", "bf16", "bf16", False, False),
        # prompts coming in: a short odd one beside shorter ones, and a long one
        _case("write_prompt_777", "write", 3, 32, 8, 128, 777, 0, 16, "i8", "bf16", "f32", True, False),
        _case("write_prompt_32k", "write", 1, 32, 8, 128, 32768, 0, 16, "i8", "bf16", "bf16", False, False),
        # tokens that leave the 8-bit cache for the bit-packed pages: their rows for the encoder
        _case("read_500", "read", 2, 32, 8, 64, 4001, 500, 32, "e4m3", "f16", "f16", True, False),
        _case("read_8k", "read", 4, 32, 8, 128, 8190, 8000, 128, "i8", "bf16", "f32", True, False),
        # decode attention, the serving loop: the shapes of the decode cases of perf/cases.py
        _case("decode_b1_2k_dh64", "decode", 1, 32, 8, 64, 2048, 1, 16, "i8", "f32", "f16", False, False),
        _case("decode_b16_8k", "decode", 16, 32, 8, 128, 8192, 1, 16, "i8", "bf16", "bf16", False, False),
        _case("decode_b8_32k", "decode", 8, 32, 8, 128, 32768, 1, 64, "e4m3", "bf16", "bf16", False, False),
        # rows of different, odd lengths whose oldest tokens live in another cache; fp32 for the merge with it
        _case("decode_b3_6k_first", "decode", 3, 32, 8, 128, 6001, 1, 128, "i8", "f32", "f32", True, True),
        # several tokens a sequence: short odd pieces of a batch, and a prompt's chunk behind a long context (the largest)
        _case("attend_b5_6k", "attend", 5, 32, 8, 128, 6001, 301, 128, "e4m3", "f16", "f16", True, True),
        _case("attend_b1_32k", "attend", 1, 32, 8, 128, 32768, 2048, 16, "i8", "bf16", "bf16", False, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write"] * 3 + ["read"] + ["decode"] * 4 + ["attend"] * 3)
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (16, 2), (16, 8), (8, 8), (28, 4)])
    dh = rng.choice([64, 128, 128])
    page = rng.choice([16, 16, 32, 64, 128])
    store = rng.choice(["i8", "i8", "e4m3"])
    src = rng.choice(["bf16", "bf16", "f16", "f32"])
    out = rng.choice(["bf16", "f16", "f32"])
    uneven = rng.random() < 0.6
    first = rng.random() < 0.3
    B = rng.choice([1, 1, 2, 3, 5, 8, 16])
    if kind == "write":
        if rng.random() < 0.5:
            ctx, new = _log(rng, 64, 8192), rng.choice([1, 1, 2, 5])
        else:
            B = min(B, 5)
            ctx, new = _log(rng, 64, 32768 // B), 0
        first = False
    elif kind == "read":
        ctx = _log(rng, 128, 8192)
        new = max(1, int(ctx * rng.uniform(0.1, 0.95)))
        first = False
    elif kind == "decode":
        ctx, new = _log(rng, 128, min(131072, 2000000 // (B * Hkv))), 1
    else:
        src, out = rng.choice(["bf16", "f16"]), rng.choice(["bf16", "f16"])
        B = min(B, 5)
        new = rng.choice([_log(rng, 2, 32), _log(rng, 32, 1024), _log(rng, 32, 1024)])
        ctx = _log(rng, max(128, new), max(256, min(32768, 16000000 // (B * new))))
    c = _case("", kind, B, Hq, Hkv, dh, ctx, new, page, store, src, out, uneven, first)
    c.pop("name")
    return c


# ---- what a case's rows hold -----------------------------------------------------------------------------------
def _lens(c):
    """Tokens of every sequence, the new ones among them: all `ctx`, or an uneven batch down to a quarter of it."""
    if not c["uneven"]:
        return [c["ctx"]] * c["B"]
    B = c["B"]
    return [max(1, c["ctx"] - (3 * c["ctx"] * b) // (4 * B) - (b % 2)) for b in range(B)]


def _news(c):
    """Tokens of every sequence that this call is about; `new` 0 stands for whole prompts."""
    n = _lens(c)
    if c["new"] == 0:
        return n
    if not c["uneven"] or c["kind"] == "decode" or c["new"] <= 5:
        return [min(c["new"], x) for x in n]
    return [min(x, max(1, c["new"] - (c["new"] * b) // c["B"])) for b, x in enumerate(n)]


def _back(c):
    """Tokens of every sequence that a `write` reads back: a prompt's own, or about a page's where tokens are appended."""
    if c["kind"] != "write" or c["new"] == 0:
        return _news(c)
    return [min(x, c["page"]) for x in _lens(c)]


def _firsts(c):
    return [x // 3 if c["first"] else 0 for x in _lens(c)]


def _pairs(c):
    """(query, key) pairs that attention of one head has to look at, over all sequences."""
    total = 0
    for length, n, f in zip(_lens(c), _news(c), _firsts(c)):
        lo = max(length - n, f)  # positions below `first` see nothing
        total += sum((lo + 1 - f, length - f)) * (length - lo) // 2 if length > lo else 0
    return total


def work(c):
    row = c["Hkv"] * c["dh"]
    new = sum(_news(c))
    if c["kind"] == "write":
        old = 0 if c["new"] == 0 else sum(_back(c)) - new
        return {"bytes": 2 * row * (new * SIZE[c["src"]] + new + old + sum(_back(c)) * SIZE[c["out"]]), "flops": 6 * row * new}
    if c["kind"] == "read":
        return {"bytes": 2 * row * new * (1 + SIZE[c["out"]]), "flops": 2 * row * new}
    keys = sum(x - f for x, f in zip(_lens(c), _firsts(c)))
    heads = c["Hq"] * c["dh"]
    return {"bytes": 2 * row * keys + new * heads * (SIZE[c["src"]] + SIZE[c["out"]]), "flops": 4 * heads * _pairs(c)}


# ---- inputs ----------------------------------------------------------------------------------------------------
def _filled(g, scale, pages, c):
    """Pages of random tokens in 8 bits with their scales."""
    kind, top = STORE[c["store"]]
    x = torch.randn(pages, c["Hkv"], c["page"], c["dh"], generator=g, device=DEV).mul_(scale)
    s = x.abs().amax((2, 3)) / top
    x.div_(s[:, :, None, None])
    return (x.round_() if kind is torch.int8 else x).to(kind), s


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    lens, news, back = _lens(c), _news(c), _back(c)
    B, N = c["B"], c["page"]
    blocks = [-(-x // N) for x in lens]
    pages = sum(blocks)
    table = torch.full((B, max(blocks)), -1, dtype=torch.int32)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed))).to(torch.int32)
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = order[at:at + n]
        at += n
    scale = torch.exp(0.5 * torch.randn(c["dh"], generator=g, device=DEV))
    k_codes, k_scale = _filled(g, scale, pages, c)
    v_codes, v_scale = _filled(g, scale, pages, c)
    i32 = dict(dtype=torch.int32, device=DEV)
    offsets = [[sum(n[:b]) for b in range(B + 1)] for n in (news, back)]
    s = dict(kind=c["kind"], page=N, Hkv=c["Hkv"], top=STORE[c["store"]][1], rows=sum(news), rows_back=sum(back), most=max(news),
             out=DT[c["out"]], sm_scale=1.0 / math.sqrt(c["dh"]), table=table.to(DEV), lens=torch.tensor(lens, **i32),
             cu=torch.tensor(offsets[0], **i32), cu_back=torch.tensor(offsets[1], **i32), k_codes=k_codes, v_codes=v_codes, k_scale=k_scale,
             v_scale=v_scale, first=torch.tensor(_firsts(c), **i32) if c["first"] else None)
    if c["kind"] == "write":
        s["k"] = (torch.randn(sum(news), c["Hkv"], c["dh"], generator=g, device=DEV) * scale).to(DT[c["src"]])
        s["v"] = (torch.randn(sum(news), c["Hkv"], c["dh"], generator=g, device=DEV) * scale).to(DT[c["src"]])
    elif c["kind"] != "read":
        s["q"] = (torch.randn(sum(news), c["Hq"], c["dh"], generator=g, device=DEV) * scale).to(DT[c["src"]])
    if own:  # the handle that a serving program keeps for its whole life
        import importlib
        sk = importlib.import_module("spherical-kv_b200")
        s["sk"] = sk
        s["cache"] = sk.BlockCache(k_codes=k_codes, v_codes=v_codes, k_scale=k_scale, v_scale=v_scale, block_table=s["table"],
                                   seq_lens=s["lens"])
    return s


# ---- the plain form --------------------------------------------------------------------------------------------
def _places(s, cu, rows):
    """Row, position, page and slot of each of `rows` tokens, the last cu[b + 1] - cu[b] of every sequence b."""
    i = torch.arange(rows, device=DEV)
    b = torch.searchsorted(cu.long(), i, right=True) - 1
    pos = s["lens"].long()[b] - cu.long()[b + 1] + i
    return b, pos, s["table"].long()[b, pos // s["page"]], pos % s["page"]


def _rounded(x, codes):
    """float64 quotients in the cache's 8 bits: the nearest code, ties to the even one."""
    if codes.dtype is torch.int8:
        return x.round().to(torch.int8)
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -20))), min=-6.0) - 3.0)
    return ((x / step).round() * step).float().to(codes.dtype)


def _write_side(s, x, codes, scale):
    b, pos, page, slot = _places(s, s["cu"], s["rows"])
    start = s["lens"].long() - (s["cu"][1:] - s["cu"][:-1]).long()
    begun = (s["cu"][1:] > s["cu"][:-1]) & (start % s["page"] > 0)  # sequences whose first new token joins a begun page
    head = s["table"].long().gather(1, (start // s["page"]).clamp(max=s["table"].shape[1] - 1)[:, None])[:, 0].clamp(min=0)
    need = (torch.zeros_like(scale).index_reduce_(0, page, x.float().abs().amax(-1), "amax").double() / s["top"]).float()
    before = torch.where(begun[:, None], scale[head], 0.0)                     # [B, Hkv]
    after = torch.where(begun[:, None], torch.maximum(before, need[head]), 0.0)
    touched = torch.zeros(scale.shape[0], dtype=torch.bool, device=DEV)
    touched[page] = True
    scale.copy_(torch.where(touched[:, None], need, scale))
    scale.index_reduce_(0, head, after, "amax")
    ratio = torch.where((before > 0)[..., None, None], before.double()[..., None, None] / after.double()[..., None, None], 1.0)
    old = codes[head].double() * ratio
    held = begun[:, None, None, None] & (torch.arange(s["page"], device=DEV) < (start % s["page"])[:, None])[:, None, :, None]
    kept = torch.where(held, _rounded(old, codes).float(), codes[head].float())
    codes[head] = torch.where(begun[:, None, None, None], kept, codes[head].float()).to(codes.dtype)
    codes[page, :, slot] = _rounded(x.double() / scale[page].double()[..., None].clamp(min=2.0 ** -126), codes)


def _read_side(s, cu, rows, codes, scale):
    b, pos, page, slot = _places(s, cu, rows)
    return (codes[page, :, slot].float() * scale[page][..., None]).to(s["out"])


def _attend(s):
    B, N, most = s["lens"].shape[0], s["page"], s["most"]
    q = s["q"].float()
    b, pos, _, _ = _places(s, s["cu"], s["rows"])
    i = torch.arange(s["rows"], device=DEV) - s["cu"].long()[b]
    padded = q.new_zeros(B, most, *q.shape[1:])
    padded[b, i] = q
    at = torch.full((B, most), -1, device=DEV)
    at[b, i] = pos
    page = s["table"].long().clamp(min=0)                                      # [B, blocks]
    k = (s["k_codes"][page].float() * s["k_scale"][page][..., None, None]).transpose(1, 2).flatten(2, 3)  # [B, Hkv, T, dh]
    v = (s["v_codes"][page].float() * s["v_scale"][page][..., None, None]).transpose(1, 2).flatten(2, 3)
    group = q.shape[1] // s["Hkv"]
    rows = padded.reshape(B, most, s["Hkv"], group, -1).permute(0, 2, 3, 1, 4).flatten(2, 3)              # [B, Hkv, group * most, dh]
    x = torch.matmul(rows, k.transpose(2, 3)).mul_(s["sm_scale"]).unflatten(2, (group, most))
    t = torch.arange(k.shape[2], device=DEV)
    seen = t <= at[:, :, None]
    if s["first"] is not None:
        seen = seen & (t >= s["first"].long()[:, None, None])
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    w = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.flatten(2, 3), v).unflatten(2, (group, most)) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3)[b, i].to(s["out"])           # [rows, Hq, dh]


def run(s):
    if own:
        sk, cache = s["sk"], s["cache"]
        if s["kind"] == "write":
            sk.append_blocks(cache, s["k"], s["v"], cu_new=s["cu"])
            return sk.read_blocks(cache, cu_rows=s["cu_back"], rows=s["rows_back"], out_dtype=s["out"])
        if s["kind"] == "read":
            return sk.read_blocks(cache, cu_rows=s["cu_back"], rows=s["rows_back"], out_dtype=s["out"])
        if s["kind"] == "decode":
            return sk.decode_blocks(s["q"], cache, first=s["first"], out_dtype=s["out"])
        return sk.attend_blocks(s["q"], cache, cu_new=s["cu"], first=s["first"], out_dtype=s["out"])
    if s["kind"] == "write":
        _write_side(s, s["k"], s["k_codes"], s["k_scale"])
        _write_side(s, s["v"], s["v_codes"], s["v_scale"])
    if s["kind"] in ("write", "read"):
        return (_read_side(s, s["cu_back"], s["rows_back"], s["k_codes"], s["k_scale"]),
                _read_side(s, s["cu_back"], s["rows_back"], s["v_codes"], s["v_scale"]))
    return _attend(s)


# ---- from the definition, in 64 bits ----------------------------------------------------------------------------
def _nearest(y, store):
    """The nearest value of the 8-bit format, by the list of its values (ties to the even code)."""
    if store == "i8":
        f = torch.floor(y)
        up = (y - f > 0.5) | ((y - f == 0.5) & (f % 2 != 0))
        return (f + up).clamp(-127, 127)
    values = torch.arange(0, 127, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn).double()
    mid = (values[1:] + values[:-1]) / 2
    a = y.abs()
    i = torch.bucketize(a, mid)                     # first midpoint that is not below a
    tie = (i < mid.numel()) & (a == mid[i.clamp(max=mid.numel() - 1)])
    return values[i + (tie & (i % 2 == 1))] * torch.sign(y)


def exact(c, seed):
    s = prepare(c, seed)
    lens, news, back, firsts, N = _lens(c), _news(c), _back(c), _firsts(c), c["page"]
    table = s["table"].tolist()
    if c["kind"] in ("write", "read"):
        sides = []
        for side in ("k", "v"):
            codes, scale = s[side + "_codes"].double(), s[side + "_scale"].double()
            at = 0
            for b in range(c["B"]) if c["kind"] == "write" else ():
                x = s[side][at:at + news[b]].double().transpose(0, 1)       # [Hkv, n, dh]
                at += news[b]
                p = lens[b] - news[b]
                done = 0
                while p < lens[b]:
                    pg, lo = table[b][p // N], p % N
                    n = min(N - lo, lens[b] - p)
                    part = x[:, done:done + n]
                    top = (part.abs().amax((1, 2)) / s["top"]).float().double()
                    if lo:
                        grown = torch.maximum(top, scale[pg])
                        moved = _nearest(codes[pg, :, :lo] * scale[pg][:, None, None] / grown[:, None, None], c["store"])
                        codes[pg, :, :lo] = torch.where((grown > scale[pg])[:, None, None], moved, codes[pg, :, :lo])
                        top = grown
                    scale[pg] = top
                    codes[pg, :, lo:lo + n] = _nearest(part / top[:, None, None], c["store"])
                    p, done = p + n, done + n
            out = []
            for b in range(c["B"]):
                t = torch.arange(lens[b] - back[b], lens[b], device=DEV)
                pg = s["table"][b].long()[t // N]
                out.append(codes[pg, :, t % N] * scale[pg][..., None])
            sides.append(torch.cat(out))
        return tuple(sides)
    out, at, group = [], 0, c["Hq"] // c["Hkv"]
    for b in range(c["B"]):
        t = torch.arange(firsts[b], lens[b], device=DEV)
        pg = s["table"][b].long()[t // N]
        q = s["q"][at:at + news[b]].double()
        at += news[b]
        i = torch.arange(lens[b] - news[b], lens[b], device=DEV)
        hidden = t[None, :] > i[:, None]
        heads = []
        for h in range(c["Hkv"]):
            k = s["k_codes"][pg, h, t % N].double() * s["k_scale"][pg, h].double()[:, None]
            v = s["v_codes"][pg, h, t % N].double() * s["v_scale"][pg, h].double()[:, None]
            for j in range(group):
                x = (q[:, h * group + j] @ k.T / math.sqrt(c["dh"])).masked_fill(hidden, -math.inf)
                p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0) if t.numel() else x
                heads.append(p @ v)
        out.append(torch.stack(heads, 1))
    return torch.cat(out)
