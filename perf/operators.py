"""Operators of token models in few bits, as cases that can be timed and compared: each in plain torch operations and
through the entry points of `fastertnn_amd.lib`.

Kinds of cases:

  quantize   rows of floats to 8-bit codes with a scale per row (quantize_rows_i8); the codes are whole numbers
  mm8        product of 8-bit rows with scales per token and channel (mm_i8)
  rows       the same against packed ternary or binary weights (mm_i8_rows)
  append     new keys and values, keys and queries rotated by position, into a paged cache of 4-bit codes (kv4_append);
             what the cache then holds of them comes back as values (kv4_read)
  attend     causal attention of the new tokens over such a cache (kv4_attention)

The cache: uint8 [pages][bytes of a page].  A page holds `page` tokens, one block per head: key codes [page][dim], value codes
[page / 8][dim][8] (8 tokens of a channel lie together), two codes per byte, the lower nibble first, then a scale and a zero
in bfloat16 per token for the keys, and the same for the values.  A code c stands for zero + scale c.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # the activations of a few tokens in front of a layer: latency
        dict(kind="quantize", type="bf16", rows=8, k=4096, name="quantize_tokens"),
        # a whole prompt's, in the framework's own fp32, rows of an odd length
        dict(kind="quantize", type="f32", rows=8192, k=11007, name="quantize_prompt"),
        # one token through a layer: the weights are read once
        dict(kind="mm8", type="bf16", m=1, n=4096, k=4096, bias=False, name="mm8_token"),
        # a batch of tokens being generated, odd sizes
        dict(kind="mm8", type="f16", m=61, n=14336, k=4100, bias=True, name="mm8_batch"),
        # a long prompt: bound by the matrix cores
        dict(kind="mm8", type="bf16", m=8192, n=8192, k=8192, bias=False, name="mm8_prompt"),
        # one token through the largest fully connected layer of the reference's driver, ternary weights
        dict(kind="rows", type="bf16", weights="ternary", m=1, n=16384, k=16384, bias=False, name="rows_token"),
        # a prompt against binary weights, odd sizes, the framework's own fp32 result
        dict(kind="rows", type="f32", weights="binary", m=1999, n=5003, k=4100, bias=True, name="rows_prompt"),
        # a step of 48 sequences: one new token each
        dict(kind="append", type="bf16", batch=48, new=1, len=5000, heads=8, group=4, dim=128, page=64, rot=128, pairs="halves", name="append_step"),
        # prompts of different lengths behind what the cache holds already
        dict(kind="append", type="f16", batch=5, new=4001, len=6000, heads=8, group=2, dim=64, page=16, rot=32, pairs="neighbours", name="append_prompts"),
        # one sequence, one token, a long cache: few rows, much to read
        dict(kind="attend", type="bf16", batch=1, new=1, len=65003, heads=8, group=4, dim=128, page=64, name="attend_long"),
        # a batch of sequences of different lengths, one token each
        dict(kind="attend", type="f16", batch=48, new=1, len=5000, heads=8, group=8, dim=64, page=16, name="attend_batch"),
        # prompts of different lengths, the last part of each new
        dict(kind="attend", type="bf16", batch=2, new=2500, len=4099, heads=8, group=4, dim=128, page=32, name="attend_prompts"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(("quantize", "mm8", "mm8", "rows", "rows", "append", "attend", "attend"))
    typ = rng.choice(sorted(TYPES))
    if kind == "quantize":
        return dict(kind=kind, type=typ, rows=_log(rng, 1, 8192), k=_log(rng, 64, 16384))
    if kind in ("mm8", "rows"):
        c = dict(kind=kind, type=typ, m=rng.choice((1, _log(rng, 1, 64), _log(rng, 1, 8192))), n=_log(rng, 64, 16384), k=_log(rng, 64, 16384),
                 bias=rng.random() < 0.5)
        return dict(c, weights=rng.choice(("ternary", "ternary", "binary"))) if kind == "rows" else c
    c = dict(kind=kind, type=rng.choice(("f16", "bf16")), heads=rng.choice((1, 2, 4, 8, 8, 16)), group=rng.choice((1, 2, 3, 4, 4, 7, 8)),
             dim=rng.choice((64, 64, 96, 128, 128, 128, 256)), page=rng.choice((16, 32, 64, 128, 256)))
    if rng.random() < 0.6:
        c.update(batch=_log(rng, 1, 64), new=1, len=_log(rng, 1, 65536))
    else:
        new = _log(rng, 2, 4096)
        c.update(batch=_log(rng, 1, 8), new=new, len=new + _log(rng, 1, 4096) - 1)
    if kind == "append":
        c.update(rot=rng.choice((c["dim"], c["dim"], 32, 0)), pairs=rng.choice(("halves", "neighbours")))
    return c


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 5e12, w["flops"] / 1e15)


def draw(rng):
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0.0), _cost(c))
    while True:
        c = _draw(rng)
        # the plain form's scores and its copy of the cache in fp32 fit the card several times over
        if _cost(c) <= most[c["kind"]] and (c["kind"] != "attend" or _plain_values(c) < 3e9):
            return c


def _plain_values(c):
    return c["batch"] * c["heads"] * c["len"] * (c["new"] * c["group"] + 2 * c["dim"])


def _lengths(c):
    """tokens of each sequence in the cache, the new ones among them, and how many are new: from the case alone"""
    b = c["batch"]
    lens = [max(1, c["len"] - i * c["len"] // (2 * b)) for i in range(b)]
    return lens, [min(lens[i], max(1, c["new"] - i * c["new"] // (2 * b))) for i in range(b)]


def work(case):
    c = case
    if c["kind"] == "quantize":
        n = c["rows"] * c["k"]
        return {"bytes": n * (1 + TYPES[c["type"]].itemsize) + 4 * c["rows"], "flops": 0}
    if c["kind"] in ("mm8", "rows"):
        m, n, k = c["m"], c["n"], c["k"]
        bits = 8 if c["kind"] == "mm8" else 2 if c["weights"] == "ternary" else 1
        return {"bytes": m * k + n * k * bits / 8 + m * n * TYPES[c["type"]].itemsize + 4 * (m + n), "flops": 2 * m * n * k}
    lens, new = _lengths(c)
    h, d, heads_q = c["heads"], c["dim"], c["heads"] * c["group"]
    if c["kind"] == "append":   # keys, values and queries in; 4-bit codes, a scale and a zero, and queries out; what is read back
        return {"bytes": sum(new) * (d * 2 * (2 * h + 2 * heads_q) + 2 * h * (d // 2 + 4) * 2 + 2 * h * d * 2), "flops": 0}
    pairs = sum(n * t - n * (n - 1) // 2 for n, t in zip(new, lens))   # visible (query, key) pairs
    return {"bytes": sum(lens) * h * (d + 8) + 2 * 2 * sum(new) * heads_q * d, "flops": 4 * pairs * heads_q * d}


# ------------------------------------------------------------------------------------------------------------ inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _codes8(g, rows, k):
    """8-bit codes of rows of about normal values, padded with zeros to whole groups of 16, and their scales"""
    q = (torch.randn((rows, k), generator=g, device="cuda") * 32).round_().clamp_(-127, 127).to(torch.int8)
    codes = torch.zeros((rows, -(-k // 16) * 16), dtype=torch.int8, device="cuda")
    codes[:, :k] = q
    return codes, torch.rand((rows,), generator=g, device="cuda") * 0.02 + 0.01


def _words(bits):
    """[rows][64 w] truth values -> [rows][w] words, lane 0 in the lowest bit"""
    b = bits.view(bits.shape[0], -1, 8).to(torch.uint8) << torch.arange(8, device="cuda", dtype=torch.uint8)
    return b.sum(-1, dtype=torch.uint8).view(torch.int64)


def _packed(g, n, k, ternary):
    """rows of uniform lanes as Packing 2 holds them: groups of four words per plane, signs then zeros; binary: signs only"""
    kw = -(-k // 256) * 4
    t = torch.randint(-1, 2, (n, k), generator=g, device="cuda", dtype=torch.int8) if ternary else \
        torch.randint(0, 2, (n, k), generator=g, device="cuda", dtype=torch.int8) * 2 - 1
    sign = torch.zeros((n, kw * 64), dtype=torch.bool, device="cuda")
    sign[:, :k] = t < 0
    if not ternary:
        return _words(sign).reshape(-1)
    zero = torch.ones((n, kw * 64), dtype=torch.bool, device="cuda")
    zero[:, :k] = t == 0
    return torch.stack([_words(sign).view(n, kw // 4, 4), _words(zero).view(n, kw // 4, 4)], 2).reshape(-1)


def _cache(g, c, pages):
    h, d, page = c["heads"], c["dim"], c["page"]
    block = torch.empty((pages, h, page * (d + 8)), dtype=torch.uint8, device="cuda")
    n = page * d
    codes = (torch.randn((pages, h, 2 * n), generator=g, device="cuda") * 3 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
    block[:, :, :n] = codes[..., 0::2] | codes[..., 1::2] << 4
    scale = torch.rand((pages, h, 2 * page), generator=g, device="cuda") * 0.2 + 0.2
    zero = -scale * (7 + torch.rand((pages, h, 2 * page), generator=g, device="cuda"))
    block[:, :, n:] = torch.stack([scale, zero], -1).to(torch.bfloat16).view(pages, h, -1).view(torch.uint8)
    return block.view(pages, -1)


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    kind, typ = case["kind"], TYPES[case["type"]]
    s["dtype"] = typ
    if kind == "quantize":
        s["x"] = (torch.randn((case["rows"], case["k"]), generator=g, device="cuda") * (0.5 + torch.rand((case["rows"], 1), generator=g, device="cuda"))).to(typ)
        return s
    if kind in ("mm8", "rows"):
        s["a"], s["sa"] = _codes8(g, case["m"], case["k"])
        s["bias_n"] = torch.randn((case["n"],), generator=g, device="cuda") if case["bias"] else None
        if kind == "mm8":
            s["b"], s["sb"] = _codes8(g, case["n"], case["k"])
        else:
            s["b"] = _packed(g, case["n"], case["k"], case["weights"] == "ternary")
            s["sb"] = torch.rand((case["n"],), generator=g, device="cuda") * 0.02 + 0.01
        return s
    lens, new = _lengths(case)
    page = case["page"]
    width = -(-max(lens) // page)
    pages = case["batch"] * width + 3
    s["cache"] = _cache(g, case, pages)
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    s["table"] = torch.tensor(order[:case["batch"] * width], dtype=torch.int32, device="cuda").view(case["batch"], width)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["tokens"], s["most_new"], s["most_len"] = starts[-1], max(new), max(lens)
    t, h, d = starts[-1], case["heads"], case["dim"]
    s["q"] = torch.randn((t, h * case["group"], d), generator=g, device="cuda").to(typ)
    if kind == "append":
        s["k"], s["v"] = (torch.randn((t, h, d), generator=g, device="cuda").to(typ) for _ in range(2))
        s["cos"] = s["sin"] = None
        if case["rot"]:
            rot = case["rot"]
            at = torch.arange(width * page, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
            s["cos"], s["sin"] = at.cos().float(), at.sin().float()
    return s


# -------------------------------------------------------------------------------------------------------- plain forms

def _plain_quantize(s):
    x = s["x"]
    most = x.float().abs().amax(1)
    q = torch.round(x.double() * 127 / most.double()[:, None].clamp_min(1e-300)).to(torch.int8)   # 64 bits: codes next to a border
    pad = -(-x.shape[1] // 16) * 16 - x.shape[1]
    return {"q": torch.nn.functional.pad(q, (0, pad)), "scale": (most.double() / 127).float()}


def _bits(words, n):
    """[n][...] words as lanes of truth values, [n][lanes]"""
    b = words.view(torch.uint8).view(n, -1, 1) >> torch.arange(8, device="cuda", dtype=torch.uint8)
    return (b & 1).view(n, -1)


def _plain_product(s):
    n, k = s["n"], s["k"]
    if s["kind"] == "mm8":
        b = s["b"][:, :k].float()
    elif s["weights"] == "ternary":
        planes = s["b"].view(n, -1, 2, 4)
        sign, zero = (_bits(planes[:, :, i].contiguous(), n)[:, :k] for i in (0, 1))
        b = (1 - 2 * sign.float()) * (1 - zero.float())
    else:
        b = 1 - 2 * _bits(s["b"], n)[:, :k].float()
    y = torch.matmul(s["a"][:, :k].float(), b.t()) * s["sa"][:, None] * s["sb"]
    return (y if s["bias_n"] is None else y + s["bias_n"]).to(s["dtype"])


def _split(cache, s):
    """views of a cache's parts: key codes [pages][heads][page][dim / 2], value codes [pages][heads][page / 8][dim][4], (scale, zero) of each"""
    h, d, page = s["heads"], s["dim"], s["page"]
    block = cache.view(cache.shape[0], h, page * (d + 8))
    n = page * d // 2
    params = block[:, :, 2 * n:].view(torch.bfloat16).unflatten(2, (2, page, 2))
    return (block[:, :, :n].unflatten(2, (page, d // 2)), block[:, :, n:2 * n].unflatten(2, (page // 8, d, 4)), params[:, :, 0], params[:, :, 1])


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _places(s):
    """sequence and position of each new token"""
    t = torch.arange(s["tokens"], device="cuda")
    b = torch.searchsorted(s["starts"][1:].long(), t, right=True)
    return t, b, s["lens"].long()[b] - s["starts"].long()[b + 1] + t


def _plain_rotate(x, s, pos):
    """the rotated values, computed in 64 bits and rounded once to 32"""
    if not s["rot"]:
        return x.float()
    rot = s["rot"]
    c, n = s["cos"][pos].double()[:, None], s["sin"][pos].double()[:, None]
    y = x.double()
    if s["pairs"] == "halves":
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        turned = torch.cat([a * c - b * n, b * c + a * n], -1)
    else:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    return torch.cat([turned, y[..., rot:]], -1).float()


def _plain_codes(y):
    y = y.double()   # 64 bits: values next to a border between two codes
    low, high = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    zero, scale = low.float().to(torch.bfloat16), ((high - low) / 15).float().to(torch.bfloat16)
    code = torch.round((y - zero.double()) / scale.double()).clamp_(0, 15)
    return torch.where(scale.float() > 0, code, 0).to(torch.uint8), torch.cat([scale, zero], -1)


def _plain_append(s):
    t, b, pos = _places(s)
    d, page = s["dim"], s["page"]
    kc, vc, kp, vp = _split(s["cache"], s)
    at, slot = s["table"].long()[b, pos // page], pos % page
    codes, params = _plain_codes(_plain_rotate(s["k"], s, pos))
    kc[at, :, slot] = codes[..., 0::2] | codes[..., 1::2] << 4
    kp[at, :, slot] = params
    codes, params = _plain_codes(s["v"].float())
    vp[at, :, slot] = params
    # a byte holds a channel's codes of two tokens: its other token is the neighbour, if that is new too, or what the cache holds
    held = vc[at, :, slot // 8, :, slot % 8 // 2]
    odd = (pos % 2 == 1)[:, None, None]
    other = torch.where(pos % 2 == 1, t - 1, t + 1)
    there = (other >= s["starts"].long()[b]) & (other < s["starts"].long()[b + 1])
    other = torch.where(there[:, None, None], codes[other.clamp(0, s["tokens"] - 1)], torch.where(odd, held & 15, held >> 4))
    vc[at, :, slot // 8, :, slot % 8 // 2] = torch.where(odd, other | codes << 4, codes | other << 4)
    # and what it holds of the new tokens now
    k = _nibbles(kc[at, :, slot]).float() * kp[at, :, slot][..., :1].float() + kp[at, :, slot][..., 1:].float()
    v = vc[at, :, slot // 8, :, slot % 8 // 2]
    v = torch.where(odd, v >> 4, v & 15).float() * vp[at, :, slot][..., :1].float() + vp[at, :, slot][..., 1:].float()
    return {"q": _plain_rotate(s["q"], s, pos).to(s["dtype"]), "k": k.to(s["dtype"]), "v": v.to(s["dtype"])}


def _plain_attend(s):
    h, g, d, page, n = s["heads"], s["group"], s["dim"], s["page"], s["most_new"]
    batch, width = s["table"].shape
    kc, vc, kp, vp = _split(s["cache"], s)
    at = s["table"].long()
    k = _nibbles(kc[at]).float() * kp[at][..., :1].float() + kp[at][..., 1:].float()                      # [batch][width][heads][page][dim]
    v = _nibbles(vc[at]).permute(0, 1, 2, 3, 5, 4).flatten(3, 4).float() * vp[at][..., :1].float() + vp[at][..., 1:].float()
    k, v = (x.transpose(1, 2).reshape(batch, h, width * page, d)[:, :, :s["most_len"]] for x in (k, v))
    starts, lens = s["starts"].long(), s["lens"].long()
    new = starts[1:] - starts[:-1]
    row = (starts[:-1, None] + torch.arange(n, device="cuda")).clamp_(max=s["tokens"] - 1)
    q = s["q"][row].float().view(batch, n, h, g, d).permute(0, 2, 1, 3, 4).reshape(batch, h, n * g, d)
    p = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5).view(batch, h, n, g, -1)
    last = (lens - new)[:, None] + torch.arange(n, device="cuda")                                           # a token sees itself and what lies before it
    p.masked_fill_((torch.arange(s["most_len"], device="cuda") > last[..., None])[:, None, :, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p.view(batch, h, n * g, -1), v).view(batch, h, n, g, d) / p.sum(-1, keepdim=True)
    t, b, _ = _places(s)
    return o.permute(0, 2, 1, 3, 4).flatten(2, 3)[b, t - starts[b]].to(s["dtype"])


# ------------------------------------------------------------------------------------------------------------- passes

def _own(s):
    import fastertnn_amd.lib as lib
    kind = s["kind"]
    if kind == "quantize":
        q, scale = lib.quantize_rows_i8(s["x"])
        return {"q": q, "scale": scale}
    if kind == "mm8":
        return lib.mm_i8(s["a"], s["sa"], s["b"], s["sb"], s["k"], bias=s["bias_n"], dtype=s["dtype"])
    if kind == "rows":
        return lib.mm_i8_rows(s["a"], s["sa"], s["b"], s["sb"], s["n"], s["k"], s["weights"] == "ternary", bias=s["bias_n"], dtype=s["dtype"])
    if kind == "append":
        q = lib.kv4_append(s["cache"], s["table"], s["lens"], s["starts"], s["k"], s["v"], s["page"], q=s["q"], cos=s["cos"], sin=s["sin"],
                           neighbours=s["pairs"] == "neighbours")
        k, v = lib.kv4_read(s["cache"], s["table"], s["lens"], s["starts"], s["tokens"], s["heads"], s["dim"], s["page"], dtype=s["dtype"])
        return {"q": q, "k": k, "v": v}
    return lib.kv4_attention(s["q"], s["cache"], s["table"], s["lens"], s["starts"], s["heads"], s["page"])


def run(s):
    if own:
        return _own(s)
    kind = s["kind"]
    if kind == "quantize":
        return _plain_quantize(s)
    if kind in ("mm8", "rows"):
        return _plain_product(s)
    return _plain_append(s) if kind == "append" else _plain_attend(s)


# ------------------------------------------------------------------------------------------------------ from 64 bits

def _exact_sequence(s, b, head, length, values):
    """a head's keys or values of a sequence, [length][dim] in 64 bits"""
    d, size = s["dim"], s["page"]
    t, i = torch.arange(length, device="cuda")[:, None], torch.arange(d, device="cuda")
    page, slot, start, n = s["table"][b].long()[t // size], t % size, head * size * (d + 8), size * d // 2
    if values:
        code = s["cache"][page, start + n + (slot // 8 * d + i) * 4 + slot % 8 // 2] >> (4 * (slot % 2)).to(torch.uint8)
    else:
        code = s["cache"][page, start + slot * (d // 2) + i // 2] >> (4 * (i % 2)).to(torch.uint8)
    four = s["cache"][page, start + 2 * n + values * 4 * size + slot * 4 + torch.arange(4, device="cuda")]
    scale, zero = four.view(torch.bfloat16).double().split(1, 1)
    return zero + scale * (code & 15).double()


def _exact_attend(s):
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    starts, g = s["starts"].tolist(), s["group"]
    for b, length in enumerate(s["lens"].tolist()):
        new = starts[b + 1] - starts[b]
        hidden = torch.arange(length, device="cuda") > torch.arange(length - new, length, device="cuda")[:, None]
        for head in range(s["heads"]):
            k, v = (_exact_sequence(s, b, head, length, i) for i in (0, 1))
            for j in range(head * g, (head + 1) * g):
                q = s["q"][starts[b]:starts[b + 1], j].double()
                score = (q @ k.t().contiguous() / math.sqrt(s["dim"])).masked_fill(hidden, -math.inf)
                out[starts[b]:starts[b + 1], j] = torch.softmax(score, -1) @ v
    return out


def _exact_turn(x, s, pos):
    x = x.double().clone()
    rot = s["rot"]
    for i in range(rot // 2):
        a, b = (i, i + rot // 2) if s["pairs"] == "halves" else (2 * i, 2 * i + 1)
        c, n = (s[f][pos, i].double()[:, None] for f in ("cos", "sin"))
        x[..., a], x[..., b] = x[..., a] * c - x[..., b] * n, x[..., b] * c + x[..., a] * n
    return x


def _exact_append(s):
    starts = s["starts"].tolist()
    pos = torch.cat([torch.arange(n - (starts[b + 1] - starts[b]), n, device="cuda") for b, n in enumerate(s["lens"].tolist())])
    got = {"q": _exact_turn(s["q"], s, pos)}
    for name in ("k", "v"):
        y = _exact_turn(s["k"], s, pos) if name == "k" else s["v"].double()
        zero = y.min(-1, keepdim=True)[0].float().bfloat16().double()
        scale = ((y.max(-1, keepdim=True)[0] - y.min(-1, keepdim=True)[0]) / 15).float().bfloat16().double()
        got[name] = zero + scale * torch.nan_to_num(((y - zero) / scale).round().clamp(0, 15), nan=0.0)
    return got


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        x = s["x"].double()
        return {"q": None, "scale": x.abs().max(1)[0] / 127}
    if kind in ("mm8", "rows"):
        n, k = case["n"], case["k"]
        if kind == "mm8":
            b = s["b"][:, :k].double()
        else:
            ternary = case["weights"] == "ternary"
            words = s["b"].view(n, -1, 8) if ternary else s["b"].view(n, -1, 4)
            b = torch.empty((n, words.shape[1] * 256), dtype=torch.float64, device="cuda")
            for bit in range(64):
                lane = (1 - 2 * (words[:, :, :4] >> bit & 1)).double()
                if ternary:
                    lane *= 1 - (words[:, :, 4:] >> bit & 1)
                b[:, bit::64] = lane.view(n, -1)
            b = b[:, :k]
        y = s["sa"].double()[:, None] * (s["a"][:, :k].double() @ b.t().contiguous()) * s["sb"].double()
        return y if s["bias_n"] is None else y + s["bias_n"].double()
    return _exact_append(s) if kind == "append" else _exact_attend(s)
