"""The cache of keys and values in 4-bit codes, bit for bit, and attention over it, against 64 bits."""
import math
import random

import pytest

torch = pytest.importorskip("torch")
import fastertnn_amd.lib as lib
from tests import tokens_oracle as ref

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _setup(seed, heads, dim, page, lens, new, spare=2, tokens=None, calm=True):
    """a cache of random bytes (`calm`: scales and zeros of ordinary size), a shuffled table, and the arrays of a call"""
    g = _gen(seed)
    width = max(1, -(-max(lens + [1]) // page))
    pages = len(lens) * width + spare
    raw = torch.randint(0, 256, (pages, lib.kv4_page_bytes(heads, dim, page)), generator=g, dtype=torch.uint8)
    if calm:
        block = raw.view(pages, heads, -1)
        scale = torch.rand((pages, heads, 2, page), generator=g) * 0.3 + 0.05
        zero = -scale * (5 + 4 * torch.rand((pages, heads, 2, page), generator=g))
        block[:, :, page * dim:] = torch.stack([scale, zero], -1).bfloat16().view(torch.uint8).reshape(pages, heads, -1)
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    table = torch.tensor(order[:len(lens) * width], dtype=torch.int32).view(len(lens), width)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return raw, table, torch.tensor(lens, dtype=torch.int32), torch.tensor(starts, dtype=torch.int32), tokens or starts[-1]


def _cuda(*tensors):
    return [t.cuda() for t in tensors]


def _tables(positions, rot):
    at = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return at.cos().float(), at.sin().float()


# heads, dim, page, lens, new, rotated channels
APPENDS = [(1, 64, 16, [1], [1], 64), (2, 128, 64, [5, 1, 130], [5, 1, 1], 128), (3, 96, 32, [40, 33], [17, 9], 96), (2, 256, 128, [300, 7, 129], [290, 7, 2], 64),
           (8, 128, 16, [100, 8, 9, 16, 17, 63], [3, 8, 1, 7, 17, 50], 32), (1, 64, 256, [700], [699], 6), (2, 96, 16, [31, 0, 40], [8, 0, 0], 0),
           (4, 128, 64, [64] * 70, [1] * 70, 128)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("heads,dim,page,lens,new,rot", APPENDS)
def test_append_and_read(heads, dim, page, lens, new, rot, neighbours, dtype):
    t = TYPES[dtype]
    raw, table, ln, st, tokens = _setup(dim + page, heads, dim, page, lens, new)
    g = _gen(rot + len(lens))
    k, v, q = (torch.randn((tokens, h, dim), generator=g).to(t) for h in (heads, heads, 2 * heads))
    cos, sin = _tables(max(lens), rot) if rot else (None, None)
    want = ref.Cache(raw, heads, dim, page)
    assert torch.equal(want.raw(), raw)
    wq = torch.empty_like(q)
    ref.append(want, table, ln, st, k, v, cos, sin, neighbours, q, wq)
    cache, dt, dl, ds = _cuda(raw, table, ln, st)
    args = (cache, dt, dl, ds)
    got = lib.kv4_append(*args, k.cuda(), v.cuda(), page, q=q.cuda(), cos=None if cos is None else cos.cuda(), sin=None if sin is None else sin.cuda(),
                         neighbours=neighbours)
    assert torch.equal(cache.cpu(), want.raw())
    assert torch.equal(got.cpu(), wq)
    gk, gv = lib.kv4_read(*args, tokens, heads, dim, page, dtype=t)
    wk, wv = ref.read(want, table, ln, st, tokens, t)
    assert torch.equal(gk.cpu(), wk) and torch.equal(gv.cpu(), wv)


def test_append_token_by_token_gives_the_cache_of_one_call():
    heads, dim, page, n = 2, 128, 32, 45
    raw, table, ln, st, _ = _setup(3, heads, dim, page, [n, n - 9], [n, n - 9])
    g = _gen(4)
    k, v = (torch.randn((2 * n - 9, heads, dim), generator=g).bfloat16().cuda() for _ in range(2))
    cos, sin = _cuda(*_tables(n, dim))
    once, table = _cuda(raw, table)
    lib.kv4_append(once, table, ln.cuda(), st.cuda(), k, v, page, cos=cos, sin=sin)
    steps = raw.cuda()
    for i in range(n):
        new = [1, int(i < n - 9)]
        rows = [i, n + i][:sum(new)]
        starts = torch.tensor([0, 1, sum(new)], dtype=torch.int32).cuda()
        lens = torch.tensor([i + 1, min(i + 1, n - 9)], dtype=torch.int32).cuda()
        lib.kv4_append(steps, table, lens, starts, k[rows], v[rows], page, cos=cos, sin=sin)
    assert torch.equal(once, steps)


@pytest.mark.parametrize("dtype", TYPES)
def test_append_of_special_values(dtype):
    """constant groups, zeros, a NaN, an infinity, the largest and the smallest numbers, values at borders between codes"""
    t = TYPES[dtype]
    heads, dim, page = 1, 64, 16
    raw, table, ln, st, n = _setup(5, heads, dim, page, [12], [12])
    k = torch.randn((n, 1, dim), generator=_gen(6)).to(t)
    k[0], k[1], k[2, 0, 5], k[3, 0, 63], k[4, 0, 0] = 0.0, 1.7, math.nan, math.inf, -math.inf
    k[5] = torch.linspace(-1, 1, dim).to(t) * torch.finfo(t).max
    k[6] = torch.linspace(0, 1, dim).to(t) * torch.finfo(t).smallest_normal
    k[7] = torch.arange(dim) / 2 % 15.5
    k[8] = -(torch.arange(dim) / 4 % 15.25)
    k[9, 0, :] = -0.0
    k[10] = (torch.arange(dim) * 3 % 31) / 64 - 0.25
    v = k.flip(0)
    want = ref.Cache(raw, heads, dim, page)
    ref.append(want, table, ln, st, k, v)
    cache, dt, dl, ds = _cuda(raw, table, ln, st)
    lib.kv4_append(cache, dt, dl, ds, k.cuda(), v.cuda(), page)
    got = ref.Cache(cache.cpu(), heads, dim, page)
    assert torch.equal(got.k, want.k) and torch.equal(got.v, want.v)
    for a, b in ((got.kp, want.kp), (got.vp, want.vp)):
        assert torch.equal(torch.nan_to_num(a.float(), nan=7.5), torch.nan_to_num(b.float(), nan=7.5))
    gk, _ = lib.kv4_read(cache, dt, dl, ds, n, heads, dim, page)
    assert torch.isnan(gk[2:5]).all() and torch.isfinite(gk[[0, 1, 6, 7, 8, 9, 10, 11]]).all()


def test_append_what_has_no_place():
    """pages outside of the cache, positions before the sequence and behind its table or the rotation's, rows of no sequence"""
    heads, dim, page = 2, 64, 16
    raw, table, ln, st, _ = _setup(7, heads, dim, page, [40, 60, 3, 80, 20], [9, 20, 6, 40, 2])
    table[0, 2], table[1, 3], table[1, 2] = -1, raw.shape[0], 1 << 30
    ln[3] = 5000   # behind its table
    tokens = int(st[-1]) + 11
    g = _gen(8)
    k, v, q = (torch.randn((tokens, h, dim), generator=g).half() for h in (heads, heads, 4))
    for cos, sin in ((None, None), _tables(55, dim)):
        want, wq = ref.Cache(raw, heads, dim, page), torch.full_like(q, 3.0)
        ref.append(want, table, ln, st, k, v, cos, sin, False, q, wq)
        cache, dt, dl, ds = _cuda(raw, table, ln, st)
        gq = torch.full_like(q, 3.0).cuda()
        lib.kv4_append(cache, dt, dl, ds, k.cuda(), v.cuda(), page, q=q.cuda(), q_out=gq, cos=None if cos is None else cos.cuda(), sin=None if sin is None else sin.cuda())
        assert torch.equal(cache.cpu(), want.raw()) and torch.equal(gq.cpu(), wq)
        gk, gv = (torch.full((tokens, heads, dim), 3.0, device="cuda") for _ in range(2))
        lib.kv4_read(cache, dt, dl, ds, tokens, heads, dim, page, k=gk, v=gv)
        wk, wv = ref.read(want, table, ln, st, tokens, torch.float32)
        wk[int(st[-1]):] = wv[int(st[-1]):] = 3.0
        assert torch.equal(gk.cpu(), wk) and torch.equal(gv.cpu(), wv)


def test_append_of_strided_tensors():
    """keys, values and queries as slices of one projection's result"""
    heads, group, dim, page = 2, 3, 96, 32
    raw, table, ln, st, n = _setup(9, heads, dim, page, [50, 20], [30, 20])
    qkv = torch.randn((n, heads * (group + 2) * dim + 5), generator=_gen(10)).bfloat16()
    cut = lambda t, a, b: t[:, a * dim + 5:b * dim + 5].unflatten(1, (b - a, dim))
    parts = lambda t: (cut(t, 0, heads * group), cut(t, heads * group, heads * (group + 1)), cut(t, heads * (group + 1), heads * (group + 2)))
    q, k, v = parts(qkv)
    cos, sin = _tables(50, 48)
    want, wq = ref.Cache(raw, heads, dim, page), torch.empty(q.shape, dtype=q.dtype)
    ref.append(want, table, ln, st, k, v, cos, sin, True, q, wq)
    cache, dt, dl, ds, cos, sin = _cuda(raw, table, ln, st, cos, sin)
    q, k, v = parts(qkv.cuda())
    got = lib.kv4_append(cache, dt, dl, ds, k, v, page, q=q, cos=cos, sin=sin, neighbours=True)
    assert torch.equal(cache.cpu(), want.raw()) and torch.equal(got.cpu(), wq)


def _attend(seed, heads, group, dim, page, lens, new, dtype, calm=True, max_len=0, scale=None, change=None, tokens=None):
    raw, table, ln, st, tokens = _setup(seed, heads, dim, page, lens, new, calm=calm, tokens=tokens)
    if change:
        change(raw, table, ln, st)
    q = torch.randn((tokens, heads * group, dim), generator=_gen(seed + 1)).to(TYPES[dtype])
    want, slack = ref.attention(ref.Cache(raw, heads, dim, page), table, ln, st, q, scale)
    cache, dt, dl, ds = _cuda(raw, table, ln, st)
    out = torch.full(q.shape, 5.0, dtype=q.dtype, device="cuda")
    lib.kv4_attention(q.cuda(), cache, dt, dl, ds, heads, page, scale=scale, max_len=max_len, out=out)
    out, last = out.cpu().double(), int(st[-1])
    assert (out[last:] == 5).all()
    off = (out - want)[:last].abs()
    assert torch.isfinite(out[:last]).all()
    assert bool((off <= slack[:last]).all()), "off by up to %.3g of the allowed" % float((off / slack[:last].clamp_min(1e-30)).max())
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,group,dim,page,lens,new", [
    (1, 1, 64, 16, [1], [1]), (2, 4, 128, 64, [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257], [1] * 16),
    (1, 8, 96, 32, [100, 31], [1, 1]), (2, 2, 256, 16, [77, 300], [1, 1]), (1, 7, 128, 128, [500, 1, 130], [1, 1, 1]), (1, 20, 64, 32, [90, 40], [1, 1]),
    (2, 3, 64, 16, [40, 9, 100], [40, 1, 33]), (1, 1, 128, 64, [150], [150]), (4, 4, 128, 32, [70, 64, 31], [5, 64, 1]), (1, 16, 96, 16, [50], [17]),
    (2, 5, 256, 256, [280], [23]), (3, 2, 64, 64, [33, 0, 20, 65], [33, 0, 0, 2]), (1, 40, 64, 16, [60], [9]), (1, 4, 128, 16, [3] * 130, [1] * 130)])
def test_attention(heads, group, dim, page, lens, new, dtype):
    _attend(dim + page + len(lens), heads, group, dim, page, lens, new, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,group,dim,page,lens,new", [(32, 2, 64, 16, [700, 300, 200], [600, 300, 123]), (16, 4, 128, 64, [990, 64, 1], [900, 64, 1]),
                                                           (16, 5, 96, 32, [500, 420], [400, 419]), (8, 4, 256, 16, [1000, 70], [930, 70])])
def test_attention_of_many_rows(heads, group, dim, page, lens, new, dtype):
    """enough rows to fill the chip with wavefronts on all tokens each"""
    assert sum(new) * group // (64 if dim == 256 else 128) * heads >= 480
    _attend(dim, heads, group, dim, page, lens, new, dtype, tokens=sum(new) + 3)


def test_attention_of_many_rows_with_holes():
    """bad pages in the middle, at the end and for all of a sequence; garbage behind the sequences"""
    def change(raw, table, ln, st):
        raw[table[0, 9].item()] = 255   # NaN
        ln[0] = 575                     # in the page behind
        table[0, 3], table[0, 8], table[1, 0], table[2] = -1, raw.shape[0], 1 << 30, -5
    _attend(25, 16, 4, 128, 64, [640, 300, 200], [500, 300, 200], "bf16", change=change)


@pytest.mark.parametrize("max_len", [0, 1, 3000, 100000])
def test_attention_over_a_long_cache(max_len):
    """split over workgroups, whatever the hint says"""
    _attend(11, 2, 4, 128, 64, [3000, 40, 1], [1, 1, 1], "bf16", max_len=max_len)
    _attend(12, 1, 6, 64, 16, [2500], [3], "f16", max_len=max_len)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attention_does_not_look_behind_the_sequence(dtype):
    """random bytes, NaN and infinite scales and zeros among them, behind what was appended"""
    heads, dim, page = 2, 128, 32
    lens, new = [45, 1, 64], [45, 1, 64]

    def fill(raw, table, ln, st):
        g = _gen(14)
        k, v = (torch.randn((sum(new), heads, dim), generator=g).bfloat16() for _ in range(2))
        c = ref.Cache(raw, heads, dim, page)
        ref.append(c, table, ln, st, k, v)
        raw.copy_(c.raw())

    for max_len in (0, 5000):
        _attend(13, heads, 4, dim, page, lens, new, dtype, calm=False, change=fill, max_len=max_len)


def test_attention_of_rows_that_see_nothing():
    """more new tokens than a sequence holds, an empty one, bad pages, rows behind the last sequence"""
    def change(raw, table, ln, st):
        ln[0], ln[1], ln[3] = 3, 0, -7
        table[2, 0], table[2, 1] = -1, raw.shape[0]
        table[4, 0] = 1 << 30
    out = _attend(15, 2, 3, 64, 16, [20, 20, 30, 20, 40], [9, 4, 30, 5, 12], "bf16", change=change, tokens=70)
    assert (out[:6] == 0).all() and (out[9:13] == 0).all() and (out[13:43] == 0).all() and (out[43:48] == 0).all() and (out[6:9] != 0).any()


@pytest.mark.parametrize("scale", [1e-3, 0.5, 4.0])
def test_attention_with_a_scale(scale):
    """from weights that are all alike to one that takes all"""
    _attend(16, 1, 4, 128, 32, [300, 40], [1, 3], "f16", scale=scale)


def test_attention_with_not_a_number():
    """a token of NaN is seen by those behind it only"""
    heads, dim, page, n = 1, 64, 16, 30
    raw, table, ln, st, _ = _setup(17, heads, dim, page, [n], [n])
    cache, dt, dl, ds = _cuda(raw, table, ln, st)
    k, v, q = (torch.randn((n, 1, dim), generator=_gen(i)).bfloat16().cuda() for i in (1, 2, 3))
    for x in (k, v):
        bad = x.clone()
        bad[20, 0, 3] = math.nan
        lib.kv4_append(cache, dt, dl, ds, *((bad, v) if x is k else (k, bad)), page)
        out = lib.kv4_attention(q, cache, dt, dl, ds, 1, page)
        assert torch.isnan(out[20:]).all() and torch.isfinite(out[:20]).all()


def test_attention_of_strided_queries_and_a_wide_table():
    heads, group, dim, page = 2, 2, 64, 16
    raw, table, ln, st, n = _setup(18, heads, dim, page, [50, 33], [4, 1])
    wide = torch.full((2, 9), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    q = torch.randn((n, 4 * dim + 8), generator=_gen(19)).bfloat16()
    cache, dt, dl, ds, dw, dq = _cuda(raw, table, ln, st, wide, q)
    a = lib.kv4_attention(dq[:, 4:4 + 4 * dim].unflatten(1, (4, dim)), cache, dt, dl, ds, heads, page)
    b = lib.kv4_attention(dq[:, 4:4 + 4 * dim].unflatten(1, (4, dim)).contiguous(), cache, dw, dl, ds, heads, page, max_len=50)
    c = lib.kv4_attention(dq[:, 4:4 + 4 * dim].unflatten(1, (4, dim)), cache, dw[:, :table.shape[1]], dl, ds, heads, page)
    want, slack = ref.attention(ref.Cache(raw, heads, dim, page), table, ln, st, q[:, 4:4 + 4 * dim].unflatten(1, (4, dim)))
    for out in (a, b, c):
        assert bool(((out.cpu().double() - want).abs() <= slack).all())


def test_page_far_into_the_cache():
    """a page that begins behind 4 GiB"""
    heads, dim, page = 8, 256, 256
    nb = lib.kv4_page_bytes(heads, dim, page)
    pages = (1 << 32) // nb + 3
    cache = torch.zeros((pages, nb), dtype=torch.uint8, device="cuda")
    table = torch.tensor([[pages - 1]], dtype=torch.int32)
    ln, st = torch.tensor([10], dtype=torch.int32), torch.tensor([0, 10], dtype=torch.int32)
    k, v, q = (torch.randn((10, heads, dim), generator=_gen(i)).bfloat16() for i in (4, 5, 6))
    args = [cache] + _cuda(table, ln, st)
    lib.kv4_append(*args, k.cuda(), v.cuda(), page)
    small = ref.Cache(torch.zeros((1, nb), dtype=torch.uint8), heads, dim, page)
    ref.append(small, table * 0, ln, st, k, v)
    assert torch.equal(cache[-1].cpu(), small.raw()[0]) and not cache[:-1].any()
    out = lib.kv4_attention(q.cuda(), *args, heads, page)
    want, slack = ref.attention(small, table * 0, ln, st, q)
    assert bool(((out.cpu().double() - want).abs() <= slack).all())


def test_a_block_of_a_model_step_by_step():
    """projection in 8 bits, append, attention, projection back with ternary weights: eager, and captured and replayed with the lengths
    moved on by the graph's own work"""
    hidden, heads, group, dim, page, batch = 192, 2, 2, 64, 16, 3
    g = _gen(20)
    w_in = lib.quantize_rows_i8(torch.randn((heads * (group + 2) * dim, hidden), generator=g).cuda())
    lanes = ref.lanes(hidden, heads * group * dim, True, g)
    w_out = lib.pack_weights(lanes.float().view(*lanes.shape, 1, 1).cuda(), torch.full((hidden,), 0.5, device="cuda"), True)
    s_out = (torch.rand(hidden, generator=g) * 0.01).cuda()
    raw, table, ln, _, _ = _setup(21, heads, dim, page, [60, 60, 60], [1, 1, 1])
    table = table.cuda()
    cos, sin = _cuda(*_tables(60, dim))
    starts = torch.arange(batch + 1, dtype=torch.int32).cuda()
    x = torch.randn((batch, hidden), generator=g).bfloat16().cuda()
    first = torch.tensor([7, 1, 30], dtype=torch.int32).cuda()

    def step(cache, lens):
        q8, s8 = lib.quantize_rows_i8(x)
        qkv = lib.mm_i8(q8, s8, *w_in, hidden, dtype=torch.bfloat16).view(batch, heads * (group + 2), dim)
        k, v = qkv[:, heads * group:heads * (group + 1)], qkv[:, heads * (group + 1):]
        q = lib.kv4_append(cache, table, lens, starts, k, v, page, q=qkv[:, :heads * group], cos=cos, sin=sin)
        o = lib.kv4_attention(q, cache, table, lens, starts, heads, page)
        o8, os = lib.quantize_rows_i8(o.view(batch, -1))
        return qkv, q, o, o8, os, lib.mm_i8_rows(o8, os, w_out, s_out, hidden, heads * group * dim, True, dtype=torch.bfloat16)

    cache, lens = raw.cuda(), first.clone()
    oracle = ref.Cache(raw, heads, dim, page)
    results = []
    for i in range(4):
        qkv, q, o, o8, os, y = (t.cpu() for t in step(cache, lens))
        hl, hs = lens.cpu(), starts.cpu()
        wq = torch.empty_like(q)
        ref.append(oracle, table.cpu(), hl, hs, qkv[:, heads * group:heads * (group + 1)], qkv[:, heads * (group + 1):], cos.cpu(), sin.cpu(), False,
                   qkv[:, :heads * group], wq)
        assert torch.equal(cache.cpu(), oracle.raw()) and torch.equal(q, wq)
        want, slack = ref.attention(oracle, table.cpu(), hl, hs, q)
        assert bool(((o.double() - want).abs() <= slack).all())
        want, slack = ref.product(o8, os, lanes, s_out.cpu(), None, torch.bfloat16)
        assert bool(((y.double() - want).abs() <= slack).all())
        results.append(y)
        lens += 1

    cache, lens = raw.cuda(), first.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache.clone(), lens.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(cache, lens)[-1]
        lens += 1
    cache.copy_(raw), lens.copy_(first)
    for want in results:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.cpu(), want)
        (x * 2).sum()   # eager work between the replays
    assert torch.equal(cache.cpu(), oracle.raw())


def test_refusals():
    raw, table, ln, st, n = _setup(22, 2, 64, 16, [20, 20], [2, 2])
    cache, table, ln, st = _cuda(raw, table, ln, st)
    k = torch.zeros((n, 2, 64), device="cuda").bfloat16()
    q = torch.zeros((n, 4, 64), device="cuda").bfloat16()
    a = (cache, table, ln, st)
    for bad, text in ((lambda: lib.kv4_append(*a, k, k[:3], 16), "expected 4 tokens"), (lambda: lib.kv4_append(*a, k, q, 16), "heads"),
                      (lambda: lib.kv4_append(*a, k, k.half(), 16), "bfloat16"), (lambda: lib.kv4_append(*a, k, k, 32), "pages of"),
                      (lambda: lib.kv4_append(*a, k, k, 24), "24 tokens"), (lambda: lib.kv4_append(cache, table, ln[:1], st, k, k, 16), "lens"),
                      (lambda: lib.kv4_append(cache, table.long(), ln, st, k, k, 16), "int32"), (lambda: lib.kv4_append(*a, k, k, 16, cos=torch.zeros((4, 32), device="cuda")), "together"),
                      (lambda: lib.kv4_append(*a, k, k, 16, q_out=q), "without q"), (lambda: lib.kv4_append(*a, k.cpu(), k, 16), "current GPU"),
                      (lambda: lib.kv4_append(*a, k.transpose(1, 2).contiguous().transpose(1, 2), k, 16), "contiguous"),
                      (lambda: lib.kv4_attention(q[:, :3], *a, 2, 16), "query heads"), (lambda: lib.kv4_attention(q.float(), *a, 2, 16), "FTNN_F16"),
                      (lambda: lib.kv4_attention(q, *a, 2, 16, scale=0.0), "scale"), (lambda: lib.kv4_attention(q, *a, 2, 16, scale=math.inf), "scale"),
                      (lambda: lib.kv4_attention(q, *a, 2, 16, max_len=-1), "max_len"), (lambda: lib.kv4_attention(q, *a, 2, 16, out=q[:, :2]), "shape"),
                      (lambda: lib.kv4_attention(q[..., :32], *a, 2, 16), "32 channels"), (lambda: lib.kv4_read(*a, n, 0, 64, 16), "heads")):
        with pytest.raises(lib.FtnnError, match=text):
            bad()
    assert torch.equal(cache.cpu(), raw)
    none = lib.kv4_attention(q[:0], *a, 2, 16)
    assert none.shape == (0, 4, 64)


def test_both_ways_into_the_library(monkeypatch):
    """the calls through csrc/py_call.cpp give what those through ctypes give, take what they are given, and leave the rest to ctypes"""
    heads, group, dim, page = 2, 2, 64, 16
    raw, table, ln, st, n = _setup(30, heads, dim, page, [50, 33], [4, 9])
    cos, sin, dt, dl, ds = _cuda(*_tables(50, 32), table, ln, st)
    g = _gen(31)
    k, v, q = (torch.randn((n, h, dim), generator=g).bfloat16().cuda() for h in (heads, heads, heads * group))
    x, w, bias = torch.randn((7, 100), generator=g).cuda(), torch.randn((200, 100), generator=g).cuda(), torch.randn(200, generator=g).cuda()
    lanes = lib.pack_weights(torch.randint(-1, 2, (200, 100, 1, 1), generator=g).float().cuda(), torch.full((200,), 0.5, device="cuda"), True)
    scratch = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")

    def calls(yes=True):   # yes: 1 where the plain form is left
        out = []
        c = raw.cuda()
        out += [*lib.quantize_rows_i8(x)]
        b = lib.quantize_rows_i8(w)
        out += [lib.mm_i8(*out[:2], *b, 100), lib.mm_i8(*out[:2], *b, 100, bias=bias, dtype=torch.bfloat16), lib.mm_i8(*out[:2], *b, 100, out=torch.empty((7, 200), device="cuda").half())]
        out += [lib.mm_i8_rows(*out[:2], lanes, b[1], 200, 100, yes), lib.mm_i8_rows(*out[:2], lanes, b[1], 200, 100, yes, bias=bias, dtype=torch.float16, scratch=scratch)]
        lib.kv4_append(c, dt, dl, ds, k, v, page)
        out += [c.clone(), lib.kv4_append(c, dt, dl, ds, k, v, page, q=q, cos=cos, sin=sin, neighbours=yes), c]
        out += [*lib.kv4_read(c, dt, dl, ds, n, heads, dim, page, dtype=torch.float16), lib.kv4_attention(q, c, dt, dl, ds, heads, page),
                lib.kv4_attention(q, c, dt, dl, ds, heads, page, scale=0.2, max_len=9000, out=torch.empty_like(q), scratch=scratch)]
        return out

    native, answered = lib._native(), []

    class Spy:
        def __getattr__(self, name):
            def fn(*args):
                r = getattr(native, name)(*args)
                answered.append(r is not None)
                return r
            return fn

    monkeypatch.setattr(lib, "_call", Spy())
    fast = calls()
    assert len(answered) == 12 and all(answered)
    same = lambda a, b: all(torch.equal(s, t) and s.dtype == t.dtype for s, t in zip(a, b))
    assert same(fast, calls(1))
    monkeypatch.setattr(lib, "_call", lib._ThroughCtypes())
    assert same(fast, calls())
