"""Rows of 8-bit codes and their products, against 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")
import fastertnn_amd.lib as lib
from tests import i8_shapes
from tests import tokens_oracle as ref

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _rand(seed, shape, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _same_codes(x, q, scale):
    want, ws = ref.quantize_rows(x)
    k = x.shape[1]
    assert torch.equal(q[:, :k].cpu().long(), want)
    assert not q[:, k:lib.i8_row_bytes(k)].any()
    assert torch.equal(torch.nan_to_num(scale.cpu(), nan=-1.0), torch.nan_to_num(ws, nan=-1.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 15), (1, 16), (5, 17), (2, 100), (70, 257), (7, 512), (5, 520), (4, 1024), (6, 1040), (13, 2048), (3, 2049), (9, 4100), (2, 16384), (1, 16387), (3, 40001)])
def test_codes_of_rows(dtype, rows, k):
    x = _rand(rows * 1000 + k, (rows, k), TYPES[dtype])
    _same_codes(x, *lib.quantize_rows_i8(x.cuda()))


@pytest.mark.parametrize("dtype", TYPES)
def test_codes_next_to_borders(dtype):
    """quotients at and next to halves: x = (2 i + 1) / 254 of the maximum, and the neighbours of it in the type"""
    t = TYPES[dtype]
    rows = []
    for top in (1.0, 127.0, 254.0, 0.8515625, 100.0, 1.9921875):
        base = torch.tensor([top * (2 * i + 1) / 254 for i in range(127)], dtype=torch.float64).to(t)
        bits = base.view(torch.int32 if t is torch.float32 else torch.int16)
        rows.append(torch.cat([(bits + d).view(t) for d in (-2, -1, 0, 1, 2)] + [torch.tensor([top], dtype=t)]).clamp(-top, top))
    x = torch.stack(rows)
    _same_codes(x, *lib.quantize_rows_i8(x.cuda()))
    _same_codes(-x, *lib.quantize_rows_i8((-x).cuda()))


@pytest.mark.parametrize("dtype", TYPES)
def test_codes_of_special_rows(dtype):
    t = TYPES[dtype]
    tiny = torch.finfo(t).smallest_normal
    x = torch.zeros((9, 77), dtype=t)
    x[1, 5] = math.nan
    x[2, 76] = math.inf
    x[3, 0] = -math.inf
    x[4] = _rand(1, (77,)).to(t) * tiny            # at the edge of subnormal numbers
    x[5, 3] = torch.finfo(t).smallest_normal * 2.0 ** -7
    x[6] = torch.linspace(-1, 1, 77).to(t) * torch.finfo(t).max
    x[7] = 1.0
    x[8] = -0.0
    q, s = lib.quantize_rows_i8(x.cuda())
    _same_codes(x, q, s)
    assert not q[:4].any() and torch.isnan(s[1:4]).all() and s[0] == 0 and s[8] == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_codes_of_strided_rows_into_given_tensors(dtype):
    x = _rand(3, (7, 301), TYPES[dtype]).cuda()[:, 3:204]
    q = torch.full((7, 240), 99, dtype=torch.int8, device="cuda")
    got, s = lib.quantize_rows_i8(x, q=q[:, :208], scale=torch.empty(7, device="cuda"))
    _same_codes(x.cpu(), got, s)
    assert (q[:, 208:] == 99).all()
    wide = torch.full((7, 256), 99, dtype=torch.int8, device="cuda")
    lib.quantize_rows_i8(x, q=wide)
    assert (wide[:, 208:] == 99).all() and not wide[:, 201:208].any()
    empty, s = lib.quantize_rows_i8(x[:0])
    assert empty.shape == (0, 208) and s.shape == (0,)
    one = x[:1].expand(4, 201)   # the same row again and again
    _same_codes(one.cpu(), *lib.quantize_rows_i8(one))


def _codes(seed, rows, k, full=False):
    g = torch.Generator().manual_seed(seed)
    q = torch.zeros((rows, lib.i8_row_bytes(k)), dtype=torch.int8)
    q[:, :k] = torch.randint(-128, 128, (rows, k), generator=g).to(torch.int8)
    if full:
        q[:, :k] = -128
    return q, torch.rand(rows, generator=g) * 0.1 + 0.01


def _check_product(y, a, sa, b, sb, bias, k):
    want, slack = ref.product(a[:, :k], sa, b[:, :k], sb, bias, y.dtype)
    off = (y.cpu().double() - want).abs()
    assert bool((off <= slack).all()), "off by up to %.3g of the allowed" % float((off / slack).max())


SIZES = [(1, 1, 1), (1, 16, 16), (1, 17, 33), (2, 100, 64), (7, 64, 65), (15, 33, 127), (16, 256, 1000), (17, 31, 513), (33, 130, 129), (64, 64, 4096),
         (1, 4099, 1500), (65, 200, 320), (100, 300, 700), (128, 128, 128), (129, 257, 1025), (300, 520, 260), (1, 130, 20000), (512, 33, 64), (1000, 257, 144)]


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product_of_codes(m, n, k, bias):
    a, sa = _codes(m + n + k, m, k)
    b, sb = _codes(m * n + k, n, k)
    bb = _rand(k, (n,)) if bias else None
    for t in TYPES.values():
        y = lib.mm_i8(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), k, bias=None if bb is None else bb.cuda(), dtype=t)
        assert y.dtype == t
        _check_product(y, a, sa, b, sb, bb, k)


def test_product_of_the_largest_sums():
    """131071 products of -128 * -128: the largest sum that 32 bits hold"""
    k = 131071
    for m, n in ((1, 3), (40, 18), (130, 140)):
        a, sa = _codes(1, m, k, full=True)
        b, sb = _codes(2, n, k, full=True)
        y = lib.mm_i8(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), k)
        _check_product(y, a, sa, b, sb, None, k)


@pytest.mark.parametrize("m,n,k", [(m, n, k) for (m, n), ks in i8_shapes.TILES.values() for k in ks] + [(*s, k) for s in i8_shapes.FEW_CODES.values() for k in (16, 1025, 3000)])
def test_product_of_codes_in_each_form(m, n, k):
    a, sa = _codes(m + n + k, m, k)
    b, sb = _codes(m * n + k, n, k)
    bias = _rand(k, (n,))
    for t, bb in ((torch.float32, bias), (torch.bfloat16, None)):
        y = lib.mm_i8(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), k, bias=None if bb is None else bb.cuda(), dtype=t)
        _check_product(y, a, sa, b, sb, bb, k)


@pytest.mark.parametrize("m", [3, 40, 200])
def test_product_with_strides(m):
    """rows apart, a result inside of a larger tensor, and bytes behind the K-th code of one operand that are not zero"""
    k, n = 200, 77
    a, sa = _codes(5, m, k)
    b, sb = _codes(6, n, k)
    wide_a = torch.full((m, 256), 77, dtype=torch.int8)
    wide_a[:, :208] = a
    wide_b = torch.full((n, 320), 55, dtype=torch.int8)
    wide_b[:, :k] = b[:, :k]
    y = torch.full((m, 101), 7.0, dtype=torch.bfloat16, device="cuda")
    lib.mm_i8(wide_a.cuda(), sa.cuda(), wide_b.cuda()[:, :240], sb.cuda(), k, out=y[:, 13:13 + n])
    _check_product(y[:, 13:13 + n], a, sa, b, sb, None, k)
    assert (y[:, :13] == 7).all() and (y[:, 13 + n:] == 7).all()
    assert lib.mm_i8(a[:0].cuda(), sa[:0].cuda(), b.cuda(), sb.cuda(), k).shape == (0, n)


def _packed(lanes, ternary):
    w = lanes.float().view(*lanes.shape, 1, 1).cuda()
    return lib.pack_weights(w, torch.full((lanes.shape[0],), 0.5 if ternary else 0.0, device="cuda"), ternary)


@pytest.mark.parametrize("ternary", [True, False])
@pytest.mark.parametrize("m,n,k", SIZES + [(1, 64, 256), (5, 48, 512), (2, 20, 255), (3, 20, 257), (16, 1000, 2049)])
def test_product_with_packed_rows(m, n, k, ternary):
    a, sa = _codes(m + n + k, m, k)
    w = ref.lanes(n, k, ternary, torch.Generator().manual_seed(n * k))
    sb, bias = torch.rand(n) * 0.1 + 0.01, _rand(n, (n,))
    rows = _packed(w, ternary)
    for t, bb in ((torch.float32, None), (torch.bfloat16, bias), (torch.float16, bias)):
        y = lib.mm_i8_rows(a.cuda(), sa.cuda(), rows, sb.cuda(), n, k, ternary, bias=None if bb is None else bb.cuda(), dtype=t)
        _check_product(y, a, sa, w, sb, bb, k)


@pytest.mark.parametrize("ternary", [True, False])
@pytest.mark.parametrize("m,n,k", [(m, n, ks[-1]) for (m, n), ks in i8_shapes.TILES.values()] + [(*s, k) for s in i8_shapes.FEW_PACKED.values() for k in (16, 1025, 5000)])
def test_product_with_packed_rows_in_each_form(m, n, k, ternary):
    a, sa = _codes(m + n + k, m, k)
    w = ref.lanes(n, k, ternary, torch.Generator().manual_seed(n * k))
    sb = torch.rand(n) * 0.1 + 0.01
    y = lib.mm_i8_rows(a.cuda(), sa.cuda(), _packed(w, ternary), sb.cuda(), n, k, ternary)
    _check_product(y, a, sa, w, sb, None, k)


def test_product_of_rows_far_apart():
    """strides beyond what tiles take"""
    k, m, n = 100, 90, 9000
    a, sa = _codes(1, m, k)
    b, sb = _codes(2, n, k)
    far = torch.zeros((m, 9 << 20), dtype=torch.int8, device="cuda")
    far[:, :112] = a.cuda()
    _check_product(lib.mm_i8(far, sa.cuda(), b.cuda(), sb.cuda(), k), a, sa, b, sb, None, k)


@pytest.mark.parametrize("m", [2, 300])
def test_product_with_rows_of_the_gemm_packer(m):
    a, sa = _codes(8, m, 512)
    w = ref.lanes(70, 512, True, torch.Generator().manual_seed(8))
    sb = torch.rand(70) + 0.1
    rows = lib.pack_gemm_operand(w.float().cuda())
    need = lib.mm_i8_rows_scratch_bytes(True, m, 70, 512)
    y = lib.mm_i8_rows(a.cuda(), sa.cuda(), rows, sb.cuda(), 70, 512, True, scratch=torch.empty(need + 16, dtype=torch.uint8, device="cuda"))
    _check_product(y, a, sa, w, sb, None, 512)


def test_not_a_number_goes_through():
    """a row whose scale is NaN gives NaN, and no other row does"""
    x = _rand(9, (5, 64))
    x[2, 7] = math.inf
    w = _rand(10, (33, 64))
    q, s = lib.quantize_rows_i8(x.cuda())
    y = lib.mm_i8(q, s, *lib.quantize_rows_i8(w.cuda()), 64)
    assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3, 4]]).all()


def test_on_streams_and_in_graphs():
    """a captured pair of calls, replayed on new inputs, and the same calls on another stream"""
    x = _rand(11, (20, 300), torch.bfloat16).cuda()
    w = _rand(12, (90, 300)).cuda()
    b, sb = lib.quantize_rows_i8(w)

    def step():
        q, s = lib.quantize_rows_i8(x)
        return lib.mm_i8(q, s, b, sb, 300, dtype=torch.bfloat16)

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, step())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step()
    for i in range(3):
        x.copy_(_rand(20 + i, (20, 300), torch.bfloat16))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, step())


def test_two_graphs_of_packed_products():
    """tiles behind the launch that unpacks: two captured calls with a workspace of their own each, replayed in turn and on two streams"""
    (m, n), ks = i8_shapes.TILES["T128Two"]
    k = ks[-1]
    assert lib.mm_i8_rows_scratch_bytes(True, m, n, k) > 0
    q, s = lib.quantize_rows_i8(_rand(13, (m, k), torch.bfloat16).cuda())
    sets = []
    for i in range(2):
        w = torch.randint(-1, 2, (n, k, 1, 1), generator=torch.Generator().manual_seed(40 + i)).float().cuda()
        sets.append((lib.pack_weights(w, torch.full((n,), 0.5, device="cuda"), True), torch.full((n,), 0.5 + i, device="cuda")))
    want = [lib.mm_i8_rows(q, s, rows, scale, n, k, True) for rows, scale in sets]
    assert not torch.equal(want[0], want[1])
    graphs, got = [], []
    for rows, scale in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(lib.mm_i8_rows(q, s, rows, scale, n, k, True))
        graphs.append(g)
    sides = [torch.cuda.Stream() for _ in graphs]
    for i in range(4):
        for y in got:
            y.zero_()
        torch.cuda.synchronize()
        for g, side in zip(graphs, sides):
            with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_more_rows_than_a_launch_holds():
    rows = (1 << 23) + 3
    x = torch.randn((rows, 16), dtype=torch.bfloat16, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    q, s = lib.quantize_rows_i8(x)
    at = torch.tensor([0, 1, (1 << 23) - 1, 1 << 23, rows - 1], device="cuda")
    _same_codes(x[at].cpu(), q[at], s[at])
    most = x.float().abs().amax(1).cpu().double()
    assert torch.equal(s.cpu(), (most / 127).float())   # (a quotient of 24 bits by 7 is no tie in 53)


def test_refusals():
    q, s = (t.cuda() for t in _codes(1, 4, 64))
    w, ws = (t.cuda() for t in _codes(2, 8, 64))
    for bad, text in ((lambda: lib.mm_i8(q.cpu(), s, w, ws, 64), "current GPU"), (lambda: lib.mm_i8(q, s[:3], w, ws, 64), "shape"),
                      (lambda: lib.mm_i8(q, s, w, ws, 80), "rows of 64 codes"), (lambda: lib.mm_i8(q.float(), s, w, ws, 64), "int8"),
                      (lambda: lib.mm_i8(q, s.double(), w, ws, 64), "float32"), (lambda: lib.mm_i8(q, s, w, ws, 64, dtype=torch.int8), "bfloat16"),
                      (lambda: lib.mm_i8(q[:, 1:49], s, w, ws, 48), "16-byte"), (lambda: lib.mm_i8(q.t().contiguous().t(), s, w, ws, 64), "contiguous"),
                      (lambda: lib.mm_i8(q, s, w, ws, 64, out=torch.empty((4, 9), device="cuda")), "shape"),
                      (lambda: lib.mm_i8(q, s, w, ws, 0), "rows of 0"), (lambda: lib.quantize_rows_i8(q), "float32"),
                      (lambda: lib.quantize_rows_i8(s), "dimensions"), (lambda: lib.quantize_rows_i8(ws.view(1, 8).expand(2, 8), q=q), "rows of at least"),
                      (lambda: lib.mm_i8_rows(q, s, torch.zeros(8, dtype=torch.int64, device="cuda"), ws, 8, 64, True), "packed rows")):
        with pytest.raises(lib.FtnnError, match=text):
            bad()
