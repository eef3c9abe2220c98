"""Tensors at the edge of what the calls of token models take: single rows out of wider ones, tensors without storage."""
import pytest

torch = pytest.importorskip("torch")
import fastertnn_amd.lib as lib

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["module", "ctypes"])
def way(request, monkeypatch):
    monkeypatch.setattr(lib, "_call", lib._native() if request.param == "module" else lib._ThroughCtypes())


def test_a_single_row_of_any_width(way):
    """the distance between rows of one row is not looked at"""
    k = 100
    x = torch.randn((3, k), generator=torch.Generator().manual_seed(1)).cuda()
    q, s = lib.quantize_rows_i8(x)
    w, ws = lib.quantize_rows_i8(torch.randn((40, k), generator=torch.Generator().manual_seed(2)).cuda())
    wide = torch.zeros((3, 128), dtype=torch.int8, device="cuda")
    wide[:, :112] = q
    ww = torch.zeros((40, 128), dtype=torch.int8, device="cuda")
    ww[:, :112] = w
    want = lib.mm_i8(q, s, w, ws, k)
    for m in (1, 3):
        assert torch.equal(lib.mm_i8(wide[:m, :120], s[:m], w, ws, k), want[:m])
        assert torch.equal(lib.mm_i8(q, s, ww[:m, :117], ws[:m], k), want[:, :m])
        got, scale = lib.quantize_rows_i8(x[:m], q=torch.zeros((m, 128), dtype=torch.int8, device="cuda")[:, :120])
        assert torch.equal(got[:, :112], q[:m]) and torch.equal(scale, s[:m])
    lanes = lib.pack_weights(torch.ones((40, k, 1, 1), device="cuda"), torch.full((40,), 0.5, device="cuda"), True)
    rows = lib.mm_i8_rows(q, s, lanes, ws, 40, k, True)
    assert torch.equal(lib.mm_i8_rows(wide[:1, :120], s[:1], lanes, ws, 40, k, True), rows[:1])


def test_tensors_without_storage(way):
    """what a call sees under vmap has sizes and strides, and no data: an error, whichever tensor it is"""
    g = torch.Generator().manual_seed(3)
    x = torch.randn((2, 4, 64), generator=g).cuda()
    w, ws = lib.quantize_rows_i8(torch.randn((8, 64), generator=g).cuda())
    q, s = lib.quantize_rows_i8(x[0])
    lanes = lib.pack_weights(torch.ones((8, 64, 1, 1), device="cuda"), torch.full((8,), 0.5, device="cuda"), True)
    heads, dim, page = 2, 64, 16
    cache = torch.zeros((2, lib.kv4_page_bytes(heads, dim, page)), dtype=torch.uint8, device="cuda")
    table, lens, starts = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([[0]], [4], [0, 4]))
    k, many = torch.zeros((4, heads, dim), dtype=torch.bfloat16, device="cuda"), torch.zeros((2, 4, heads, dim), dtype=torch.bfloat16, device="cuda")
    two = lambda t: torch.stack([t, t])
    held = (table, lens, starts)
    calls = [(lib.quantize_rows_i8, x), (lambda t: lib.mm_i8(t, s, w, ws, 64), two(q)), (lambda t: lib.mm_i8(q, s, t, ws, 64), two(w)), (lambda t: lib.mm_i8(q, t, w, ws, 64), two(s)),
             (lambda t: lib.mm_i8(q, s, w, ws, 64, out=t), torch.zeros((2, 4, 8), device="cuda")), (lambda t: lib.mm_i8_rows(t, s, lanes, ws, 8, 64, True), two(q)),
             (lambda t: lib.mm_i8_rows(q, s, t, ws, 8, 64, True), two(lanes)), (lambda t: lib.kv4_append(cache, *held, t, k, page), many), (lambda t: lib.kv4_append(cache, *held, k, t, page), many),
             (lambda t: lib.kv4_append(cache, *held, k, k, page, q=t), many), (lambda t: lib.kv4_read(t, *held, 4, heads, dim, page, dtype=torch.float16), two(cache)),
             (lambda t: lib.kv4_attention(t, cache, *held, heads, page), many), (lambda t: lib.kv4_attention(k, t, *held, heads, page), two(cache))]
    for fn, t in calls:
        with pytest.raises((lib.FtnnError, RuntimeError)):
            torch.vmap(fn)(t)
    assert torch.equal(lib.quantize_rows_i8(x[0])[0], q)
    torch.cuda.synchronize()
