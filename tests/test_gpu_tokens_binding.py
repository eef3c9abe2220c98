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
