"""The entry points of token models in few bits without a GPU: sizes, and what is refused before any device work."""
import ctypes as C

import pytest

import fastertnn_amd.lib as lib

L = lib._L
BUF = (C.c_char * 8192)()
P = (C.addressof(BUF) + 255) & ~255


def test_sizes():
    assert [lib.i8_row_bytes(k) for k in (1, 15, 16, 17, 131071)] == [16, 16, 16, 32, 131072]
    assert lib.kv4_page_bytes(1, 64, 16) == 16 * 72 and lib.kv4_page_bytes(8, 128, 64) == 8 * 64 * 136
    for bad in ((0, 64, 16), (1, 80, 16), (1, 64, 8), (1, 64, 48), (1, 64, 512), (-1, 64, 16)):
        with pytest.raises(lib.FtnnError):
            lib.kv4_page_bytes(*bad)
    assert lib.mm_i8_rows_scratch_bytes(True, 0, 5, 5) == 0 and lib.mm_i8_rows_scratch_bytes(True, 1, 4096, 4096) == 0


def refused(rc, text):
    return rc == -1 and text in L.ftnn_last_error()


def test_quantize_rows():
    f = L.ftnn_quantize_rows_i8
    assert refused(f(3, P, 64, 2, 64, P, 64, P, None), b"element type")
    assert refused(f(0, P, 64, -1, 64, P, 64, P, None), b"-1 rows")
    assert refused(f(0, P, 64, 2, 0, P, 64, P, None), b"0 values")
    assert refused(f(0, None, 64, 2, 64, P, 64, P, None), b"null")
    assert refused(f(0, P, 64, 2, 64, P + 8, 64, P, None), b"aligned")
    assert refused(f(1, P + 1, 64, 2, 64, P, 64, P, None), b"aligned")
    assert refused(f(0, P, 64, 2, 65, P, 64, P, None), b"80 at least")
    assert refused(f(0, P, 64, 2, 60, P, 72, P, None), b"multiple of 16")
    assert refused(f(0, P, -64, 2, 60, P, 64, P, None), b"stride")
    assert f(0, None, 64, 0, 64, None, 64, None, None) == 0   # no rows: nothing to do


def test_products():
    f = L.ftnn_mm_i8
    ok = dict(dtype=0, a=P, a_stride=64, sa=P, b=P, b_stride=64, sb=P, bias=None, m=2, n=3, k=64, y=P, y_stride=3)
    call = lambda **kw: f(*{**ok, **kw}.values(), None)
    for change, text in (({"dtype": -1}, b"element type"), ({"m": -1}, b"dimension"), ({"n": 0}, b"dimension"), ({"k": 0}, b"dimension"),
                         ({"k": 131072, "a_stride": 131072, "b_stride": 131072}, b"32-bit sums"), ({"a": None}, b"null"), ({"sb": None}, b"null"), ({"y": None}, b"null"),
                         ({"a": P + 4}, b"16-byte"), ({"b": P + 1}, b"16-byte"), ({"bias": P + 2}, b"aligned"), ({"y": P + 2}, b"aligned"),
                         ({"a_stride": 48}, b"64 at least"), ({"b_stride": 72}, b"multiple of 16"), ({"y_stride": 2}, b"overlap"),
                         ({"m": 1 << 31}, b"2^31"), ({"m": 1 << 20, "n": 1 << 20, "y_stride": 1 << 20}, b"2^40")):
        assert refused(call(**change), text), change
    assert call(m=0) == 0
    g = L.ftnn_mm_i8_rows
    rows = lambda **kw: g(*{**dict(ternary=1, dtype=0, a=P, a_stride=64, sa=P, b=P, sb=P, bias=None, m=2, n=3, k=64, y=P, y_stride=3, scratch=None, bytes=0), **kw}.values(), None)
    assert refused(rows(b=P + 8), b"16-byte") and refused(rows(k=65), b"80 at least") and refused(rows(n=0), b"dimension")
    need = lib.mm_i8_rows_scratch_bytes(True, 4096, 512, 512)
    if need:
        big = dict(m=4096, n=512, k=512, a_stride=512, y_stride=512)
        assert refused(rows(**big), b"scratch") and refused(rows(**big, scratch=P, bytes=need - 1), b"scratch") and refused(rows(**big, scratch=P + 8, bytes=need), b"scratch")


def _kv(**kw):
    d = lib.Kv4Desc(P, 4, 2, 64, 16, 2, 3, 2, 2, P, P, P)
    for k, v in kw.items():
        setattr(d, k, v)
    return C.byref(d)


BAD = [({"dim": 80}, b"dim 80"), ({"page": 24}, b"page 24"), ({"heads": 0}, b"heads 0"), ({"heads": 40000}, b"heads"), ({"pages": 0}, b"dimension"), ({"tokens": -1}, b"dimension"),
       ({"width": 0}, b"dimension"), ({"table_stride": 1}, b"overlap"), ({"d_cache": None}, b"null"), ({"d_lens": None}, b"null"), ({"d_starts": None}, b"null"),
       ({"d_cache": P + 8}, b"16-byte"), ({"d_table": P + 2}, b"aligned")]


def test_cache():
    append = lambda kv, dtype=2, k=P, v=P, cos=None, sin=None, positions=0, rot=0, heads_q=0, q=None, q_out=None: L.ftnn_kv4_append(
        kv, dtype, k, 128, 64, v, 128, 64, cos, sin, positions, rot, 0, heads_q, q, 256, 64, q_out, None)
    read = lambda kv, dtype=2, k=P, v=P: L.ftnn_kv4_read(kv, dtype, k, v, None)
    for change, text in BAD:
        assert refused(append(_kv(**change)), text) and refused(read(_kv(**change)), text), change
    assert refused(append(None), b"null") and refused(append(_kv(), dtype=5), b"element type") and refused(append(_kv(), k=None), b"null")
    assert refused(append(_kv(), rot=3), b"rotation") and refused(append(_kv(), rot=66), b"rotation") and refused(append(_kv(), rot=-2), b"rotation")
    assert refused(append(_kv(), rot=4, positions=7, cos=P), b"tables") and refused(append(_kv(), heads_q=4), b"null") and refused(append(_kv(), heads_q=-1), b"query heads")
    assert refused(append(_kv(), v=P + 1), b"aligned") and refused(read(_kv(), k=P + 1), b"aligned")
    assert append(_kv(tokens=0), k=None, v=None) == 0 and append(_kv(sequences=0, d_lens=None)) == 0
    assert read(_kv(tokens=0)) == 0 and read(_kv(), k=None, v=None) == 0


def test_attention():
    attend = lambda kv, dtype=2, heads_q=4, q=P, scale=1.0, max_len=0, out=P, scratch=P, n=1 << 20: L.ftnn_kv4_attention(
        kv, dtype, heads_q, q, 256, 64, scale, max_len, out, scratch, n, None)
    for change, text in BAD:
        assert refused(attend(_kv(**change)), text), change
    for kw, text in (({"dtype": 0}, b"FTNN_F16"), ({"heads_q": 3}, b"3 query heads"), ({"heads_q": 0}, b"query heads"), ({"scale": 0.0}, b"scale"), ({"scale": -1.0}, b"scale"),
                     ({"scale": float("nan")}, b"scale"), ({"scale": float("inf")}, b"scale"), ({"max_len": -1}, b"max_len"), ({"q": None}, b"null"), ({"out": P + 1}, b"aligned")):
        assert refused(attend(_kv(), **kw), text), kw
    long = dict(width=4096, table_stride=4096)
    need = int(L.ftnn_kv4_attention_scratch_bytes(_kv(**long), 4, 0))
    assert need > 0 and refused(attend(_kv(**long), scratch=None, n=0), b"scratch") and refused(attend(_kv(**long), n=need - 1), b"scratch")
    assert refused(attend(_kv(**long), scratch=P + 8), b"scratch")
    assert L.ftnn_kv4_attention_scratch_bytes(_kv(**long), 4, 20) < need   # a sequence known to be short is not split as far
    assert attend(_kv(tokens=0), q=None, out=None, scratch=None, n=0) == 0 and attend(_kv(sequences=0)) == 0
