"""Calls on the 4-bit cache that are larger than a launch: refused before any device work.  CPU only."""
import ctypes as C

import fastertnn_amd.lib as lib

L = lib._L
BUF = (C.c_char * 8192)()
P = (C.addressof(BUF) + 255) & ~255


def _too_large(rc):
    return rc < -1 and b"invalid configuration" in L.ftnn_last_error()


def test_more_tokens_than_a_launch_holds():
    kv = lambda tokens, dim=64: C.byref(lib.Kv4Desc(P, 4, 1, dim, 16, 1, tokens, 2, 2, P, P, P))
    for tokens in (1 << 27, (1 << 31) - 1):
        assert _too_large(L.ftnn_kv4_append(kv(tokens), 2, P, 64, 64, P, 64, 64, None, None, 0, 0, 0, 0, None, 0, 0, None, None))
        assert _too_large(L.ftnn_kv4_read(kv(tokens), 2, P, P, None))
    for dim, tokens in ((64, (1 << 31) - 1), (256, 1 << 30)):
        assert _too_large(L.ftnn_kv4_attention(kv(tokens, dim), 2, 1, P, dim, dim, 1.0, 0, P, P, 1 << 40, None))
