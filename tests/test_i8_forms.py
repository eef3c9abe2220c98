"""Which form a product of 8-bit rows takes (fastertnn_amd/csrc/i8_forms.h, the code the launchers run): the shapes of the GPU tests are
held to the forms that they are there for.  CPU only."""
import os
import subprocess

import pytest

import fastertnn_amd.lib as lib
from tests import i8_shapes

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAMES = ["T256", "T128", "T128Two", "T128x64", "T64", "T64Split"]


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    """(packed, m, n, k) -> ((nb, mb), form of tiles)"""
    tmp = tmp_path_factory.mktemp("i8")
    src, exe = tmp / "forms.cpp", tmp / "forms"
    src.write_text(r"""
#include <stdio.h>
#include "i8_forms.h"
int main() {
    long long m, n;
    int packed, k;
    while (scanf("%d %lld %lld %d", &packed, &m, &n, &k) == 4) {
        const ftnn::I8Few f = ftnn::i8_few(packed, m, n, k);
        printf("%d %d %d\n", f.nb, f.mb, (int)ftnn::i8_form(m, n, k));
    }
}
""")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", os.path.join(ROOT, "fastertnn_amd", "csrc"), str(src), "-o", str(exe)],
                   check=True, timeout=120)

    def run(shapes):
        r = subprocess.run([str(exe)], input="\n".join("%d %d %d %d" % s for s in shapes), capture_output=True, text=True, check=True, timeout=120)
        return [((int(a), int(b)), NAMES[int(c)]) for a, b, c in (line.split() for line in r.stdout.splitlines())]

    return run


def test_shapes_of_the_gpu_tests(choose):
    for name, ((m, n), ks) in i8_shapes.TILES.items():
        assert choose([(0, m, n, k) for k in ks]) == [((0, 0), name)] * len(ks)
        assert [f[1] for f in choose([(1, m, n, k) for k in ks])] == [name] * len(ks)
    for name in i8_shapes.TILES_PACKED:
        (m, n), ks = i8_shapes.TILES[name]
        assert choose([(1, m, n, ks[-1])]) == [((0, 0), name)]
    for packed, table in ((0, i8_shapes.FEW_CODES), (1, i8_shapes.FEW_PACKED)):
        for form, (m, n) in table.items():
            for k in i8_shapes.FEW_K:
                assert choose([(packed, m, n, k)])[0][0] == form
                assert not packed or lib.mm_i8_rows_scratch_bytes(True, m, n, k) == 0


def test_every_size_has_a_form(choose):
    """up to the largest that a call may have"""
    most = 2**31 - 1
    shapes = [(p, m, n, k) for p in (0, 1) for m in (1, 16, 17, 1000, 65536, most) for n in (1, 15, 4096, 65537, most) if m * n < 2**40 for k in (1, 128, 131071)]
    for (p, m, n, k), ((nb, mb), form) in zip(shapes, choose(shapes)):
        if nb:
            assert -(-n // (16 * nb)) * -(-m // (16 * mb)) < 2**31
        else:
            edge = {"T256": 256 * 256, "T128": 128 * 128, "T128Two": 128 * 128, "T128x64": 128 * 64}.get(form, 64 * 64)
            assert m * n // edge < 2**28   # numbers of tiles are 32 bits
