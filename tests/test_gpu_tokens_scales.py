"""Scales of the 4-bit cache where a quotient is next to halfway between two numbers of bfloat16."""
import math

import pytest

torch = pytest.importorskip("torch")
import fastertnn_amd.lib as lib
from tests import tokens_oracle as ref

pytestmark = pytest.mark.gpu


def _ends():
    """smallest and largest values whose difference is 15 times a number halfway between two of bfloat16 (9 bits, the last one set), or a step of fp32 beside that:
    a quotient that is not halfway, until it is rounded to fp32"""
    for i in range(64):
        middle = (257 + 2 * i) / 2.0 ** 10
        low = -float(int(15 * middle))
        at = torch.tensor(15 * middle + low, dtype=torch.float32)
        for high in (at, torch.nextafter(at, torch.tensor(math.inf)), torch.nextafter(at, torch.tensor(-math.inf))):
            assert torch.tensor((float(high) - low) / 15).float() == middle
            yield low, float(high)


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_scales_are_rounded_to_fp32_first(dim):
    ends = list(_ends())
    low, high = (torch.tensor(e, dtype=torch.float32)[:, None] for e in zip(*ends))
    k = torch.minimum(torch.maximum(torch.linspace(0, 1, dim) * (high - low) + low, low), high)
    k[:, :1], k[:, -1:] = low, high
    k, n, page = k[:, None], len(ends), 64
    raw = torch.zeros((n // page, lib.kv4_page_bytes(1, dim, page)), dtype=torch.uint8)
    table, lens, starts = torch.arange(n // page, dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32), torch.tensor([0, n], dtype=torch.int32)
    want = ref.Cache(raw, 1, dim, page)
    ref.append(want, table, lens, starts, k, -k)
    cache = raw.cuda()
    lib.kv4_append(cache, table.cuda(), lens.cuda(), starts.cuda(), k.cuda(), -k.cuda(), page)
    assert torch.equal(cache.cpu(), want.raw())
