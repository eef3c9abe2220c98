"""Attention over the 4-bit cache held to the bound of its arithmetic (tests/attention_bound.py), where that can go wrong."""
import pytest

torch = pytest.importorskip("torch")
import fastertnn_amd.lib as lib
from tests import attention_bound, attention_cases as cases

pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _run(call, max_len=0):
    cache, table, lens, starts, q = call
    return lib.kv4_attention(q.cuda(), cache.raw().cuda(), table.cuda(), lens.cuda(), starts.cuda(), cache.heads, cache.page, max_len=max_len).cpu()


def _check(call, max_len=0):
    out = _run(call, max_len)
    want, slack = attention_bound.bound(*call)
    off = (out.double() - want).abs()
    assert torch.isfinite(out).all()
    assert bool((off <= slack).all()), "off by up to %.3g of the allowed" % float((off / slack).max())
    return out


def _many(heads, group, dim, new):
    """rows enough that wavefronts have all tokens of theirs"""
    assert new * group // (64 if dim == 256 else 128) * heads >= 480
    return heads, group, dim


# heads, group, dim, page, tokens, new ones
FORMS = [(1, 4, 64, 16, 300, 5), (2, 4, 128, 64, 300, 1), (1, 3, 96, 32, 90, 40), (1, 2, 256, 16, 200, 9), (16, 4, 64, 32, 1100, 1000), (12, 5, 128, 64, 1100, 1050), (16, 2, 256, 128, 1100, 1000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,group,dim,page,length,new", FORMS)
def test_a_token_of_large_values_that_rows_do_not_see(heads, group, dim, page, length, new, dtype):
    """the rows before it have the bits that they have without it"""
    if new >= 1000:
        _many(heads, group, dim, new)
    call = cases.unseen(heads, group, dim, page, length, max(new, 2), 2.0 ** 20, TYPES[dtype])
    out = _check(call)
    assert torch.equal(out[:-1], _run(cases.unseen(heads, group, dim, page, length, max(new, 2), 1.0, TYPES[dtype]))[:-1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ratio", [2.0 ** 12, 2.0 ** 20, 2.0 ** 40])
@pytest.mark.parametrize("heads,group,dim,page,length,new", FORMS)
def test_tokens_of_large_values_and_no_weight(heads, group, dim, page, length, new, ratio, dtype):
    """the first token of the sequence, one in the middle and one that the last step holds"""
    call = cases.weightless(heads, group, dim, page, [length], [1 if new < 1000 else new], ratio, TYPES[dtype], (0, length // 2, length - 2) if new < 1000 else (0, 40, 45))
    _check(call)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,group,dim,page,length,new", FORMS)
def test_tokens_of_all_scales(heads, group, dim, page, length, new, dtype):
    _check(cases.mixed(heads, group, dim, page, [length], [new], 6, TYPES[dtype]))


@pytest.mark.parametrize("max_len", [0, 4000])
def test_tokens_of_large_values_over_parts(max_len):
    """split over workgroups and wavefronts, most of which hold none of them"""
    _check(cases.weightless(1, 4, 128, 64, [4000], [1], 2.0 ** 30, torch.bfloat16, (0, 1333, 2666, 3998)), max_len)


@pytest.mark.parametrize("dtype", TYPES)
def test_sums_do_not_grow_with_the_length(dtype):
    """131072 tokens in one wavefront's sums, whose values cancel step by step.  In 16 steps sums of code * weight and of 8 * weight grow to 9 and 8 times the weights of
    those steps, half of that in the mean, and each step rounds both, by up to 2 u of them where what does not fit is cut off: 16 * 17 u = 272 u of the weights, and
    no more over all steps together.  (Sums over all tokens are as large as 9 times all weights, in each of 4096 steps.)"""
    call = cases.cancelling(2, 16383, 64, 131072, 2, TYPES[dtype])
    out = _run(call).double()
    assert float(out.square().mean().sqrt()) <= 272 * 2.0 ** -24 * 1024


@pytest.mark.parametrize("mean", [1, 5, 14])
def test_sums_far_from_the_middle_of_the_codes(mean):
    """the same with values that cancel about another code than 8, where what codes add and what the tokens' zeros add cancel too.  In 16 steps sums of code * weight
    and of 8 * weight grow to 15 and 8 times the weights of those steps: 16 * 2 u * (15 + 8) / 2 = 368 u of the weights.  The zeros add 7 times the weights, through 128
    tokens in a lane: if all adds went one way, 128 u / 2 * 7 / 2 = 224 u.  The weights themselves are float16 twice: 2^-22 of 7 times them, 28 u"""
    call = cases.cancelling(2, 16383, 64, 131072, 2, torch.float16, mean)
    out = _run(call).double()
    assert float(out.square().mean().sqrt()) <= 620 * 2.0 ** -24 * 1024


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,group,dim,lens,new", [(2, 4, 128, [5, 16, 33, 48, 330, 650], [1] * 6), (1, 8, 64, [1290, 17], [1, 1]), (1, 4, 256, [1001, 500], [3, 2]), (12, 5, 128, [1290], [1050]), (16, 4, 64, [1101], [1000])])
def test_what_the_table_holds_behind_the_sequences(heads, group, dim, lens, new, dtype):
    """pages of 16 tokens, half of a step: good pages behind the last one, bad ones, none at all"""
    cache, table, ln, starts, g = cases.make(heads, dim, 16, [max(lens) + 64] * len(lens), new, 6)
    ln = torch.tensor(lens, dtype=torch.int32)
    q = torch.randn((int(starts[-1]), heads * group, dim), generator=g).to(TYPES[dtype])
    want, slack = attention_bound.bound(cache, table, ln, starts, q)
    good = _run((cache, table, ln, starts, q), max(lens))
    assert bool(((good.double() - want).abs() <= slack).all())
    behind = torch.arange(table.shape[1]) >= (ln[:, None] + 15) // 16
    for bad in (-1, 1 << 30):
        assert torch.equal(_run((cache, torch.where(behind, bad, table), ln, starts, q), max(lens)), good)
    assert torch.equal(_run((cache, table[:, :(max(lens) + 15) // 16].contiguous(), ln, starts, q), max(lens)), good)


# from one token to thousands, ragged, odd numbers of heads: tokens split over wavefronts and workgroups, and wavefronts on all tokens
SHAPES = [(1, 1, 64, 16, [1], [1]), (2, 4, 128, 64, [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257], [1] * 16), (1, 8, 96, 32, [100, 31], [1, 1]),
          (2, 2, 256, 16, [77, 300], [1, 1]), (1, 20, 64, 32, [90, 40], [1, 1]), (2, 3, 64, 16, [40, 9, 100], [40, 1, 33]), (4, 4, 128, 32, [70, 64, 31], [5, 64, 1]),
          (2, 5, 256, 256, [280], [23]), (2, 4, 128, 64, [3000, 40, 1], [1, 1, 1]), (1, 6, 64, 16, [2500], [3]), (32, 2, 64, 64, [700, 300, 200], [600, 300, 123]),
          (16, 4, 128, 16, [990, 64, 1], [900, 64, 1]), (16, 5, 96, 32, [500, 420], [400, 419]), (8, 4, 256, 16, [1000, 70], [930, 70])]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,group,dim,page,lens,new", SHAPES)
def test_within_the_bound_of_its_arithmetic(heads, group, dim, page, lens, new, dtype):
    cache, table, ln, starts, g = cases.make(heads, dim, page, lens, new, dim + page + len(lens))
    q = torch.randn((int(starts[-1]), heads * group, dim), generator=g).to(TYPES[dtype])
    _check((cache, table, ln, starts, q))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,group,dim,page,sequences", [(2, 64, 64, 16, 1), (1, 30, 128, 32, 3), (1, 17, 96, 16, 2), (1, 16, 256, 64, 1), (8, 512, 64, 32, 16)])
def test_the_rounding_of_the_weights(heads, group, dim, page, sequences, dtype):
    """what a float16 result is held to takes both parts of its weights (one: 14 times the bound), what a bfloat16 result is held to takes float16 and not bfloat16"""
    _check(cases.two_halves(heads, group, dim, page, TYPES[dtype], sequences))


@pytest.mark.parametrize("exponent", [-100, 110])
@pytest.mark.parametrize("heads,group,dim,page,length,new", FORMS)
def test_values_at_the_ends_of_bfloat16(heads, group, dim, page, length, new, exponent):
    call = cases.mixed(heads, group, dim, page, [length], [new], 6, torch.bfloat16)
    call[0].vp *= 2.0 ** exponent
    _check(call)


@pytest.mark.parametrize("some", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,group,dim,page,length,new", [(1, 4, 64, 16, 9000, 1), (2, 4, 128, 64, 5000, 2), (1, 2, 256, 16, 5000, 3), (16, 4, 64, 32, 1700, 1000), (12, 5, 128, 64, 1700, 1050)])
def test_values_that_are_all_alike_in_a_token(heads, group, dim, page, length, new, dtype, some):
    """scales of 0 beside zeros that are not, over more than one run of 16 steps; `some`: tokens of ordinary values among them, small ones"""
    cache, table, lens, starts, g = cases.make(heads, dim, page, [length], [new], 7)
    alike = torch.rand(cache.vp.shape[:-1], generator=g) < (0.9 if some else 2)
    cache.vp *= 2.0 ** -10
    cache.vp[..., 0].masked_fill_(alike, 0.0)
    cache.vp[..., 1] = torch.where(alike, torch.randn(alike.shape, generator=g) * (1e4 if dtype == "f16" else 1e32), cache.vp[..., 1].float()).bfloat16()
    _check((cache, table, lens, starts, cases.queries(cache, starts, group, TYPES[dtype], g)))
