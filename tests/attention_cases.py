"""Calls of attention over the 4-bit cache at which its arithmetic can be told apart: caches that are written code by code."""
import torch

import fastertnn_amd.lib as lib
from tests import tokens_oracle as ref


def make(heads, dim, page, lens, new, seed):
    """an empty cache with its pages in order, and the arrays of a call"""
    width = -(-max(lens) // page)
    pages = len(lens) * width
    cache = ref.Cache(torch.zeros((pages, lib.kv4_page_bytes(heads, dim, page)), dtype=torch.uint8), heads, dim, page)
    g = torch.Generator().manual_seed(seed)
    for codes in (cache.k, cache.v):
        codes.copy_(torch.randint(0, 16, codes.shape, generator=g))
    for params in (cache.kp, cache.vp):
        scale = torch.rand(params.shape[:-1], generator=g) * 0.3 + 0.05
        params.copy_(torch.stack([scale, -scale * (6 + 3 * torch.rand(scale.shape, generator=g))], -1))
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    table = torch.arange(pages, dtype=torch.int32).view(len(lens), width)
    return cache, table, torch.tensor(lens, dtype=torch.int32), torch.tensor(starts, dtype=torch.int32), g


def set_scale(cache, table, s, t, factor):
    """the values of token t of sequence s times a power of two"""
    cache.vp[table[s, t // cache.page].item(), :, t % cache.page] *= factor


def set_score(cache, table, s, t, zero):
    """token t's keys all `zero`: its scores go by the sum of a query"""
    at = (table[s, t // cache.page].item(), slice(None), t % cache.page)
    cache.kp[at] = torch.tensor([0.0, zero], dtype=torch.bfloat16)


def queries(cache, starts, group, dtype, g):
    """positive, so that their sums are about 0.8 dim"""
    return torch.randn((int(starts[-1]), cache.heads * group, cache.dim), generator=g).abs().to(dtype)


def unseen(heads, group, dim, page, length, new, ratio, dtype, seed=1):
    """the last token's values are `ratio` times the others': only the last row sees it"""
    cache, table, lens, starts, g = make(heads, dim, page, [length], [new], seed)
    q = queries(cache, starts, group, dtype, g)
    cache.vp *= 2.0 ** -8   # (float16 holds what the last row makes of it)
    set_scale(cache, table, 0, length - 1, ratio)
    return cache, table, lens, starts, q


def weightless(heads, group, dim, page, lens, new, ratio, dtype, where, seed=2):
    """tokens `where` of each sequence: values `ratio` times the others', and weights of exp(-60) or so: a key of -c gives -c 0.8 sqrt(dim)"""
    cache, table, ln, starts, g = make(heads, dim, page, lens, new, seed)
    q = queries(cache, starts, group, dtype, g)
    cache.kp[..., 1] = -cache.kp[..., 0] * 7.5   # others: about 0
    cache.vp *= 2.0 ** -8
    for s in range(len(lens)):
        for t in where:
            set_scale(cache, table, s, t, ratio)
            set_score(cache, table, s, t, -60 / (0.8 * dim ** 0.5))
    return cache, table, ln, starts, q


def mixed(heads, group, dim, page, lens, new, spread, dtype, seed=3):
    """every token's scale its own, over 2^-spread .. 2^spread"""
    cache, table, ln, starts, g = make(heads, dim, page, lens, new, seed)
    cache.vp *= 2.0 ** torch.randint(-spread, spread + 1, cache.vp.shape[:-1], generator=g)[..., None].float()
    return cache, table, ln, starts, queries(cache, starts, group, dtype, g) * 0.5


def two_halves(heads, group, dim, page, dtype, sequences=1, seed=4):
    """32 tokens, the first half with key codes 0 and values of one sign, the second with key codes 15 and values of the other; queries of one value other
    than 0.  Scores are next to exact, weights are any numbers, outputs are small beside what they are sums of: the rounding of the weights is what is left"""
    cache, table, lens, starts, g = make(heads, dim, page, [32] * sequences, [1] * sequences, seed)
    n = torch.arange(32)
    at = table.long()[:, n // page], n % page
    second = (n >= 16).view(1, 32, 1, 1)
    kc = torch.where(second, 15, 0).expand(sequences, 32, heads, dim)
    swing = torch.randint(1, 8, (sequences, 1, heads, dim), generator=g)
    vc = torch.where(second, 8 + swing, 8 - swing.roll(1, 3)).expand(sequences, 32, heads, dim)
    for codes, c in ((cache.k, kc), (cache.v, vc)):
        codes[at[0], :, at[1]] = c.to(torch.uint8)
    cache.kp[..., 0], cache.kp[..., 1] = 0.125, -0.9375
    cache.vp[..., 0], cache.vp[..., 1] = 1.0, -8.0
    q = torch.zeros((sequences, heads * group, dim))
    one = torch.randint(0, dim, q.shape[:-1], generator=g)
    q.scatter_(2, one[..., None], (torch.rand(one.shape, generator=g) * 2 - 1)[..., None] * 0.5 * dim ** 0.5)
    return cache, table, lens, starts, q.to(dtype)


def cancelling(heads, group, page, length, sequences, dtype, mean=8, seed=5):
    """every 32 tokens are followed by 32 of the same keys and the opposite values: outputs are 0, whatever the weights.  One long sequence, which all sequences of
    the call share; values are 1024 (code - mean)"""
    dim = 64
    cache, table, lens, starts, g = make(heads, dim, page, [length], [1], seed)
    at = torch.arange(length) // page, torch.arange(length) % page
    twice = lambda a, b: torch.stack([a, b], 1).view(length, heads, dim)
    keys = torch.randint(0, 16, (length // 64, 32, heads, dim), generator=g, dtype=torch.uint8)
    side = torch.randint(0, 2, (length // 64, 32, heads, dim), generator=g, dtype=torch.uint8) * 2 + mean - 1
    cache.k[at[0], :, at[1]], cache.v[at[0], :, at[1]] = twice(keys, keys), twice(side, 2 * mean - side)
    cache.kp[..., 0], cache.kp[..., 1] = 0.125, -0.9375
    cache.vp[..., 0], cache.vp[..., 1] = 1024.0, -1024.0 * mean
    q = torch.zeros((sequences, heads * group, dim))
    one = torch.randint(0, dim, q.shape[:-1], generator=g)
    q.scatter_(2, one[..., None], (torch.rand(one.shape, generator=g) * 2 - 1)[..., None] * dim ** 0.5)
    return cache, table.expand(sequences, -1).contiguous(), lens.repeat(sequences), torch.arange(sequences + 1, dtype=torch.int32), q.to(dtype)
