"""The operators of token models in few bits in 64 bits on the CPU: what the GPU tests compare with."""
import math

import torch


def quantize_rows(x):
    """codes (whole numbers) and scales; rows with a NaN or an infinity: zeros and NaN"""
    y = x.double()
    most = y.abs().amax(1)
    fine = torch.isfinite(most)   # amax hands a NaN on
    safe = torch.where(fine & (most > 0), most, 1.0)
    q = torch.where((fine & (most > 0))[:, None], torch.round(torch.nan_to_num(y * 127) / safe[:, None]), 0.0)
    return q.to(torch.int64), torch.where(fine, (most / 127).float(), math.nan)


def product(a, sa, b, sb, bias, dtype):
    """the result and how far one of `dtype` may be from it: the sum to fp32, two scales and a bias, half a step each, and the result's
    own rounding, half a step: eps / 2 of the value, or of the smallest normal number below that, where steps no longer shrink (float16: 2^-25)"""
    s = a.double() @ b.double().t()   # exact: below 2^53
    y = s * sa.double()[:, None] * sb.double()
    slack = y.abs() * 4 * 2.0 ** -24
    if bias is not None:
        y = y + bias.double()
    return y, slack + y.abs() * (2.0 ** -24 + torch.finfo(dtype).eps / 2) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def lanes(n, k, ternary, generator):
    t = torch.randint(-1, 2, (n, k), generator=generator) if ternary else torch.randint(0, 2, (n, k), generator=generator) * 2 - 1
    return t.double()


# ------------------------------------------------------------------------------------------------------ the cache

class Cache:
    """pages as a dense array of codes and parameters, laid out as bytes on demand"""

    def __init__(self, raw, heads, dim, page):
        self.heads, self.dim, self.page = heads, dim, page
        pages, n = raw.shape[0], page * dim // 2
        block = raw.view(pages, heads, page * (dim + 8))
        self.k = self._nibbles(block[:, :, :n].reshape(pages, heads, page, dim // 2))
        v = self._nibbles(block[:, :, n:2 * n].reshape(pages, heads, page // 8, dim, 4))
        self.v = v.permute(0, 1, 2, 4, 3).reshape(pages, heads, page, dim).contiguous()
        params = block[:, :, 2 * n:].contiguous().view(torch.bfloat16).view(pages, heads, 2, page, 2)
        self.kp, self.vp = params[:, :, 0].clone(), params[:, :, 1].clone()

    @staticmethod
    def _nibbles(b):
        return torch.stack([b & 15, b >> 4], -1).flatten(-2).contiguous()

    def raw(self):
        pages, d, page = self.k.shape[0], self.dim, self.page
        k = self.k[..., 0::2] | self.k[..., 1::2] << 4
        v = self.v.view(pages, self.heads, page // 8, 8, d).transpose(3, 4)
        v = v[..., 0::2] | v[..., 1::2] << 4
        params = torch.stack([self.kp, self.vp], 2).contiguous().view(torch.uint8)
        flat = lambda x: x.reshape(pages, self.heads, -1)
        return torch.cat([flat(k), flat(v), flat(params)], 2).reshape(pages, -1)


def rotate(x, pos, cos, sin, neighbours):
    """[heads][dim] at a position, rounded to fp32"""
    y = x.double().clone()
    if cos is not None:
        half = cos.shape[1]
        i = torch.arange(half)
        a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + half)
        c, s = cos[pos].double(), sin[pos].double()
        y[:, a], y[:, b] = y[:, a] * c - y[:, b] * s, y[:, b] * c + y[:, a] * s
    return y.float()


def codes(y):
    """[heads][dim] in fp32 -> codes, (scale, zero) in bfloat16"""
    y = y.double()
    low, high = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    zero, scale = low.float().bfloat16(), ((high - low) / 15).float().bfloat16()
    fine = torch.isfinite(y).all(-1, keepdim=True) & torch.isfinite(zero)
    zero, scale = (torch.where(fine, p, torch.tensor(math.nan, dtype=torch.bfloat16)) for p in (zero, scale))
    q = torch.round((y - zero.double()) / scale.double()).clamp(0, 15)
    return torch.where(scale.double() > 0, q, 0.0).to(torch.uint8), torch.cat([scale, zero], -1)


def new_tokens(table, lens, starts, tokens):
    """(row, sequence, position) of every token of a call"""
    for s, n in enumerate(lens.tolist()):
        for t in range(int(starts[s]), min(int(starts[s + 1]), tokens)):
            yield t, s, n - int(starts[s + 1]) + t


def slot(cache, table, s, pos, pages):
    """(page, slot) of a position, or None where there is none"""
    if pos < 0 or pos // cache.page >= table.shape[1]:
        return None
    page = int(table[s, pos // cache.page])
    return (page, pos % cache.page) if 0 <= page < pages else None


def append(cache, table, lens, starts, k, v, cos=None, sin=None, neighbours=False, q=None, q_out=None):
    for t, s, pos in new_tokens(table, lens, starts, k.shape[0]):
        if pos < 0 or (cos is not None and pos >= cos.shape[0]):
            continue
        if q is not None:
            q_out[t] = rotate(q[t], pos, cos, sin, neighbours).to(q.dtype)
        at = slot(cache, table, s, pos, cache.k.shape[0])
        if at:
            cache.k[at[0], :, at[1]], cache.kp[at[0], :, at[1]] = codes(rotate(k[t], pos, cos, sin, neighbours))
            cache.v[at[0], :, at[1]], cache.vp[at[0], :, at[1]] = codes(v[t].float())


def values(cache, page, i):
    """keys and values of a slot, [heads][dim]"""
    return [p[page, :, i, 1:].double() + p[page, :, i, :1].double() * c[page, :, i].double() for c, p in ((cache.k, cache.kp), (cache.v, cache.vp))]


def read(cache, table, lens, starts, tokens, dtype):
    out = torch.zeros((2, tokens, cache.heads, cache.dim), dtype=torch.float64)
    for t, s, pos in new_tokens(table, lens, starts, tokens):
        at = slot(cache, table, s, pos, cache.k.shape[0])
        if at:
            out[0, t], out[1, t] = values(cache, *at)
    return [x.float().to(dtype) for x in out]   # zero + scale * code: its product is exact, one rounding to fp32


def attention(cache, table, lens, starts, q, scale=None):
    """the outputs of the call's rows and how far those of the kernel may be.  The bound of a row, with u = 2^-24:
      scores   a sum of dim products of at most 143 |q| and their correction, in fp32: (dim + 8) u (143 ks + |kz|) sum |q|, times the
               scale the relative error of a weight, and 2^-21 for the power of two
      weights  rounded to a unit of 2^-8 (float16: 2^-16 by two parts) where they meet code - 8
      sums     fp32 over steps of 32 tokens, of terms up to 143 + 136 times scale * weight
    (a bound for products in bfloat16 with an offset of 128; ones in float16 without it are well inside)
      result   half a step of its type (below its normal numbers: of the smallest of those)"""
    tokens, heads_q, dim = q.shape
    group, scale = heads_q // cache.heads, dim ** -0.5 if scale is None else scale
    out, slack = torch.zeros((tokens, heads_q, dim), dtype=torch.float64), torch.zeros((tokens, heads_q, dim), dtype=torch.float64)
    u, unit = 2.0 ** -24, 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -16
    for s, n in enumerate(lens.tolist()):
        first, last = int(starts[s]), min(int(starts[s + 1]), tokens)
        if last <= first:
            continue
        at = [(p, slot(cache, table, s, p, cache.k.shape[0])) for p in range(max(n, 0))]
        at = [(p, a) for p, a in at if a]
        if not at:
            continue
        pos = torch.tensor([p for p, _ in at])
        page, i = torch.tensor([a[0] for _, a in at]), torch.tensor([a[1] for _, a in at])
        for h in range(cache.heads):
            kp, vp = cache.kp[page, h, i].double(), cache.vp[page, h, i].double()
            k, v = kp[:, 1:] + kp[:, :1] * cache.k[page, h, i], vp[:, 1:] + vp[:, :1] * cache.v[page, h, i]
            x = q[first:last, h * group:(h + 1) * group].double().reshape(-1, dim)
            row_pos = (n - int(starts[s + 1]) + torch.arange(first, last)).repeat_interleave(group)
            hidden = pos > row_pos[:, None]
            score = (x @ k.t() * scale).masked_fill(hidden, -math.inf)
            blind = hidden.all(1)
            p = torch.softmax(score.masked_fill(blind[:, None], 0.0), 1).masked_fill(blind[:, None], 0.0)
            p = p.masked_fill(hidden, 0.0)
            looked = (~hidden).any(0)   # what no row sees adds nothing, whatever it is
            kp, vp, v = (torch.where(looked[:, None], a, 0.0) for a in (kp, vp, v))
            o = p @ v
            most = lambda a: torch.where(hidden, 0.0, a).amax(1)   # of what a row sees
            rel = scale * (dim + 8) * u * x.abs().sum(1) * most(143 * kp[:, 0] + kp[:, 1].abs()) + 2.0 ** -21
            vmax = most(v.abs().amax(1))
            round_w = p @ (vp[:, :1] * (cache.v[page, h, i].double() - 8).abs())
            sums = (p @ vp[:, 0])[:, None] * 279 * (len(at) / 32 + 64) * u
            e = unit * round_w + 4 * rel[:, None] * vmax[:, None] + sums + o.abs() * (torch.finfo(q.dtype).eps / 2 + 8 * u) + torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps / 2
            out[first:last, h * group:(h + 1) * group] = o.view(last - first, group, dim)
            slack[first:last, h * group:(h + 1) * group] = e.view(last - first, group, dim)
    return out, slack
