"""Attention over the 4-bit cache in 64 bits, with a bound of the kernel's own arithmetic (fastertnn_amd/csrc/kv4_kernels.hip), and that
arithmetic's rounding of the weights on the CPU, to hold the bound to.

The bound of a result o = sum_t P_t v_t, with u = 2^-24, key k_t = kz + ks code and value v_t = vz + vs (code - 8), vz = zero + 8 vs:
  scores    products q code are exact; their sum is one of as many terms as the query has values other than 0, in fp32, then a
            multiply-add: (terms + 4) u sum |q| (15 ks + |kz|); queries keep what is above 2^-34 of their largest value.  The argument of the power of
            two is off by u of itself and 3 u of the score, the power by 2^-22.  A relative error of the weights e_t moves o by sum_t P_t e_t |v_t - o| at most
  weights   P vs is rounded to float16: 2^-11 of itself, or 2^-22 as the sum of two (float16 results), after two roundings in fp32; what is below
            float16's smallest step is lost: 2^-27 of the row's largest P vs
  sums      over 16 steps of 32 tokens sums of code * weight and of 8 * weight grow to (15 + 8) sum P vs of theirs, half of that in the mean, and each
            instruction is off by up to 8 u of what it sums (addends aligned, cut off and rounded): 16 * 8 u * 23 / 2 = 64 * 23 u of sum P vs; the sum of P vz runs
            through 128 tokens in a lane meanwhile.  What they make together is added to the output so far, at most sum P |v|, by which each of n / 32 steps is off by
            8 u again; the sum of P runs through a quarter of all tokens in a lane
  result    8 u of it for the quotient, and half a step of its type (below its normal numbers: of the smallest of those)"""
import math

import torch

from tests import tokens_oracle as ref

U = 2.0 ** -24


def _heads(cache, table, lens, starts, q, scale):
    """each sequence and head: the rows of the call, the query heads, and what the bound is made of"""
    tokens, heads_q, dim = q.shape
    group, scale = heads_q // cache.heads, dim ** -0.5 if scale is None else scale
    for s, n in enumerate(lens.tolist()):
        first, last = int(starts[s]), min(int(starts[s + 1]), tokens)
        at = [(p, ref.slot(cache, table, s, p, cache.k.shape[0])) for p in range(max(n, 0))] if last > first else []
        at = [(p, a) for p, a in at if a]
        if not at:
            continue
        pos = torch.tensor([p for p, _ in at])
        page, i = torch.tensor([a[0] for _, a in at]), torch.tensor([a[1] for _, a in at])
        for h in range(cache.heads):
            x = q[first:last, h * group:(h + 1) * group].double().reshape(-1, dim)
            hidden = pos > (n - int(starts[s + 1]) + torch.arange(first, last)).repeat_interleave(group)[:, None]
            seen = ~hidden.all(0)   # what no row sees may be any bytes
            ks, kz, vs, zero = (torch.where(seen, params[page, h, i, j].double(), 0.0) for params, j in ((cache.kp, 0), (cache.kp, 1), (cache.vp, 0), (cache.vp, 1)))
            kc, vc = cache.k[page, h, i].double(), cache.v[page, h, i].double() - 8
            score = (x @ (kz[:, None] + ks[:, None] * kc).t() * scale).masked_fill(hidden, -math.inf)
            blind = hidden.all(1)
            p = torch.softmax(score.masked_fill(blind[:, None], 0.0), 1).masked_fill(hidden, 0.0)
            yield (slice(first, last), slice(h * group, (h + 1) * group)), (last - first, group, dim), x, scale, score, hidden, p, ks, kz, vs, vc, zero + 8 * vs


def bound(cache, table, lens, starts, q, scale=None):
    """the outputs of the call's rows and how far the kernel's may be from them"""
    out, slack = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    info = torch.finfo(q.dtype)
    unit = 2.0 ** -22 if q.dtype == torch.float16 else 2.0 ** -11
    for rows, shape, x, scale_, score, hidden, p, ks, kz, vs, vc, vz in _heads(cache, table, lens, starts, q, scale):
        n = score.shape[1]
        v = vz[:, None] + vs[:, None] * vc
        o = p @ v
        key = 15 * ks + kz.abs()
        fine = score.masked_fill(hidden, 0.0)
        most = score.amax(1, keepdim=True).masked_fill(hidden.all(1, keepdim=True), 0.0)
        terms = (x != 0).sum(1)
        e = scale_ * ((terms + 4) * U * x.abs().sum(1) + terms * 2.0 ** -34 * x.abs().amax(1))[:, None] * key + U * (3 * fine.abs() + (fine - most).abs()) + 2.0 ** -22
        pe, w = p * e, p * vs
        from_scores = pe @ v.abs() + o.abs() * pe.sum(1, keepdim=True)
        size = w @ vc.abs()
        lost = 2.0 ** -27 * w.amax(1, keepdim=True) * ((~hidden).double() @ vc.abs())
        sums = 64 * 23 * U * w.sum(1, keepdim=True) + (n / 4 + 2) * U * (p @ v.abs()) + (min(n / 4, 128) + 64) * U * (p @ vz.abs())[:, None] + (n / 4 + 64) * U * o.abs()
        total = from_scores + (unit + 2 * U) * size + lost + sums + o.abs() * (info.eps / 2 + 8 * U) + info.smallest_normal * info.eps / 2
        out[rows], slack[rows] = o.view(shape), total.view(shape)
    return out, slack


def emulate(cache, table, lens, starts, q, scale=None, parts=None, round_to=torch.float16, by_scale=False):
    """the outputs with weights rounded as the kernel rounds them and all else in 64 bits.  `parts`: numbers that a weight is the sum of, `round_to`: their
    type; `by_scale`: weights in units of the largest vs, whatever a row makes of it"""
    out = torch.zeros(q.shape, dtype=torch.float64)
    parts = parts or (2 if q.dtype == torch.float16 else 1)
    for rows, shape, x, _, score, hidden, p, ks, kz, vs, vc, vz in _heads(cache, table, lens, starts, q, scale):
        w = p * vs
        w[:, 1::2] /= 16   # at the other elements codes count 16 times as much
        top = (vs.max().expand(w.shape[0], 1) if by_scale else w.amax(1, keepdim=True)).clamp_min(1e-300)
        unit = 2.0 ** (6 - torch.floor(torch.log2(top)))
        held, rest = torch.zeros_like(w), w * unit
        for _ in range(parts):
            part = rest.float().to(round_to).double()
            held, rest = held + part, rest - part
        held = held / unit
        held[:, 1::2] *= 16
        out[rows] = (held @ vc + p @ (vz[:, None]).expand(-1, vc.shape[1])).view(shape)
    return out.float().to(q.dtype).double()
