"""The paged key/value cache and its attention from their definitions, in 64 bits.

Shared by the paged tests. Everything here is plain indexing and float64 arithmetic on the host
or device torch offers; nothing calls the library.
"""
import math

import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
FORMATS = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "i8": torch.int8}
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def round_e4m3(x):
    """float64 -> nearest e4m3 value (ties to even, saturating), as float64."""
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(e - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def stored(x, dtype):
    """(codes as float64, scale as float64 [..., 1]) of rows x [..., hd] in a cache of `dtype`."""
    x = x.double()
    if dtype == torch.bfloat16:
        return x.bfloat16().double(), torch.ones_like(x[..., :1])
    fine = torch.isfinite(x).all(-1, keepdim=True)
    x = torch.where(fine, x, 0.0)
    s = (x.abs().amax(-1, keepdim=True) / TOP[dtype]).float().double()
    s = torch.where(s > 0, s, 1.0)
    q = (x / s).float().double()
    q = round_e4m3(q) if dtype == torch.float8_e4m3fn else torch.round(q).clamp(-127, 127)
    return q, torch.where(fine, s, math.nan)


def codes(t):
    """Cache codes as float64."""
    return t.float().double()


def values(t, scale):
    """What cache codes t [..., hd] with scales [...] stand for, float64."""
    x = codes(t)
    return x if scale is None else x * scale.double()[..., None]


def make_pages(lens, page, max_pages=None, spare=2, seed=0):
    """(pages [S, max_pages] int32, pool size): shuffled, no page used twice."""
    used = [-(-n // page) for n in lens]
    pool = sum(used) + spare
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    pages = torch.full((len(lens), max(max_pages or 0, *used, 1)), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(used):
        pages[s, :n] = order[at:at + n]
        at += n
    return pages, pool


def sequence(vals, pages, n):
    """Rows 0..n-1 of one sequence: vals [n_pages, heads, page, hd] -> [n, heads, hd]."""
    page = vals.shape[2]
    p = pages[: -(-n // page)].long().to(vals.device)
    return vals[p].permute(0, 2, 1, 3).reshape(-1, vals.shape[1], vals.shape[3])[:n]


def attend(q, k, v, pos0, scale, window=0):
    """q [n, H, hd], k / v [keys, Hkv, hd] float64, query i at position pos0 + i. Returns
    (o, sum_j p_j |v_j|, max_j scale * sum_d |q_d k_d|, keys * max |v|): the result and what its
    error scales with. Rows that see nothing are 0."""
    n, H, hd = q.shape
    G = H // k.shape[1]
    kh, vh = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    j = torch.arange(k.shape[0], device=q.device)
    p = pos0 + torch.arange(n, device=q.device)[:, None]
    see = (j <= p) & (j > p - (window or 1 << 40))
    s = torch.einsum("nhd,khd->hnk", q, kh) * scale
    s = s.masked_fill(~see, -math.inf)
    m = s.amax(-1, keepdim=True) if k.shape[0] else torch.zeros((H, n, 1), dtype=q.dtype, device=q.device)
    w = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
    # a key that a row does not see does not reach it, whatever its value
    vz = torch.where(torch.isfinite(vh), vh, 0.0)
    o = torch.einsum("hnk,khd->nhd", w, vz)
    a = torch.einsum("hnk,khd->nhd", w, vz.abs())
    b = torch.einsum("nhd,khd->hnk", q.abs(), kh.abs()) * scale
    b = b.masked_fill(~see, 0.0).amax(-1).T[..., None] if k.shape[0] else torch.zeros_like(o[..., :1])
    u = k.shape[0] * vz.abs().amax((0, 2))[:, None] if k.shape[0] else torch.zeros_like(o[..., :1])
    return o, a, b, u


def tolerance(o, a, b, u, dtype, cache):
    """Bound on |out - o|, elementwise.

    Scores: an operand is within 2^-22 of itself (binary16 hi + lo; three bfloat16 terms do
    better), a sum of 128 products takes at most 9 tensor-core additions per term of the operand,
    each short of its largest partial sum by at most 17 * 2^-24: below 2^-16 b in all for the
    terms together. exp turns an absolute error d of a score into a relative 2 d of its weight at
    most, and again of the sum that divides. Weights and values: as the operands, 2^-17 of a.
    BF16 queries may have weights rounded to BF16 (half a step, 2^-8) before a BF16 cache, binary16
    (2^-11) before an 8-bit one. The result is rounded to dtype (half a step).

    Before an 8-bit cache a weight times its value's scale is held in binary16, whose smallest step
    is 2^-24: as hi + lo it is off by up to 2^-25, however small it is itself, where the row's largest
    weight and the largest scale make 2^13 (F32) or 2^5 (BF16) to twice that. So each of the keys
    may add 2^-38 (2^-30) of the largest value, which u sums; 2^-37 (2^-29) for the factor of two."""
    t = a * (4 * b * 2.0 ** -16 + 2.0 ** -17)
    if cache != torch.bfloat16:
        t = t + u * (2.0 ** -37 if dtype == torch.float32 else 2.0 ** -29)
    if dtype == torch.bfloat16:
        t = t + a * (2.0 ** -8 if cache == torch.bfloat16 else 2.0 ** -11) + (o.abs() + t) * 2.0 ** -8
    return t + 1e-37
