"""Bounds that hold F32 queries over the paged cache to what the split operands promise, and inputs that
show every term of them.

A dense product hides the last terms of its operands: the errors of 128 products and of hundreds of
weights average out, and the tensor cores' truncated sums err as much. So here a query row has one
element that is not 0 (each column in turn, in rows of different heads and tokens) and a column of V one
key that is not 0 (each key in turn): a score is one product, an output one weight times one value, and
nothing averages.

Bound on |out - o| / |o| of such inputs, S the largest |score| that a row sees (natural units):
  operands of a score: two binary16 terms leave 2^-22 of the query, three bfloat16 ones 2^-24; the terms'
    products with a cache value (8 bits) are exact, and the F32 additions that join them round or
    truncate by 2^-23 at most, two of them: 2^-22; scale, key scale and log2 e: 3 roundings of 2^-24 (a
    constant itself rounded: a fourth); the difference from the maximum: 2^-24 of S. In all (1 + 1 +
    5/4) 2^-22 S < 2^-20 S, and so much of the weight.
  the weight besides: the hardware's 2^x 2^-22, split terms 2^-22 (and 2^-38 of the row's largest, below
    2^-26 of weights above e^-8), value scale and the power that lifts them 2 x 2^-24, the product's
    truncated sums 2 x 2^-23: below 2^-20.
  the sum that divides: the weights' own errors, 2^-20 S + 2^-22, and its additions, `adds` of 2^-24.
  the division, the joins' factors and the last rounding: 4 x 2^-24 + 2 x 2^-22 < 3 x 2^-22.
Together 2^-19 S + 2^-19 + adds 2^-24.

Dense inputs are held by their root mean square: a score's truncated sums, 8 steps of at most 17 x 2^-24
(half of it on the average) of partial sums that are about 1 here, come to 2^-18, its weight's and the
sum's errors with them to 2^-17 of sum p |v|.
"""
import math

import torch


def bound(S, adds):
    return 2.0 ** -19 * S + 2.0 ** -19 + adds * 2.0 ** -24


DENSE_RMS = 2.0 ** -17


def sparse_queries(rows, H, hd, size, gen, device="cpu"):
    """[rows, H * hd] F32 with one element of magnitude size/2 .. size and full mantissa per head."""
    at = (torch.arange(rows, device=device)[:, None] * H + torch.arange(H, device=device)) % hd
    x = torch.rand((rows, H), generator=gen, device=device) * 0.5 + 0.5
    x = x * size * (1 - 2 * torch.randint(0, 2, x.shape, generator=gen, device=device))
    q = torch.zeros((rows, H, hd), device=device)
    q.scatter_(2, at[..., None], x[..., None].float())
    return q.view(rows, H * hd)


def sparse_values(L, Hkv, hd, gen, device="cpu"):
    """[L, Hkv * hd] F32: column d of head h is not 0 at key (d * 7 + h * 5) % L alone."""
    d = torch.arange(hd, device=device)
    v = torch.zeros((L, Hkv, hd), device=device)
    for h in range(Hkv):
        v[(d * 7 + h * 5) % L, h, d] = torch.rand(hd, generator=gen, device=device) + 0.5
    return v.view(L, Hkv * hd)


def cut(x, dtype, terms):
    """float64 x as the sum of its first `terms` roundings to dtype."""
    left, got = x.clone(), torch.zeros_like(x)
    for _ in range(terms):
        t = left.to(dtype).double()
        got, left = got + t, left - t
    return got


def attend(q, k, v, pos0, scale, dtype=None, q_terms=9, w_terms=9):
    """(o, S): causal attention in 64 bits, with q and the weights (relative to the row's largest times
    2^13, as the kernels hold them) cut to terms of dtype if there is one. q [n, H, hd], k, v [L, H, hd]."""
    n, L = q.shape[0], k.shape[0]
    see = torch.arange(L, device=q.device) <= pos0 + torch.arange(n, device=q.device)[:, None]
    if dtype == torch.float16:  # lifted to [2^13, 2^14)
        up = torch.exp2(13 - torch.floor(torch.log2(q.abs().amax(-1, keepdim=True).clamp_min(1e-300))))
        q = cut(q * up, dtype, q_terms) / up
    elif dtype is not None:
        q = cut(q, dtype, q_terms)
    s = (torch.einsum("nhd,khd->hnk", q, k) * scale).masked_fill(~see, -math.inf)
    S = s.abs().masked_fill(~see, 0).amax(-1).T[..., None]
    w = torch.exp(s - s.amax(-1, keepdim=True))
    total = w.sum(-1, keepdim=True)
    if dtype is not None:
        w = cut(w * 2.0 ** 13, dtype, w_terms) / 2.0 ** 13
    return torch.einsum("hnk,khd->nhd", w / total, v), S
