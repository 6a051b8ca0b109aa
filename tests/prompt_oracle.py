"""Causal and differential paged attention in float64, with a bound on what the kernel may be off.

Plain loops over sequences and heads, from the formulas. Cache rows are what they stand for: int8
values times their scales exactly, bf16 rows as fp16 (the same value inside fp16's range).

The bound, per output element, before the result's own rounding (half a step, u_out |y|):
  * P (int8: P times V's scale) is rounded to fp16 (2^-11 of p, or 2^-25 where it is subnormal;
    the row's normaliser is at least 1): 2^-11 sum p|v| + 2^-25 sum |v|;
  * scores: D products summed in fp32 and one fma, D + 2 roundings of at most 2^-24 of sum |q k|
    each, twice (numerator and normaliser), and exp2 (2^-22);
  * sums over T tokens in fp32: T 2^-24, twice.
"""

from __future__ import annotations

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def dense_rows(cache, b):
    """K and V of sequence b, [T, Hkv, D] float64."""
    t = int(cache.seq_lens[b])
    pos = torch.arange(t, device=cache.k_cache.device)
    blk = cache.block_table[b].long()[pos // cache.block_size]
    off = pos % cache.block_size
    rows = []
    for store, scale in ((cache.k_cache, cache.k_scale), (cache.v_cache, cache.v_scale)):
        x = store[blk, off]
        if scale is not None:
            rows.append(x.double() * scale[blk, off].double()[..., None])
        else:
            rows.append(x.to(torch.float16).double())
    return rows


def one_map(q, k, v, first, scale):
    """softmax(scale q k^T) v of one head: q [n, D], k [T, D], v [T, E] float64, row i seeing tokens
    0 .. first + i. Returns the result and its bound; rows that see nothing are zeros."""
    n, d = q.shape
    t = k.shape[0]
    y = torch.zeros((n, v.shape[1]), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(y)
    for i in range(n):
        seen = min(t, first + i + 1)
        if seen <= 0:
            continue
        kk, vv = k[:seen], v[:seen]
        s = (kk @ q[i]) * scale
        p = torch.softmax(s, 0)
        y[i] = (p[:, None] * vv).sum(0)
        size = (kk.abs() @ q[i].abs()).max() * scale
        rel = 2.0 ** -11 + 2 * (d + 2) * 2.0 ** -24 * size + 2 * seen * 2.0 ** -24 + 2.0 ** -21
        bound[i] = rel * (p[:, None] * vv.abs()).sum(0) + 2.0 ** -25 * vv.abs().sum(0)
    return y, bound


def attend(q, cache, start, sm_scale=None, lam=None, norm_weight=None, norm_eps=0.0, out_scale=1.0):
    """(result, bound) for packed rows q [N, Hq, D]; `start` a list of B + 1 offsets. Rows of no
    sequence are zeros with a bound of zero."""
    n, hq, d = q.shape
    hkv = cache.shape.num_kv_heads
    maps = 1 if lam is None else 2
    group = hq // hkv
    scale = d ** -0.5 if sm_scale is None else sm_scale
    qq = q.to(torch.float16).double()
    y = torch.zeros((n, hq // maps, maps * d), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(y)
    for b in range(len(start) - 1):
        lo, hi = start[b], start[b + 1]
        if lo == hi:
            continue
        k, v = dense_rows(cache, b)
        first = k.shape[0] - (hi - lo)
        for h in range(hq // maps):
            j = h // group
            if maps == 1:
                y[lo:hi, h], bound[lo:hi, h] = one_map(qq[lo:hi, h], k[:, j], v[:, j], first, scale)
                continue
            vv = torch.cat([v[:, 2 * j], v[:, 2 * j + 1]], 1)
            one, e1 = one_map(qq[lo:hi, 2 * h], k[:, 2 * j], vv, first, scale)
            two, e2 = one_map(qq[lo:hi, 2 * h + 1], k[:, 2 * j + 1], vv, first, scale)
            w = float(lam[h])
            o, e = one - w * two, e1 + abs(w) * e2 + 2.0 ** -22 * (one.abs() + abs(w) * two.abs())
            if norm_weight is not None:
                # f = rsqrt(mean o^2 + eps) moves by at most the root mean square of e, relatively
                f = (o.square().mean(-1, keepdim=True) + norm_eps).rsqrt()
                moved = (e.square().mean(-1, keepdim=True)).sqrt() * f + 2.0 ** -20
                w = norm_weight.double() * out_scale
                e = (e + o.abs() * moved) * f * w.abs()
                o = o * f * w
            y[lo:hi, h], bound[lo:hi, h] = o, e
    return y, bound


def worst(got, want, bound):
    """The largest error as a share of what is allowed (below 1: in bounds). Infinities and NaN have
    to be the same."""
    got64 = got.double()
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got64), torch.isnan(want)), "NaN in other places"
    keep = odd & ~torch.isnan(want)
    assert torch.equal(got64[keep], want[keep]), "infinities differ"
    allowed = bound + HALF_STEP[got.dtype] * (want.abs() + bound) + 2.0 ** -25
    share = (got64 - want).abs() / allowed
    return float(share[~odd].max()) if bool((~odd).any()) else 0.0
