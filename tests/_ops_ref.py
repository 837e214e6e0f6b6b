"""64-bit definitions of the batched decode operators, and bounds for results
that are computed in f32 and rounded once.  Plain numpy, no repository code."""
from __future__ import annotations

import numpy as np

HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # of one rounding, relative
SMALLEST = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}  # half a subnormal step


def norm_rope(x, weight, offset, eps, positions, inv_freq):
    """x [T, H, D] -> (y, bound on |error| before the last rounding, in units of 1)."""
    y = x.astype(np.float64)
    D = y.shape[-1]
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * (weight.astype(np.float64) + offset)
    # f32 norm: D-1 additions of the sum of squares (halved by the square root), six more roundings
    rel = (D / 2 + 6) * 2.0 ** -24 if weight is not None else 0.0
    size = np.abs(y)
    if inv_freq is not None and len(inv_freq):
        n = len(inv_freq)
        a = positions.astype(np.float64)[:, None] * np.asarray(inv_freq, np.float64)
        c, s = np.cos(a)[:, None], np.sin(a)[:, None]
        lo, hi = y[..., :n].copy(), y[..., n:2 * n].copy()
        y[..., :n], y[..., n:2 * n] = lo * c - hi * s, hi * c + lo * s
        both = np.abs(lo) + np.abs(hi)
        size[..., :n] = size[..., n:2 * n] = both
        # cos and sin: 2 ulp of sincospi, one rounding of the angle's fraction; product and sum.
        # The 64-bit angle above itself is off by up to |a| 2^-53.
        rel += 8 * 2.0 ** -24 + np.abs(a).max() * 2.0 ** -53
    return y, size * rel


def attention(q, kc, vc, table, lens, scale, page, kind, cache_kind):
    """q [B, H, D], kc / vc [pages, page, KV, D] -> out, lse and their error bounds
    before the last rounding."""
    B, H, D = q.shape
    n_pages, KV = kc.shape[0], kc.shape[2]
    G = H // KV
    out, lse = np.zeros((B, H, D)), np.full((B, H), -np.inf)
    b_out, b_lse = np.zeros((B, H, D)), np.zeros((B, H))
    # queries of the cache's type go into the products as they are, float ones in two FP16 parts
    # (22 bits) or three BF16 parts (24)
    q_part = {"f16": 2.0 ** -22, "bf16": 0.0}[cache_kind] + 2.0 ** -24
    # and so do the probabilities of all of them (the bound allows BF16 queries 16 bits)
    p_part = 2.0 ** -22 if cache_kind == "f16" else 2.0 ** -17 if kind != "f32" else 2.0 ** -24
    for b in range(B):
        n = int(min(max(lens[b], 0), table.shape[1] * page))
        at = np.arange(n)
        pg = table[b, at // page] if n else at
        ok = (pg >= 0) & (pg < n_pages)
        if not ok.any():
            continue
        at, pg = at[ok] % page, pg[ok]
        for h in range(H):
            k = kc[pg, at, h // G].astype(np.float64)
            v = vc[pg, at, h // G].astype(np.float64)
            x = q[b, h].astype(np.float64)
            s = scale * (k @ x)
            top = s.max()
            p = np.exp(s - top)
            out[b, h] = (p @ v) / p.sum()
            lse[b, h] = top + np.log(p.sum())
            # one score: D products summed in f32 (2^-23 each: the tensor cores cut instead of rounding)
            d = ((D + 4) * 2.0 ** -23 + q_part) * abs(scale) * (np.abs(k) @ np.abs(x)).max()
            d += 4 * 2.0 ** -24 * (np.abs(s).max() + abs(top)) + 4 * 2.0 ** -23  # exponent's argument, exp2, shift
            # sums over the positions: one addition per 16 positions of a warp, a few joins
            acc = (len(s) / 16 + 40) * 2.0 ** -23
            b_out[b, h] = (2 * d + p_part + 2 * acc) * (p @ np.abs(v)) / p.sum()
            b_lse[b, h] = d + acc + 2.0 ** -22 * (1 + abs(lse[b, h]) + abs(top))
    return out, lse, b_out, b_lse


def logits(x, history=None, prompt=None, total=None, rep=None, freq=None, pres=None, ids=None, vals=None, mask=None,
           kind=np.float64):
    """The four rules in `kind`, one rounding per step; returns (x, argmax)."""
    x = np.array(x, kind)
    B, V = x.shape
    for b in range(B):
        if history is not None:
            L = history.shape[1]
            n = L if total is None else min(max(int(total[b]), 0), L)
            p = 0 if prompt is None else max(int(prompt[b]), 0)
            h = history[b, :n].astype(np.int64)
            fine = (h >= 0) & (h < V)
            written = (np.arange(n) >= p) & fine
            seen = np.bincount(h[fine], minlength=V) > 0
            count = np.bincount(h[written], minlength=V)
            with np.errstate(all="ignore"):
                if rep is not None:
                    r = kind(rep[b])
                    x[b] = np.where(seen, np.where(x[b] > 0, x[b] / r, x[b] * r), x[b])
                if freq is not None:
                    x[b] = np.where(count > 0, x[b] - kind(freq[b]) * count.astype(kind), x[b])
                if pres is not None:
                    x[b] = np.where(count > 0, x[b] - kind(pres[b]), x[b])
        if ids is not None:
            last = {int(i): kind(v) for i, v in zip(ids[b], vals[b]) if 0 <= i < V}
            for i, v in last.items():
                with np.errstate(all="ignore"):
                    x[b, i] = x[b, i] + v
        if mask is not None:
            w = mask[b].astype(np.int64) & 0xFFFFFFFF
            t = np.arange(V)
            x[b][(w[t // 32] >> (t % 32)) & 1 == 0] = -np.inf
    y = np.where(np.isnan(x), -np.inf, x)
    best = y.argmax(1).astype(np.int32)  # the lowest of equals
    return x, np.where(y.max(1) > -np.inf, best, -1).astype(np.int32)
