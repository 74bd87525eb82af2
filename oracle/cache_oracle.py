"""fp64 restatements of the query/key norm + rotation, of appending to a paged cache and of
attention over an 8-bit paged cache (numpy; the checker of their kernels only).

The rotation is the reference's rope (mlx_primitives/kernels/rope.py:451-496), the pools and
tables are those of its paged_attention (mlx_primitives/cache/paged_attention.py:44-320); norms
and 8-bit codes have no counterpart there and are stated from their definitions.
"""

from __future__ import annotations

import math

import numpy as np

QMAX = {"e4m3": 448.0, "int8": 127.0}


def norm_rope(x, weight, cos, sin, pos, eps=1e-6):
    """x (B, S, H, D), weight (D,) or None, cos/sin (n, D/2) or None, pos (B, S) ints: rows of
    negative position are zeros, rows past the tables NaN."""
    x = np.asarray(x, dtype=np.float64)
    y = x.copy()
    if weight is not None:
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    if cos is not None:
        n, h = cos.shape
        at = np.clip(pos, 0, n - 1)
        c = np.asarray(cos, np.float64)[at][:, :, None, :]
        s = np.asarray(sin, np.float64)[at][:, :, None, :]
        y = np.concatenate((y[..., :h] * c - y[..., h:] * s, y[..., :h] * s + y[..., h:] * c), -1)
        y[pos >= n] = np.nan
    y[pos < 0] = 0.0
    return y


def norm_rope_grad(gy, x, weight, cos, sin, pos, eps=1e-6):
    """(dx, dweight, sum of |terms| of dweight) of norm_rope for the output gradient gy."""
    x = np.asarray(x, dtype=np.float64)
    g = np.asarray(gy, dtype=np.float64).copy()
    live = (pos >= 0)[:, :, None, None]
    g = np.where(live, g, 0.0)
    x = np.where(live, x, 0.0)
    if cos is not None:
        n, h = cos.shape
        at = np.clip(pos, 0, n - 1)
        c = np.asarray(cos, np.float64)[at][:, :, None, :]
        s = np.asarray(sin, np.float64)[at][:, :, None, :]
        g = np.concatenate((g[..., :h] * c + g[..., h:] * s, g[..., h:] * c - g[..., :h] * s), -1)
    if weight is None:
        return g, None, None
    w = np.asarray(weight, np.float64)
    r = np.zeros(x.shape[:-1] + (1,))  # of padding rows: they add nothing, eps = 0 or not
    np.divide(1.0, np.sqrt((x * x).mean(-1, keepdims=True) + eps), out=r, where=live)
    xh = x * r
    terms = g * xh
    gw = g * w
    dx = r * (gw - xh * (gw * xh).mean(-1, keepdims=True))
    return np.where(live, dx, 0.0), terms.sum((0, 1, 2)), np.abs(terms).sum((0, 1, 2))


def round_e4m3(x):
    """Nearest e4m3 value (ties to even) of x clamped to +-448, in fp64; NaN stays."""
    x = np.clip(np.asarray(x, dtype=np.float64), -448.0, 448.0)
    _, e = np.frexp(x)
    step = np.exp2(np.maximum(e - 1, -6).astype(np.float64) - 3)
    return np.round(x / step) * step


def round_int8(x):
    return np.round(np.clip(np.nan_to_num(np.asarray(x, dtype=np.float64), nan=0.0,
                                          posinf=np.inf, neginf=-np.inf), -127.0, 127.0))


def least_scale(amax, kind):
    """The least power of two s >= 2^-126 with amax <= qmax * s."""
    s = 2.0 ** -126
    while amax > QMAX[kind] * s:
        s *= 2.0
    return s


def append(new, pool, tables, ctx, new_lens, scales=None, kind=None):
    """Writes new (B, S, Hk, D) into a copy of pool (blocks, block, Hk, D); with `kind`, pool
    holds code values and scales (blocks, Hk) is copied and updated too.  Returns (pool, scales,
    written): `written` marks the rows that received tokens."""
    pool = np.array(pool, dtype=np.float64)
    scales = None if scales is None else np.array(scales, dtype=np.float64)
    written = np.zeros(pool.shape[:2], dtype=bool)
    nblk, block, Hk, _ = pool.shape
    rnd = None if kind is None else {"e4m3": round_e4m3, "int8": round_int8}[kind]
    for b in range(new.shape[0]):
        pos = int(ctx[b]) + np.arange(min(max(int(new_lens[b]), 0), new.shape[1]))
        for slot in sorted(set((pos[pos >= 0] // block).tolist())):
            if slot >= tables.shape[1] or not 0 <= tables[b, slot] < nblk:
                continue
            blk = int(tables[b, slot])
            src = np.nonzero((pos >= 0) & (pos // block == slot))[0]
            rows = pos[src] % block
            written[blk, rows] = True
            if kind is None:
                pool[blk, rows] = new[b, src]
                continue
            for h in range(Hk):
                x = np.asarray(new[b, src, h], dtype=np.float64)
                fin = np.abs(x[np.isfinite(x)])
                s = least_scale(fin.max() if fin.size else 0.0, kind)
                if rows[0] > 0:
                    old = scales[blk, h]
                    s = max(s, old)
                    if s != old:
                        pool[blk, :rows[0], h] = rnd(pool[blk, :rows[0], h] * (old / s))
                scales[blk, h] = s
                pool[blk, rows, h] = rnd(x / s)
    return pool, scales, written


def quantized_attention(q, k_pool, v_pool, k_scales, v_scales, tables, ctx, query_lens=None,
                        scale=None, causal=True, window=None, slopes=None):
    """(o, absolute o, floor): softmax-weighted sums of v and of |v|, and max_t(w_t vs_t) times
    the sum of |codes| (what an absolute error of the weights multiplies).  q (B, S, H, D); pools
    hold code values.  Query i of n = query_lens[b] sits at ctx[b] - n + i; rows without keys are zeros."""
    q = np.asarray(q, dtype=np.float64)
    B, S, H, D = q.shape
    nblk, block, Hk, _ = k_pool.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    o, ao, floor = (np.zeros_like(q) for _ in range(3))
    for b in range(B):
        n = S if query_lens is None else min(max(int(query_lens[b]), 0), S)
        t = np.arange(max(min(int(ctx[b]), tables.shape[1] * block), 0))
        if t.size == 0 or n == 0:
            continue
        ids = tables[b, t // block]
        there = (ids >= 0) & (ids < nblk)
        t, ids = t[there], ids[there]
        k = np.asarray(k_pool, np.float64)[ids, t % block] * np.asarray(k_scales, np.float64)[ids][..., None]
        codes = np.asarray(v_pool, np.float64)[ids, t % block]
        vs = np.asarray(v_scales, np.float64)[ids]
        v = codes * vs[..., None]
        for i in range(n):
            p = int(ctx[b]) - n + i
            ok = np.ones(t.size, dtype=bool)
            if causal:
                ok &= t <= p
            if window is not None:
                ok &= np.abs(t - p) <= window
            if not ok.any():
                continue
            for h in range(H):
                s = (k[ok, h // (H // Hk)] @ q[b, i, h]) * scale
                if slopes is not None:
                    s = s + slopes[h] * (t[ok] - p)
                w = np.exp(s - s.max())
                w /= w.sum()
                o[b, i, h] = w @ v[ok, h // (H // Hk)]
                ao[b, i, h] = w @ np.abs(v[ok, h // (H // Hk)])
                floor[b, i, h] = (w * np.abs(vs[ok, h // (H // Hk)])).max() * \
                    np.abs(codes[ok, h // (H // Hk)]).sum(0)
    return o, ao, floor
