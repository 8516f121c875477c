"""Float64 statements of the long-context operators (attention with a window, over a
shared prefix, beam selection, cache reordering), in numpy, for the tests."""

from __future__ import annotations

import numpy as np

import narrow
from helpers import U16, U32

BLOCK = 32


# --------------------------------------------------------------------- caches
class Cache:
    """K and V caches of B sequences on host and device: fp16, or e4m3 with scales.
    Everything at and behind `lens` is NaN (and so are the scales of unreached blocks)."""

    def __init__(self, gpu, rng, kind, B, G, room, D, lens, sigma=1.0, edit=None):
        self.kind, self.room = kind, room
        nb = -(-room // BLOCK)
        k, v = (sigma * rng.standard_normal((2, B, G, room, D))).astype(np.float16)
        if edit is not None:
            edit(k, v)
        self.scales = []
        if kind == "f16":
            self.raw = [k.copy(), v.copy()]
            for b, n in enumerate(lens):
                for a in self.raw:
                    a[b, :, max(int(n), 0):] = np.nan
            self.values = [a.astype(np.float64) for a in self.raw]
            self.vmax = np.nanmax(np.abs(np.where(np.isfinite(self.values[1]), self.values[1], 0)), (2, 3))
            self.dev = [gpu.upload(a.view(np.uint16)) for a in self.raw]
            return
        self.raw = []
        for x in (k, v):
            p = np.zeros((B, G, nb * BLOCK, D))
            p[:, :, :room] = x
            p = p.reshape(B, G, nb, BLOCK, D)
            top = np.abs(np.where(np.isfinite(p), p, 0)).max((3, 4))
            s = np.exp2(np.clip(np.ceil(np.log2(np.where(top > 0, top, 1e-9) / 448)), -15, 8))
            c = narrow.e4m3_encode(p / s[..., None, None]).reshape(B, G, nb * BLOCK, D)[:, :, :room].copy()
            s = s.astype(np.float32)
            for b, n in enumerate(lens):
                n = max(int(n), 0)
                c[b, :, n:] = 0xFF
                s[b, :, -(-n // BLOCK):] = np.nan
            self.raw.append(c)
            self.scales.append(s)
        self.values = [narrow.kv_values(c, s) for c, s in zip(self.raw, self.scales)]
        # weights of 8-bit values are rounded as multipliers of their codes
        self.vmax = 448.0 * np.nanmax(np.where(np.isnan(self.scales[1]), 0, self.scales[1]), 2)
        self.dev = [gpu.upload(a) for a in (*self.raw, *self.scales)]

    @property
    def ptrs(self):
        return [d.ptr for d in self.dev]


# ------------------------------------------------------------------ attention
def attend_rows(q, k, v, vmax, scale):
    """(y, bound) of one query row q [D] over keys k, v [n, D] that it sees.

    u = 2^-24. Scores: q, K and the codes are exact in fp16, products exact, sums fp32:
    e_j = (D + 1) u |scale| sum |q k|. Weights 2^(s - m): roundings of the scale, the
    product and the difference and the hardware's exp2 and log2, 4 u (1.5 max |s| + 32)
    + 40 u relative; each rounded to fp16 for its product with V, 2^-11 relative and,
    where fp16 is subnormal, 2^-32 of the largest absolute, n 2^-32 vmax (vmax: the
    largest value of V, or 448 times its largest scale). The fp32 sums and the merge of
    partial states (n + 36) u; the output's rounding 2^-11 |y| + 2^-25."""
    n, D = k.shape
    if n == 0:
        return np.zeros(D), np.zeros(D)
    with np.errstate(invalid="ignore"):
        s = k @ q * scale
        w = np.exp(s - s.max())
        y = (w @ v) / w.sum()
    if not np.isfinite(s).all():
        return np.full(D, np.nan), np.zeros(D)
    fin = np.where(np.isfinite(v), v, 0)
    e = (D + 1) * U32 * abs(scale) * (np.abs(k) @ np.abs(q))
    mag = (w @ np.abs(fin)) / w.sum()
    rel = 2 * e.max() + 4 * U32 * (1.5 * np.abs(s).max() + 32) + 40 * U32 + (n + 36) * U32 + U16
    return y, U16 * np.abs(np.where(np.isfinite(y), y, 0)) + 2.0**-25 + n * 2.0**-32 * vmax + 2 * rel * mag


def seen_keys(p, window, sinks, max_len):
    """Indices of the keys that a query at position p sees."""
    j = np.arange(min(p + 1, max_len))
    return j if window == 0 else j[(j > p - window) | (j < sinks)]


def window64(q, cache, pos, n_new, window, sinks, max_len, scale, rows=None):
    """{(b, i, h): (y, bound)} for the queries that are there; `rows` picks tokens."""
    B, S, H, D = q.shape
    G = cache.values[0].shape[1]
    out = {}
    for b in range(B):
        n = S if n_new is None else min(int(n_new[b]), S)
        if pos[b] < 0:
            continue
        for i in range(n):
            if rows is not None and i not in rows:
                continue
            j = seen_keys(int(pos[b]) + i, window, sinks, max_len)
            for h in range(H):
                g = h // (H // G)
                out[b, i, h] = attend_rows(q[b, i, h], cache.values[0][b, g, j], cache.values[1][b, g, j],
                                           cache.vmax[b, g], scale)
    return out


def prefix64(q, prefix, plen, own, lens, scale):
    """{(b, h): (y, bound)}."""
    B, H, D = q.shape
    G = own.values[0].shape[1]
    per = B // len(plen)
    out = {}
    for b in range(B):
        p = b // per
        np_, n = max(int(plen[p]), 0), max(int(lens[b]), 0)
        for h in range(H):
            g = h // (H // G)
            k = np.concatenate((prefix.values[0][p, g, :np_], own.values[0][b, g, :n]))
            v = np.concatenate((prefix.values[1][p, g, :np_], own.values[1][b, g, :n]))
            vmax = max(prefix.vmax[p, g], own.vmax[b, g])
            out[b, h] = attend_rows(q[b, h], k, v, vmax, scale)
    return out


def check(got, want, what):
    """Every row of `want` ({index: (y, bound)}) in `got`, infinities and NaN in place."""
    for at, (y, bound) in want.items():
        g = got[at].astype(np.float64)
        fin = np.isfinite(y)
        assert np.array_equal(np.isnan(g), np.isnan(y)), f"{what} {at}: NaN"
        assert np.array_equal(g[~fin & ~np.isnan(y)], y[~fin & ~np.isnan(y)]), f"{what} {at}: infinities"
        err = np.abs(g[fin] - y[fin])
        bad = err > bound[fin]
        assert not bad.any(), (f"{what} {at}: error {err[bad].max():.3g} over a bound of "
                               f"{bound[fin][bad].min():.3g}, {bad.sum()} of {bad.size}")


# ---------------------------------------------------------------- beam search
def select64(logits, scores, finished, n_out, eos):
    """(scores, parent, token, finished) of one group: logits [beams, V] float64."""
    beams, V = logits.shape
    cand = np.full((beams, V), -np.inf)
    order = np.zeros((beams, V))  # candidates of a beam compare by their logits
    for b in range(beams):
        if not np.isfinite(scores[b]):
            continue
        if finished is not None and finished[b]:
            cand[b, eos] = scores[b]
            continue
        x = logits[b]
        if np.isnan(x).any() or x.max() in (np.inf, -np.inf):
            continue
        lse = x.max() + np.log(np.exp(x - x.max()).sum())
        cand[b] = scores[b] + (x - lse)
        order[b] = x
    beam = np.repeat(np.arange(beams), V)
    token = np.tile(np.arange(V), beams)
    at = np.lexsort((token, -order.reshape(-1), beam, -cand.reshape(-1)))
    at = at[:n_out]
    s, p, t = cand.reshape(-1)[at], beam[at], token[at]
    f = np.array([(finished is not None and bool(finished[b])) or u == eos for b, u in zip(p, t)])
    return s, p, t, f
