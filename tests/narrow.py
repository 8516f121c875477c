"""Float64 statements of the 4-bit weight and 8-bit cache formats and of the
operators on them, in numpy, for the tests."""

from __future__ import annotations

import numpy as np

from helpers import U16, U32

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# e4m3 magnitudes by code: 0 .. 126 are finite, 127 is NaN
E4M3 = np.array([(m / 8.0) * 2.0**-6 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7)
                 for e in range(16) for m in range(8)][:127])
BLOCK = 32


def _nearest(x, grid):
    """Code of the value of `grid` nearest to each |x|, ties to the even code."""
    a = np.abs(x)
    mid = (grid[1:] + grid[:-1]) / 2
    lo = np.searchsorted(mid, a, side="left")   # a tie stays below
    hi = np.searchsorted(mid, a, side="right")  # a tie goes above
    return np.where(lo == hi, lo, np.where(lo % 2 == 0, lo, hi))


# ------------------------------------------------------------------ weights
def mx4_encode(W):
    """W [rows, cols] -> (codes [rows, 16 nb] u8, scales [rows, nb] u8)."""
    W = np.asarray(W, np.float64)
    rows, cols = W.shape
    nb = -(-cols // BLOCK)
    p = np.zeros((rows, nb * BLOCK))
    p[:, :cols] = W
    p = p.reshape(rows, nb, BLOCK)
    bad = ~np.isfinite(p).all(-1)
    q = np.where(bad[..., None], 0.0, p)
    top = np.abs(q).max(-1)
    _, ex = np.frexp(top)  # top = f 2^ex, f in [0.5, 1)
    e = np.where(top == 0, -127, np.clip(ex - 1 - 2, -127, 127))
    code = _nearest(np.ldexp(q, -e[..., None]), E2M1) + 8 * np.signbit(q)
    code = np.where(bad[..., None], 0, code).astype(np.uint8)
    scales = np.where(bad, 255, e + 127).astype(np.uint8)
    codes = code[..., 0::2] | (code[..., 1::2] << 4)
    return codes.reshape(rows, -1).astype(np.uint8), scales


def mx4_decode(codes, scales, cols):
    rows, nb = scales.shape
    c = np.stack((codes & 15, codes >> 4), -1).reshape(rows, nb, BLOCK)
    v = np.where(c & 8, -1.0, 1.0) * E2M1[c & 7]
    v = np.ldexp(v, scales.astype(np.int64)[..., None] - 127)
    v = np.where((scales == 255)[..., None], np.nan, v)
    return v.reshape(rows, -1)[:, :cols]


def linear64(x, W, g=None, eps=None):
    """(y, sum |x w|) of x . W^T, with the RMSNorm of the rows if eps is given."""
    x = np.asarray(x, np.float64)
    s = np.ones((x.shape[0], 1))
    if eps is not None:
        s = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        if g is not None:
            x = x * np.asarray(g, np.float64)
    return s * (x @ W.T), s * (np.abs(x) @ np.abs(W).T)


def linear_bound(y, a, K, rms):
    """Products are exact and each x is three terms, so a sum has 3 K of them (and
    up to 64 partial sums), rounded one by one to fp32 (matrix instructions round
    a running sum once per 32 products, within 2 u): |error| <= 2 (3 K + 64) u a;
    as a random walk 16 sqrt(3 K + 64) u a, the smaller of the two. RMSNorm adds
    its scale's (K / 2 + 4) u |y|, its square root's halving included, and one
    rounding of x g for each product, 1 u a."""
    t = 3 * K + 64
    b = np.minimum(2 * t, 16 * np.sqrt(t)) * U32 * a + U32 * np.abs(y)
    if rms:
        b = b + (K / 2 + 4) * U32 * np.abs(y) + U32 * a
    return b


# -------------------------------------------------------------------- cache
def e4m3_encode(x):
    """Nearest e4m3 codes; NaN and infinities become NaN codes (0x7f)."""
    x = np.asarray(x, np.float64)
    fin = np.isfinite(x)
    c = _nearest(np.where(fin, x, 0.0), E4M3)
    return np.where(fin, c | (np.signbit(x) * 128), 0x7F).astype(np.uint8)


def e4m3_decode(c):
    c = np.asarray(c, np.uint8)
    mag = np.append(E4M3, np.nan)[c & 127]
    return np.where(c & 128, -mag, mag)


def kv_scale(top):
    """Least power of two in [2^-15, 2^8] with top <= 448 times it."""
    for e in range(-15, 9):
        if top <= 448.0 * 2.0**e:
            return 2.0**e
    raise AssertionError(f"no scale for {top}")


def kv_write(new, cache, scale, pos, n_new):
    """In place: new [B, S, G, D] (float64) into cache [B, G, L, D] u8 and scale
    [B, G, nb] float32."""
    B, S, G, D = new.shape
    L = cache.shape[2]
    for b in range(B):
        n = S if n_new is None else min(int(n_new[b]), S)
        p = int(pos[b])
        if p < 0 or n <= 0:
            continue
        end = min(p + n, L)
        for first in range(p // BLOCK * BLOCK, end, BLOCK):
            lo, hi = max(p, first), min(end, first + BLOCK)
            if lo >= hi:
                continue
            for h in range(G):
                x = new[b, lo - p:hi - p, h]
                fin = np.abs(x[np.isfinite(x)])
                s = kv_scale(fin.max() if fin.size else 0.0)
                k = first // BLOCK
                if lo > first:
                    old = float(scale[b, h, k])
                    s = max(s, old)
                    if s > old:
                        was = e4m3_decode(cache[b, h, first:lo])
                        cache[b, h, first:lo] = e4m3_encode(was * (old / s))
                cache[b, h, lo:hi] = e4m3_encode(x / s)
                scale[b, h, k] = s


def kv_values(cache, scale):
    B, G, L, D = cache.shape
    s = np.repeat(scale.astype(np.float64), BLOCK, axis=2)[:, :, :L, None]
    return e4m3_decode(cache) * s


def same_codes(a, b):
    """Equal e4m3 bytes, any two NaN codes being equal."""
    return ((a == b) | (((a & 127) == 127) & ((b & 127) == 127))).all()


def attend64(q, kc, vc, ks, vs, lens, scale):
    """(y, bound) of the decode attention, q [B, H, D] float64; lens already within
    the caches.

    u = 2^-24. Scores carry e_j = (D + 1) u scale sum |q k| (q and the codes are
    exact in fp16, products exact, sums fp32; the block's scale is a power of two);
    weights 2^(s' - m) with s' = fma(score, scale log2 e, log2 v scale): roundings
    of the scale, the sum, the difference and the hardware's exp2 and log2, 4 u (1.5
    max |s| + 32) + 40 u relative; V times two fp16 terms of a weight 4 u relative
    and 2^-32 absolute of the largest, so L 2^-32 448 max v scale; the fp32 sums (L
    + 36) u; the output's rounding 2^-11 |y| + 2^-25."""
    B, H, D = q.shape
    G = kc.shape[1]
    y = np.zeros((B, H, D))
    bound = np.zeros((B, H, D))
    for b in range(B):
        L = int(lens[b])
        if L <= 0:
            continue
        nb = -(-L // BLOCK)
        k64 = kv_values(kc[b:b + 1, :, :nb * BLOCK], ks[b:b + 1, :, :nb])[0][:, :L]
        v64 = kv_values(vc[b:b + 1, :, :nb * BLOCK], vs[b:b + 1, :, :nb])[0][:, :L]
        for h in range(H):
            kh, vh = k64[h // (H // G)], v64[h // (H // G)]
            s = kh @ q[b, h] * scale
            w = np.exp(s - s.max())
            y[b, h] = (w @ vh) / w.sum()
            e = (D + 1) * U32 * abs(scale) * (np.abs(kh) @ np.abs(q[b, h]))
            mag = (w @ np.abs(vh)) / w.sum() + np.abs(y[b, h])
            rel = 2 * e.max() + 4 * U32 * (1.5 * np.abs(s).max() + 32) + 40 * U32 + (L + 36) * U32
            bound[b, h] = (U16 * np.abs(y[b, h]) + 2.0**-25
                           + L * 2.0**-32 * 448 * vs[b, h // (H // G), :nb].max() + rel * mag)
    return y, bound
