"""Linear layers on 4-bit weights where the result is exact, compared for equality: sums
whose every partial sum fp32 holds, in any order. One wrong term, value or weight anywhere
shows, which a bound on rounding errors over thousands of products cannot promise."""

from __future__ import annotations

import numpy as np
import pytest

import helpers
import narrow
import test_gpu_mx4 as mx4

F = np.float32
# every kernel: 1-4 rows, X too long for 4 rows' LDS, 5-64 rows, the GEMM
ROWS = [1, 2, 3, 4, 5, 16, 17, 32, 33, 64, 65, 130, 260]
SHAPES = [(40, 4096), (333, 1000), (70, 12345), (1500, 4128)]


def third_term_pairs(rng, M, N, K):
    """X with up to eight pairs (x, -x') a row 32 apart, where x' is x without its third
    bf16 term, and W whose columns 32 apart are equal: y is the third terms' part alone.

    x is a multiple of 2^-17 below 1.13 and weights are +-0.5 and 1, so products are
    multiples of 2^-18 and their magnitudes' sum is below 16 1.13 = 18.1 (twice that under
    gains of 1 and 2): every partial sum fits 24 bits."""
    nb = -(-K // 32)
    pairs = (K - 1) // 64 + 1 if K % 64 > 32 else K // 64  # pairs of blocks, the last one in part
    codes = rng.choice(np.array([0x22, 0x2A, 0xA2, 0xAA], np.uint8), (N, nb, 16))  # +-1
    scales = rng.integers(126, 128, (N, nb)).astype(np.uint8)
    odd = np.arange(1, nb, 2)
    codes[:, odd] = codes[:, odd - 1]
    codes = codes.reshape(N, -1)
    scales[:, odd] = scales[:, odd - 1]
    X = np.zeros((M, K), F)
    for m in range(M):
        at = rng.choice(pairs, min(8, pairs), replace=False)
        at[:2] = [0, pairs - 1] if pairs > 1 else at[:2]
        at = np.unique(at)
        last = K - 64 * at - 33  # the highest place whose partner is in the row
        k = 64 * at + np.minimum(rng.integers(0, 32, at.size), last)
        n = at.size
        x = (1 + rng.integers(0, 16, n) * 2.0**-7 + 2.0**-8 + rng.integers(0, 127, n) * 2.0**-15
             + rng.integers(1, 4, n) * 2.0**-17).astype(F)
        X[m, k] = x
        X[m, k + 32] = -two_terms(x)
    assert (X != 0).any(1).all()
    return X, codes, scales


def two_terms(x):
    """x without what its first two bf16 terms (truncations) leave."""
    top = lambda v: (v.view(np.uint32) & np.uint32(0xFFFF0000)).view(F)  # noqa: E731
    h = top(np.ascontiguousarray(x, F))
    return h + top(x - h)


def test_a_dropped_third_term_shows_in_every_element():
    rng = np.random.default_rng(1)
    for N, K in SHAPES:
        X, codes, scales = third_term_pairs(rng, 6, N, K)
        W = narrow.mx4_decode(codes, scales, K)
        y, a = narrow.linear64(X, W)
        assert (y != 0).mean() > 0.8 and 2 * a.max() * 2**18 <= 2**24
        assert np.array_equal(y, y.astype(F))
        y2, _ = narrow.linear64(two_terms(X.reshape(-1)).reshape(X.shape), W)
        assert (y2 == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M", ROWS)
def test_third_terms(gpu, M):
    """Plain, and with RMSNorm and gains of 1 and 2: the sums stay exact, so what is left is
    the scale's error: 16 squares and their sums, the mean, the root and the product, below
    40 u."""
    for N, K in SHAPES:
        rng = np.random.default_rng(M + N + K)
        X, codes, scales = third_term_pairs(rng, M, N, K)
        W = narrow.mx4_decode(codes, scales, K)
        y, _ = narrow.linear64(X, W)
        assert np.array_equal(mx4.linear(gpu, X, codes, scales, N), y), f"{M} x {N} x {K}"
        g = np.repeat(rng.integers(1, 3, -(-K // 64)), 64)[:K].astype(F)
        got = mx4.linear(gpu, X, codes, scales, N, g, True)
        y, _ = narrow.linear64(X, W, g, mx4.EPS)
        helpers.assert_within(got, y, 40 * helpers.U32 * np.abs(y), f"RMSNorm {M} x {N} x {K}")


@pytest.mark.gpu
@pytest.mark.parametrize("M", ROWS)
def test_every_product_once(gpu, M):
    """Dense rows of -3 .. 3 under one scale: multiples of 0.5 below 3 6 K."""
    for N, K in SHAPES:
        rng = np.random.default_rng(M + N + K)
        X = rng.integers(-3, 4, (M, K)).astype(F)
        codes, _ = mx4.weights(rng, N, K)
        scales = np.full((N, -(-K // 32)), 127, np.uint8)
        y, a = narrow.linear64(X, narrow.mx4_decode(codes, scales, K))
        assert a.max() * 2 <= 2**24
        assert np.array_equal(mx4.linear(gpu, X, codes, scales, N), y), f"{M} x {N} x {K}"


# scale byte, exponent of x: weights below bf16's normal range, near fp32's largest values,
# and activations below the normal range themselves
EDGES = [(0, 60), (1, 100), (4, 100), (20, 60), (59, 40), (60, 0), (181, -30), (230, -80), (250, -100),
         (251, -110), (252, -110), (227, -128), (240, -126), (252, -131)]


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 3, 6, 20, 50, 70, 200])
def test_first_and_last_scale_bytes(gpu, M):
    """x of -3 .. 3 times 2^ex and all codes under one scale (at 252 the largest weight is
    6 2^125, finite): sums of multiples of one power of two, exact."""
    N, K = 50, 300
    for byte, ex in EDGES:
        rng = np.random.default_rng(M + byte)
        X = np.ldexp(rng.integers(-3, 4, (M, K)), ex).astype(F)
        codes, _ = mx4.weights(rng, N, K)
        scales = np.full((N, -(-K // 32)), byte, np.uint8)
        y, _ = narrow.linear64(X, narrow.mx4_decode(codes, scales, K))
        assert np.array_equal(mx4.linear(gpu, X, codes, scales, N), y), f"scale {byte}, x 2^{ex}"


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 3, 6, 70])
def test_weights_past_fp32(gpu, M):
    """Values of 2^128 and more (bytes 253 and 254) are infinities: what they enter is
    infinite or NaN, and nothing else is touched."""
    rng = np.random.default_rng(M)
    N, K = 40, 200
    X = rng.integers(1, 4, (M, K)).astype(F)
    codes, _ = mx4.weights(rng, N, K)
    scales = np.full((N, -(-K // 32)), 127, np.uint8)
    clean, _ = narrow.linear64(X, narrow.mx4_decode(codes, scales, K))
    codes[[3, 20], 7] = [0x70, 0x06]  # 6 at place 15, 4 at place 14
    scales[3, 0], scales[20, 0] = 254, 253
    codes[20, :7], codes[20, 8:16] = 0, 0
    codes[20, 7] = 0x06
    got = mx4.linear(gpu, X, codes, scales, N)
    rest = np.delete(np.arange(N), [3, 20])
    assert np.array_equal(got[:, rest], clean[:, rest])
    assert not np.isfinite(got[:, [3, 20]]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 3, 6, 20, 70])
def test_activations_near_the_least_subnormal(gpu, M):
    """Bits below 2^-133 are dropped, nothing above them: weights of 2^100 make both show."""
    rng = np.random.default_rng(M)
    N, K = 30, 200
    X = np.ldexp(rng.integers(-(1 << 10), 1 << 10, (M, K)), -140).astype(F)
    codes = np.full((N, -(-K // 32) * 16), 0x22, np.uint8)
    codes[:, rng.integers(0, K // 2, 40)] = 0x0A  # some -1, some zeros
    scales = np.full((N, -(-K // 32)), 227, np.uint8)
    kept = np.trunc(np.ldexp(X.astype(np.float64), 133)) * 2.0**-133
    y, _ = narrow.linear64(kept, narrow.mx4_decode(codes, scales, K))
    assert np.array_equal(mx4.linear(gpu, X, codes, scales, N), y)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [65, 70, 129, 300])
def test_special_values_in_the_gemm(gpu, M):
    mx4.test_linear_special_values(gpu, M)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 3, 6, 20, 63, 64, 65, 128])
@pytest.mark.parametrize("K", [1 << 23, (1 << 23) - 5])
def test_longest_rows_exactly(gpu, M, K):
    """X is zero but for whole numbers at a few places of each row: its first and last ones,
    both sides of units, chunks and of the byte offsets 2^31 and 2^32 of X."""
    rng = np.random.default_rng(M)
    N, nb = 3, -(-K // 32)
    codes, _ = mx4.weights(rng, N, K)
    scales = rng.integers(125, 130, (N, nb)).astype(np.uint8)
    dx = gpu.empty((M, K), F)
    dx.fill_bytes(0)
    dc, ds = gpu.upload(codes), gpu.upload(scales)
    y = gpu.empty((M, N), F)
    for places in range(2):
        want = np.zeros((M, N))
        spots = []
        for m in range(M):
            k = np.unique(np.r_[0, K - 1, rng.integers(0, K, 6), rng.integers(1, K // 256, 3) * 256 - places,
                                K - 1 - rng.integers(0, 300, 3)])
            for edge in ((1 << 29) - m * K, (1 << 30) - m * K):  # in floats
                if 0 < edge < K:
                    k = np.unique(np.r_[k, edge - 1, edge])
            x = rng.integers(1, 4, k.size).astype(F) * rng.choice([-1, 1], k.size)
            b = codes[:, k // 2]
            c = np.where(k % 2, b >> 4, b & 15)
            w = np.where(c & 8, -1.0, 1.0) * narrow.E2M1[c & 7] * np.exp2(scales[:, k // 32].astype(float) - 127)
            want[m] = w @ x
            spots += [(m * K + i, v) for i, v in zip(k, x.astype(F))]
        for at, v in spots:
            one = np.array([v], F)
            gpu.call("eng_memcpy_h2d", dx.ptr + 4 * int(at), one.ctypes.data, 4)
        y.fill_bytes(0xFF)
        gpu.call("eng_linear_mx4w_nk", dx.ptr, dc.ptr, ds.ptr, y.ptr, M, N, K, None)
        gpu.sync()
        assert np.array_equal(y.download(), want)
        zero = np.zeros(1, F)
        for at, _ in spots:
            gpu.call("eng_memcpy_h2d", dx.ptr + 4 * int(at), zero.ctypes.data, 4)
    for d in (dx, dc, ds, y):
        d.free()
