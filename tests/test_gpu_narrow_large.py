"""4-bit weights and the 8-bit cache at the sizes where a launch changes shape: more
rows than one pass, more columns than one round of tiles, one slice and many, batches of
many sequences, and matrices whose items pass 32 bits."""

from __future__ import annotations

import numpy as np
import pytest

import helpers
import narrow
from test_gpu_kv_q8 import Cache, attend, check_attend, rows
from test_gpu_mx4 import EPS, check_linear, linear, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K,rms", [
    (1, 200000, 64, True),      # more than 48 tiles for a workgroup on 256 CUs
    (3, 200001, 33, False),
    (1, 100, 20481, True),      # X no longer fits the decode kernel's LDS
    (4, 50, 6000, True),
    (8, 40000, 300, True),      # as many column groups as CUs: one slice
    (40, 100003, 96, False),
    (20, 129, 9000, True),      # few columns: many slices
    (60, 20, 40000, False),
    (100, 300, 5000, True),     # the GEMM with K split
    (65, 64, 20000, True),
    (33000, 24, 40, True),      # two passes of rows
])
def test_linear_launch_shapes(gpu, M, N, K, rms):
    check_linear(gpu, np.random.default_rng(M + N + K), M, N, K, rms)


@pytest.mark.parametrize("M", [1, 4, 5, 20, 50, 70])
@pytest.mark.parametrize("K", [2, 3, 4, 5, 6, 7, 127, 255, 256, 257, 258, 259, 511, 513])
def test_linear_ends_of_rows(gpu, M, K):
    """The last values of a row of X, every way it can end inside four values and a
    unit, with infinities behind the end (the next row's, and gamma's)."""
    rng = np.random.default_rng(1000 * M + K)
    N = 45
    x = rng.standard_normal((M + 1, K)).astype(np.float32)
    x[M] = np.inf
    g = np.append(1 + 0.1 * rng.standard_normal(K), [np.inf] * 8).astype(np.float32)
    codes, scales = weights(rng, N, K)
    dx, dg, dc, ds = (gpu.upload(a) for a in (x, g, codes, scales))
    for rms in (False, True):
        y = gpu.empty((M, N), np.float32)
        if rms:
            gpu.call("eng_rmsnorm_linear_mx4w_nk", dx.ptr, dg.ptr, dc.ptr, ds.ptr, y.ptr, M, N, K, EPS, None)
        else:
            gpu.call("eng_linear_mx4w_nk", dx.ptr, dc.ptr, ds.ptr, y.ptr, M, N, K, None)
        gpu.sync()
        want, a = narrow.linear64(x[:M], narrow.mx4_decode(codes, scales, K), g[:K] if rms else None,
                                  EPS if rms else None)
        helpers.assert_within(y.download(), want, narrow.linear_bound(want, a, K, rms), f"{M} x {K}")


@pytest.mark.parametrize("M,N,K", [(6, 33000, 257), (12, 33000, 259), (40, 50000, 258), (8, 90000, 515)])
def test_linear_ends_of_rows_after_whole_units(gpu, M, N, K):
    check_linear(gpu, np.random.default_rng(K), M, N, K, True)


@pytest.mark.parametrize("M,N,K", [(1, 5, 1 << 23), (6, 3, 1 << 23), (20, 2, (1 << 23) - 5)])
def test_linear_longest_rows(gpu, M, N, K):
    check_linear(gpu, np.random.default_rng(M), M, N, K, M > 1)


def test_linear_passes_of_rows_agree_with_single_calls(gpu):
    """Rows on both sides of a pass's end equal the same rows in a call of their own
    size class, within the bound (the order of the sums may differ)."""
    rng = np.random.default_rng(5)
    N, K, M = 16, 64, 32768 + 70
    x = rng.standard_normal((M, K)).astype(np.float32)
    codes, scales = weights(rng, N, K)
    got = linear(gpu, x, codes, scales, N)
    at = np.r_[0:3, 32766:32771, M - 2:M]
    y, a = narrow.linear64(x[at], narrow.mx4_decode(codes, scales, K))
    helpers.assert_within(got[at], y, narrow.linear_bound(y, a, K, False), "rows at the pass's end")
    assert np.isfinite(got).all()


def test_quantize_and_back_past_32_bits_of_items(gpu):
    """2^29 + 3 rows of two blocks: eight words of codes a row, over 2^32 in all. The
    first and the last rows are checked."""
    rng = np.random.default_rng(6)
    R, cols = (1 << 29) + 3, 33
    src, codes = gpu.malloc(R * cols * 2), gpu.malloc(R * 32)
    scales, back = gpu.malloc(R * 2), gpu.malloc(R * cols * 2)
    try:
        n = 64
        W = rng.standard_normal((2 * n, cols)).astype(np.float16)
        gpu.call("eng_memset", src, 0, R * cols * 2)
        gpu.call("eng_memcpy_h2d", src, W.ctypes.data, n * cols * 2)
        gpu.call("eng_memcpy_h2d", src + (R - n) * cols * 2, W[n:].ctypes.data, n * cols * 2)
        gpu.call("eng_mx4_quantize_f16", src, codes, scales, R, cols, None)
        gpu.call("eng_mx4_dequantize_f16", codes, scales, back, R, cols, None)
        gpu.sync()
        wc, ws = narrow.mx4_encode(W)
        v = narrow.mx4_decode(wc, ws, cols).astype(np.float16)
        for half, row in ((slice(0, n), 0), (slice(n, 2 * n), R - n)):
            c, s = np.empty((n, 32), np.uint8), np.empty((n, 2), np.uint8)
            b = np.empty((n, cols), np.float16)
            gpu.call("eng_memcpy_d2h", c.ctypes.data, codes + row * 32, c.nbytes)
            gpu.call("eng_memcpy_d2h", s.ctypes.data, scales + row * 2, s.nbytes)
            gpu.call("eng_memcpy_d2h", b.ctypes.data, back + row * cols * 2, b.nbytes)
            assert np.array_equal(c, wc[half]) and np.array_equal(s, ws[half])
            assert np.array_equal(b, v[half])
    finally:
        for p in (src, codes, scales, back):
            gpu.free(p)


def test_many_sequences(gpu):
    rng = np.random.default_rng(7)
    B, H, G, D, L = 150, 6, 3, 64, 96
    c = Cache(gpu, rng, B, G, L, D)
    S = 40
    pos, n = rng.integers(0, L - 20, B), rng.integers(0, S + 1, B)
    c.write(rows(rng, B, S, G, D), rows(rng, B, S, G, D), np.zeros(B, int), None)
    c.write(rows(rng, B, S, G, D), rows(rng, B, S, G, D, 3.0), np.minimum(pos, S), n)
    c.check()
    q = rng.standard_normal((B, H, D)).astype(np.float16)
    lens = np.maximum(np.minimum(np.minimum(pos, S) + n, L), 1)
    lens[rng.integers(0, B, 20)] = 0
    check_attend(gpu, c, q, lens, L)
    check_attend(gpu, c, q, lens, L, split=3)


def test_splits_that_a_sequence_does_not_reach(gpu):
    """The merge reads the scratch of splits past a sequence's end, whatever an earlier
    call left there: NaN and infinities (of q), then lengths that leave splits, or all of
    them, unused."""
    rng = np.random.default_rng(9)
    B, H, G, D, L = 5, 8, 2, 128, 640
    c = Cache(gpu, rng, B, G, L, D)
    c.write(rows(rng, B, L, G, D), rows(rng, B, L, G, D), np.zeros(B, int), None)
    q = rng.standard_normal((B, H, D)).astype(np.float16)
    for split in (0, 4, 12, 20):
        bad = q.copy()
        bad[:, ::2] = np.nan
        bad[:, 1::2, 3] = np.inf
        attend(gpu, c, bad, np.full(B, L), L, 0.1, split)
        check_attend(gpu, c, q, np.array([0, 1, 33, 320, 640]), L, split=split)


def test_rmsnorm_of_zero_and_of_large_rows(gpu):
    """A row of zeros gives zeros (eps alone under the root), rows up to 1e18 stay
    finite."""
    rng = np.random.default_rng(8)
    for M in (2, 10, 40, 90):
        x = rng.standard_normal((M, 200)).astype(np.float32)
        x[0] = 0
        x[1] *= 1e18
        g = np.ones(200, np.float32)
        codes, scales = weights(rng, 30, 200)
        got = linear(gpu, x, codes, scales, 30, g, True)
        y, a = narrow.linear64(x, narrow.mx4_decode(codes, scales, 200), g, EPS)
        assert (got[0] == 0).all()
        helpers.assert_within(got, y, narrow.linear_bound(y, a, 200, True), f"M = {M}")
