"""GPU tests of 4-bit weights: quantisation, the values back, and linear layers,
through the C-ABI, against float64. Quantisation is exact by definition and is
compared bit for bit; the linear layers' tolerance is narrow.linear_bound."""

from __future__ import annotations

import numpy as np
import pytest

import helpers
import narrow

pytestmark = pytest.mark.gpu
EPS = 1e-5
PAD = 64  # guard bytes behind every output


def out_bytes(gpu, n):
    d = gpu.empty(n + PAD, np.uint8)
    d.fill_bytes(0xA5)
    return d


def take(d, n, dtype, shape):
    a = d.download()
    assert (a[n:] == 0xA5).all(), "bytes behind the output were written"
    return a[:n].view(dtype).reshape(shape)


def quantize(gpu, W, kind, skew=0):
    """(codes, scales) of W (fp32, or fp16 as float16); skew: elements by which the
    source is off the allocation's start."""
    rows, cols = W.shape
    nb = -(-cols // 32)
    flat = np.concatenate([np.zeros(skew, W.dtype), W.reshape(-1)])
    src = gpu.upload(flat.view(np.uint16) if kind == "f16" else flat)
    codes, scales = out_bytes(gpu, rows * nb * 16), out_bytes(gpu, rows * nb)
    gpu.call("eng_mx4_quantize_" + kind, src.ptr + skew * W.itemsize, codes.ptr, scales.ptr, rows,
             cols, None)
    gpu.sync()
    return (take(codes, rows * nb * 16, np.uint8, (rows, nb * 16)),
            take(scales, rows * nb, np.uint8, (rows, nb)))


SHAPES = [(1, 1), (1, 31), (3, 32), (5, 33), (2, 64), (7, 100), (1, 4096), (509, 1023), (33, 4104)]


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_equals_the_definition(gpu, rows, cols, kind):
    rng = np.random.default_rng(rows * 7919 + cols)
    W = (0.02 * rng.standard_normal((rows, cols))).astype(np.float32)
    if kind == "f16":
        W = W.astype(np.float16)
    codes, scales = quantize(gpu, W, kind)
    want = narrow.mx4_encode(W)
    assert np.array_equal(scales, want[1])
    assert np.array_equal(codes, want[0])


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("skew", [1, 3])
def test_quantize_unaligned_source(gpu, kind, skew):
    rng = np.random.default_rng(skew)
    W = rng.standard_normal((9, 96)).astype(np.float16 if kind == "f16" else np.float32)
    codes, scales = quantize(gpu, W, kind, skew)
    want = narrow.mx4_encode(W)
    assert np.array_equal(scales, want[1]) and np.array_equal(codes, want[0])


def test_quantize_edge_values(gpu):
    f = np.float32
    rows = []
    rows.append(np.zeros(64, f))
    rows.append(np.full(64, -0.0, f))
    # every tie and its neighbours, at a scale of 2^0 (amax 4 .. 7.99)
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], f)
    t = np.concatenate([ties, np.nextafter(ties, f(9)), np.nextafter(ties, f(0)), -ties, [6, 7.5, 7.99, 4]])
    rows.append(np.resize(t, 64).astype(f))
    for e in (-149, -140, -130, -127, -126, -125, -124, 0, 100, 125, 127):
        m = np.resize(t, 64).astype(np.float64)
        with np.errstate(over="ignore"):
            rows.append(np.clip(np.ldexp(m / 8, e), -3.4e38, 3.4e38).astype(f))
    rows.append(np.full(64, np.finfo(f).max, f))
    rows.append(np.full(64, np.finfo(f).tiny / 2**20, f))
    for v in (np.nan, np.inf, -np.inf):
        r = np.ones(64, f)
        r[37] = v
        rows.append(r)
    W = np.stack(rows)
    codes, scales = quantize(gpu, W, "f32")
    want = narrow.mx4_encode(W)
    assert np.array_equal(scales, want[1])
    assert np.array_equal(codes, want[0])
    assert scales[-1].tolist() == [127 - 2, 255]  # only the block that holds it


def test_quantize_every_half(gpu):
    bits = np.arange(65536, dtype=np.uint32).astype(np.uint16)
    W = np.random.default_rng(1).permutation(bits).view(np.float16).reshape(-1, 128)
    codes, scales = quantize(gpu, W, "f16")
    want = narrow.mx4_encode(W)
    assert np.array_equal(scales, want[1]) and np.array_equal(codes, want[0])


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("cols", [32, 64, 63, 33, 1])
def test_dequantize_every_code_and_scale(gpu, kind, cols):
    rng = np.random.default_rng(cols)
    nb = -(-cols // 32)
    codes = rng.integers(0, 256, (256, nb * 16)).astype(np.uint8)
    codes[:, 0] = 0x10  # codes in order from the first block on
    codes[:, :8] = [0x10, 0x32, 0x54, 0x76, 0x98, 0xBA, 0xDC, 0xFE]
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], nb, 1)
    dt = np.float16 if kind == "f16" else np.float32
    n = 256 * cols * np.dtype(dt).itemsize
    dst = out_bytes(gpu, n)
    dc, ds = gpu.upload(codes), gpu.upload(scales)
    gpu.call("eng_mx4_dequantize_" + kind, dc.ptr, ds.ptr, dst.ptr, 256, cols, None)
    gpu.sync()
    got = take(dst, n, dt, (256, cols))
    with np.errstate(over="ignore"):
        want = narrow.mx4_decode(codes, scales, cols).astype(dt)
    assert np.array_equal(got, want, equal_nan=True)


def test_dequantize_unaligned_destination(gpu):
    rng = np.random.default_rng(2)
    codes = rng.integers(0, 256, (5, 32)).astype(np.uint8)
    scales = rng.integers(110, 140, (5, 2)).astype(np.uint8)
    dst = out_bytes(gpu, 4 + 5 * 64 * 4)
    dc, ds = gpu.upload(codes), gpu.upload(scales)
    gpu.call("eng_mx4_dequantize_f32", dc.ptr, ds.ptr, dst.ptr + 4, 5, 64, None)
    gpu.sync()
    got = take(dst, 4 + 5 * 64 * 4, np.float32, (1 + 5 * 64,))
    assert np.array_equal(got[1:].reshape(5, 64), narrow.mx4_decode(codes, scales, 64).astype(np.float32))


# ------------------------------------------------------------------- linear
def weights(rng, N, K, spread=6):
    nb = -(-K // 32)
    codes = rng.integers(0, 256, (N, nb * 16)).astype(np.uint8)
    scales = rng.integers(120 - spread, 120 + spread + 1, (N, nb)).astype(np.uint8)
    return codes, scales


def linear(gpu, x, codes, scales, N, g=None, rms=False, skew=0, stream=None):
    M, K = x.shape
    dx = gpu.upload(np.concatenate([np.zeros(skew, np.float32), x.reshape(-1)]))
    dc, ds = gpu.upload(codes), gpu.upload(scales)
    dg = None if g is None else gpu.upload(g)
    y = out_bytes(gpu, M * N * 4)
    if rms:
        gpu.call("eng_rmsnorm_linear_mx4w_nk", dx.ptr + 4 * skew, None if dg is None else dg.ptr,
                 dc.ptr, ds.ptr, y.ptr, M, N, K, EPS, stream)
    else:
        gpu.call("eng_linear_mx4w_nk", dx.ptr + 4 * skew, dc.ptr, ds.ptr, y.ptr, M, N, K, stream)
    gpu.sync()
    return take(y, M * N * 4, np.float32, (M, N))


def check_linear(gpu, rng, M, N, K, rms, gain=True, skew=0):
    x = rng.standard_normal((M, K)).astype(np.float32)
    g = (1 + 0.1 * rng.standard_normal(K)).astype(np.float32) if rms and gain else None
    codes, scales = weights(rng, N, K)
    got = linear(gpu, x, codes, scales, N, g, rms, skew)
    y, a = narrow.linear64(x, narrow.mx4_decode(codes, scales, K), g, EPS if rms else None)
    helpers.assert_within(got, y, narrow.linear_bound(y, a, K, rms), f"mx4 linear {M} x {N} x {K}")


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 15, 16, 17, 31, 32, 33, 48, 64, 65, 100, 129, 200])
@pytest.mark.parametrize("N,K", [(1, 1), (15, 31), (16, 32), (17, 33), (96, 130), (250, 516)])
def test_linear_small(gpu, M, N, K, rms):
    check_linear(gpu, np.random.default_rng(M * 31 + N * 7 + K + rms), M, N, K, rms)


@pytest.mark.parametrize("M,N,K,rms", [
    (1, 4096, 4096, False), (1, 2051, 1023, True), (2, 1000, 4096, True), (4, 528, 11008, True),
    (1, 300, 28672, False), (3, 64, 28671, True), (7, 2051, 1023, True), (16, 1024, 4096, False),
    (32, 512, 11008, True), (37, 2051, 1023, True), (64, 1024, 2048, True), (128, 768, 1024, False),
    (257, 1111, 1000, True), (512, 1024, 512, False)])
def test_linear_large(gpu, M, N, K, rms):
    check_linear(gpu, np.random.default_rng(M + N + K), M, N, K, rms)


@pytest.mark.parametrize("M", [1, 3, 6, 20, 50])
def test_linear_unaligned_x_and_no_gain(gpu, M):
    rng = np.random.default_rng(M)
    check_linear(gpu, rng, M, 70, 260, True, gain=False)
    check_linear(gpu, rng, M, 70, 260, True, skew=1)
    check_linear(gpu, rng, M, 70, 260, False, skew=3)


@pytest.mark.parametrize("M", [1, 4, 9, 30, 70])
def test_linear_wide_scales_and_tiny_activations(gpu, M):
    """Scales across 2^-60 .. 2^60 within a row, activations across 2^-40 .. 2^40:
    every product is exact, so the bound on the sum of magnitudes still holds."""
    rng = np.random.default_rng(M + 100)
    N, K = 40, 300
    x = (rng.standard_normal((M, K)) * np.exp2(rng.integers(-40, 41, (M, K)))).astype(np.float32)
    codes, scales = weights(rng, N, K, spread=60)
    got = linear(gpu, x, codes, scales, N)
    y, a = narrow.linear64(x, narrow.mx4_decode(codes, scales, K))
    helpers.assert_within(got, y, narrow.linear_bound(y, a, K, False), "wide scales")


@pytest.mark.parametrize("M", [1, 2, 5, 18, 40])
def test_linear_special_values(gpu, M):
    """A NaN scale reaches its own column only, an infinite or NaN activation its own
    row only, with the sign (or NaN against a zero weight) that fp32 gives."""
    rng = np.random.default_rng(M + 7)
    N, K = 50, 200
    codes, scales = weights(rng, N, K)
    scales[13, 2] = 255
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[0, 150] = np.inf
    if M > 1:
        x[1, 7] = np.nan
        x.view(np.uint32)[1, 8] = 0x7F800001  # a NaN whose payload is in the low bits
    if M > 4:
        x[4, 3] = np.finfo(np.float32).max / 16
    got = linear(gpu, x, codes, scales, N)
    with np.errstate(invalid="ignore", over="ignore"):
        W = narrow.mx4_decode(codes, scales, K)
        y, a = narrow.linear64(x, W)
    fin = np.isfinite(y)
    assert np.array_equal(np.isnan(got), np.isnan(y))
    assert np.array_equal(got[~fin & ~np.isnan(y)], y[~fin & ~np.isnan(y)])
    bound = narrow.linear_bound(np.where(fin, y, 0), np.where(fin, a, 0), K, False)
    helpers.assert_within(got[fin], y[fin], bound[fin], "finite elements")


def test_linear_k_zero_fills_and_rmsnorm_leaves(gpu):
    y = gpu.empty(12, np.float32)
    y.fill_bytes(0x11)
    one = gpu.empty(16, np.float32)
    gpu.call("eng_rmsnorm_linear_mx4w_nk", one.ptr, None, one.ptr, one.ptr, y.ptr, 3, 4, 0, EPS, None)
    gpu.sync()
    assert (y.download().view(np.uint8) == 0x11).all()
    gpu.call("eng_linear_mx4w_nk", one.ptr, one.ptr, one.ptr, y.ptr, 3, 4, 0, None)
    gpu.sync()
    assert (y.download() == 0).all()


@pytest.mark.parametrize("M", [1, 12, 80])
def test_linear_streams_graph_and_repeats_give_the_same_bits(gpu, M):
    rng = np.random.default_rng(M)
    N, K = 333, 1000
    x = rng.standard_normal((M, K)).astype(np.float32)
    codes, scales = weights(rng, N, K)
    first = linear(gpu, x, codes, scales, N)
    with gpu.stream() as s:
        assert np.array_equal(first, linear(gpu, x, codes, scales, N, stream=s.handle))
        dx, dc, ds = gpu.upload(x), gpu.upload(codes), gpu.upload(scales)
        y = gpu.empty((M, N), np.float32)
        args = (dx.ptr, dc.ptr, ds.ptr, y.ptr, M, N, K, s.handle)
        gpu.call("eng_linear_mx4w_nk", *args)
        s.sync()
        graph = gpu.graph(s)
        with graph:
            gpu.call("eng_linear_mx4w_nk", *args)
        for i in range(3):
            scaled = (x * (i + 1)).astype(np.float32)
            dx.upload(scaled)
            y.fill_bytes(0xFF)
            gpu.sync()
            graph.launch()
            s.sync()
            assert np.array_equal(y.download(), linear(gpu, scaled, codes, scales, N))
        graph.destroy()
