"""The long-context operators where offsets pass 32 bits: caches of more than 4 GiB a head,
logits of more than 4 GiB a row. Buffers are allocated, and only what a call reads is
written."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

import long_context as lc

pytestmark = pytest.mark.gpu
F16 = np.float16


def put(gpu, buf, at, host):
    """host into buf's bytes from `at` on."""
    host = np.ascontiguousarray(host)
    gpu.call("eng_memcpy_h2d", buf.ptr + at, host.ctypes.data_as(ctypes.c_void_p), host.nbytes)


def get(gpu, buf, at, shape, dtype):
    out = np.empty(shape, dtype)
    gpu.call("eng_memcpy_d2h", out.ctypes.data_as(ctypes.c_void_p), buf.ptr + at, out.nbytes)
    return out


@pytest.mark.parametrize("kind", ["f16", "q8"])
@pytest.mark.parametrize("S", [1, 40])
def test_window_at_the_end_of_a_long_cache(gpu, kind, S):
    rng = np.random.default_rng(S)
    H, G, D, window, sinks, tail = 4, 2, 128, 50, 2, 128
    es = 2 if kind == "f16" else 1
    room = (1 << 32) // (D * es) + 4096  # tokens; a head's bytes pass 2^32
    pos = room - S - 3
    first = (pos - window) // 32 * 32   # from here on the cache is written, and the sinks' block
    small = lc.Cache(gpu, rng, kind, 1, G, 32 + tail, D, [32 + tail])
    big = [gpu.empty((1, G, room, D), np.uint16 if es == 2 else np.uint8) for _ in range(2)]
    nb = -(-room // 32)
    if kind == "q8":
        big += [gpu.empty((1, G, nb), np.float32) for _ in range(2)]
    n = min(tail, room - first)
    for g in range(G):
        for side in range(2):
            put(gpu, big[side], g * room * D * es, small.raw[side][0, g, :32])
            put(gpu, big[side], (g * room + first) * D * es, small.raw[side][0, g, 32:32 + n])
            if kind == "q8":
                put(gpu, big[2 + side], g * nb * 4, small.scales[side][0, g, :1])
                put(gpu, big[2 + side], (g * nb + first // 32) * 4, small.scales[side][0, g, 1:1 + -(-n // 32)])
    q = rng.standard_normal((1, S, H, D)).astype(F16)
    dq, do = gpu.upload(q.view(np.uint16)), gpu.empty(q.shape, np.uint16)
    dp = gpu.upload(np.array([pos], np.int32))
    gpu.call("eng_attention_window_" + kind, dq.ptr, *[b.ptr for b in big], do.ptr, dp.ptr, None, 1, S, H, G, D,
             window, sinks, room, room, 0.1, 0, None)
    gpu.sync()
    want = {}
    for i in range(S):
        j = lc.seen_keys(pos + i, window, sinks, room)
        at = np.where(j < 32, j, j - first + 32)
        for h in range(H):
            want[0, i, h] = lc.attend_rows(q[0, i, h].astype(np.float64), small.values[0][0, h // 2, at],
                                           small.values[1][0, h // 2, at], small.vmax[0, h // 2],
                                           float(np.float32(0.1)))
    lc.check(do.download().view(F16), want, "long cache")


def test_reorder_of_long_caches(gpu):
    rng = np.random.default_rng(2)
    D, room = 128, (1 << 25) + 64  # 4 GiB and a little of 8-bit tokens each
    nb = -(-room // 32)
    k, v = gpu.empty((2, 1, room, D), np.uint8), gpu.empty((2, 1, room, D), np.uint8)
    ks, vs = gpu.empty((2, 1, nb), np.float32), gpu.empty((2, 1, nb), np.float32)
    k.fill_bytes(1), v.fill_bytes(2), ks.fill_bytes(0), vs.fill_bytes(0)
    rows = {}
    for buf in (k, v):
        for b in range(2):
            for at in (0, room // 2, room - 8):
                rows[id(buf), b, at] = rng.integers(0, 255, (8, D), dtype=np.uint8)
                put(gpu, buf, (b * room + at) * D, rows[id(buf), b, at])
    for b in range(2):
        put(gpu, ks, (b * nb + nb - 1) * 4, np.array([3.0 + b], np.float32))
    dp, dl = gpu.upload(np.array([1, 0], np.int32)), gpu.upload(np.array([room, room], np.int32))
    ptrs = [a.ptr for a in (k, v, ks, vs)]
    gpu.call("eng_kv_cache_reorder_q8", *ptrs, *ptrs, dp.ptr, dl.ptr, 1, 2, 1, D, room, room, None)
    gpu.sync()
    for buf in (k, v):
        for b in range(2):
            for at in (0, room // 2, room - 8):
                assert np.array_equal(get(gpu, buf, (b * room + at) * D, (8, D), np.uint8), rows[id(buf), 1 - b, at])
    assert [get(gpu, ks, (b * nb + nb - 1) * 4, 1, np.float32)[0] for b in range(2)] == [4.0, 3.0]


def test_select_with_rows_far_apart(gpu):
    rng = np.random.default_rng(3)
    ld, V = (1 << 30) + 32, 1000
    x = (3 * rng.standard_normal((1, 2, V))).astype(np.float32)
    big = gpu.empty(2 * ld, np.float32)
    for b in range(2):
        put(gpu, big, b * ld * 4, x[0, b])
    scores = np.array([[-1.0, -1.2]], np.float32)
    ds = gpu.upload(scores)
    outs = [gpu.empty((1, 6), t) for t in (np.float32, np.int32, np.int32, np.uint8)]
    gpu.call("eng_beam_select_f32", big.ptr, ld, ds.ptr, None, *[o.ptr for o in outs], 1, 2, 6, V, -1, None)
    gpu.sync()
    s, p, t, _ = lc.select64(x[0].astype(np.float64), scores[0].astype(np.float64), None, 6, -1)
    assert np.array_equal(outs[1].download()[0], p) and np.array_equal(outs[2].download()[0], t)
    assert np.allclose(outs[0].download()[0], s, rtol=1e-6)
