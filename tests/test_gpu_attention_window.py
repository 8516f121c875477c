"""GPU tests of eng_attention_window_*: prompts, pieces of prompts and single tokens over
fp16 and 8-bit caches, with windows and sinks, against the float64 formula within
long_context.attend_rows' bound."""

from __future__ import annotations

import numpy as np
import pytest

import long_context as lc

pytestmark = pytest.mark.gpu
F16 = np.float16


def call(gpu, kind, q, cache, pos, n_new, window, sinks, max_len, scale, split=0, stream=None, out=None,
         q_shift=0):
    """Runs the entry; rows that it must not write hold 0x7777."""
    B, S, H, D = q.shape
    G = cache.raw[0].shape[1]
    host = np.full(q.size + 8, 0x7777, np.uint16)
    host[q_shift:q_shift + q.size] = q.astype(F16).view(np.uint16).reshape(-1)
    dq = gpu.upload(host)
    do = gpu.upload(np.full(q.size + 8, 0x7777, np.uint16))
    dp = gpu.upload(np.asarray(pos, np.int32))
    dn = None if n_new is None else gpu.upload(np.asarray(n_new, np.int32))
    gpu.call("eng_attention_window_" + kind, dq.ptr + 2 * q_shift, *cache.ptrs, do.ptr + 2 * q_shift, dp.ptr,
             None if dn is None else dn.ptr, B, S, H, G, D, window, sinks, max_len, cache.room, scale,
             split, stream)
    gpu.sync()
    raw = do.download()
    assert (raw[:q_shift] == 0x7777).all() and (raw[q_shift + q.size:] == 0x7777).all()
    return raw[q_shift:q_shift + q.size].view(F16).reshape(q.shape)


def run(gpu, kind, B, S, H, G, D, pos, n_new=None, window=0, sinks=0, max_len=None, scale=None, split=0,
        seed=0, rows=None, sigma=1.0, edit=None, q_shift=0):
    rng = np.random.default_rng(seed + 1000 * B + 10 * S + H + D)
    n = [S] * B if n_new is None else [min(max(x, 0), S) for x in n_new]
    lens = [max(p, 0) + x if p >= 0 else 0 for p, x in zip(pos, n)]
    max_len = max(max(lens), 1) if max_len is None else max_len
    room = max(max(lens), max_len) + 5
    cache = lc.Cache(gpu, rng, kind, B, G, room, D, lens, sigma, edit)
    q = (sigma * rng.standard_normal((B, S, H, D))).astype(F16).astype(np.float64)
    scale = 1 / np.sqrt(D) if scale is None else scale
    got = call(gpu, kind, q, cache, pos, n_new, window, sinks, max_len, scale, split, q_shift=q_shift)
    lc.check(got, lc.window64(q, cache, pos, n_new, window, sinks, max_len, float(np.float32(scale)), rows),
             f"{kind} window {window}")
    raw = got.view(np.uint16)
    for b in range(B):
        first = n[b] if pos[b] >= 0 else 0
        assert (raw[b, first:] == 0x7777).all(), f"sequence {b}: rows behind its queries were written"
    return got


KINDS = pytest.mark.parametrize("kind", ["f16", "q8"])


@KINDS
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,S,H,G,pos,n_new,window,sinks", [
    (1, 1, 1, 1, [0], None, 0, 0),
    (1, 2, 1, 1, [0], None, 0, 0),
    (1, 33, 2, 2, [0], None, 0, 0),
    (1, 64, 2, 1, [0], None, 0, 0),
    (1, 65, 4, 1, [63], None, 0, 0),
    (2, 40, 6, 2, [0, 100], None, 0, 0),           # a group of three: tiles end inside a token
    (2, 100, 8, 1, [5, 31], [100, 17], 0, 0),
    (4, 30, 2, 1, [0, 3, -1, 50], [30, 0, 30, -2], 0, 0),
    (1, 150, 4, 2, [0], None, 1, 0),
    (1, 150, 4, 2, [0], None, 40, 0),
    (1, 150, 4, 2, [0], None, 40, 4),
    (1, 150, 4, 2, [200], None, 64, 33),
    (1, 200, 2, 1, [300], None, 65, 130),          # sinks of more than a tile
    (1, 90, 4, 1, [70], None, 1000, 7),            # a window longer than the sequence
    (3, 70, 3, 1, [0, 128, 517], [70, 69, 1], 96, 1),
    (1, 20, 40, 1, [31], None, 25, 2),             # a group of 40
    (2, 10, 4, 2, [6, 2], [99, 3], 7, 0),          # a count past s_new
])
def test_prompts(gpu, kind, D, B, S, H, G, pos, n_new, window, sinks):
    run(gpu, kind, B, S, H, G, D, pos, n_new, window, sinks)


@KINDS
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,G", [(1, 1), (4, 1), (8, 2), (12, 4), (24, 1)])
@pytest.mark.parametrize("pos,window,sinks", [
    ([0, 1, 31, 32], 0, 0),
    ([63, 64, 65, 511], 0, 0),
    ([0, 40, 300, -1], 33, 0),
    ([5, 100, 1000, 2047], 64, 4),
    ([700, 701, 702, 3], 130, 70),
    ([600, 10, 20, 30], 1, 1),
])
def test_single_tokens(gpu, kind, D, H, G, pos, window, sinks):
    run(gpu, kind, 4, 1, H, G, D, pos, None, window, sinks)


@KINDS
@pytest.mark.parametrize("S,split", [(1, 1), (1, 3), (1, 256), (7, 2), (7, 100), (130, 5)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 4)])
def test_splits(gpu, kind, S, split, window, sinks):
    run(gpu, kind, 2, S, 4, 2, 64, [0, 700], None, window, sinks, split=split)


@KINDS
def test_lengths_past_the_bound_are_cut_off(gpu, kind):
    # the second sequence's window lies behind the bound: its sinks are left, or nothing
    for sinks in (0, 3):
        run(gpu, kind, 3, 9, 2, 1, 64, [95, 200, 90], None, 20, sinks, max_len=100)
        run(gpu, kind, 3, 1, 2, 1, 64, [95, 200, 119], None, 20, sinks, max_len=100)
    run(gpu, kind, 2, 9, 2, 1, 64, [95, 200], None, 0, 0, max_len=100)
    run(gpu, kind, 2, 3, 2, 1, 128, [0, 5], None, 0, 0, max_len=0)
    run(gpu, kind, 2, 1, 2, 1, 128, [0, 5], None, 4, 2, max_len=0)


@KINDS
@pytest.mark.parametrize("S", [1, 40])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7])
def test_scales(gpu, kind, S, scale):
    run(gpu, kind, 2, S, 4, 2, 64, [0, 90], None, 50, 4, scale=scale)


@KINDS
@pytest.mark.parametrize("S", [1, 40])
def test_any_alignment_of_the_rows(gpu, kind, S):
    for shift in (1, 2, 4):
        run(gpu, kind, 2, S, 4, 2, 64, [0, 90], None, 0, 0, q_shift=shift)


@KINDS
@pytest.mark.parametrize("S", [1, 70])
def test_large_scores(gpu, kind, S):
    run(gpu, kind, 1, S, 4, 2, 128, [100], None, 0, 0, sigma=6.0)


@KINDS
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,pos,window,sinks", [
    (1, 200, 64, 4), (60, 0, 0, 0), (60, 200, 48, 4), (150, 33, 40, 36), (1, 40, 0, 0)])
def test_infinities_and_nan_in_places_that_are_not_seen(gpu, kind, D, S, pos, window, sinks):
    """NaN and infinities in K and V of some tokens: queries that do not see them are as if
    they were not there, queries that do get what the formula gives."""
    rng = np.random.default_rng(5)
    L = pos + S
    seen = lc.seen_keys(pos, window, sinks, L)
    masked = np.setdiff1d(np.arange(pos), seen)
    late = pos + S // 2 if S > 1 else None

    def edit(k, v):
        for j in masked[rng.permutation(len(masked))[:6]]:
            k[0, :, j] = np.nan
            v[0, :, j, ::2] = np.inf
            v[0, :, j, 1::2] = np.nan
        if late is not None:
            v[0, 0, late, 3] = np.nan
            v[0, 0, late, 5] = np.nan if kind == "q8" else np.inf
            v[0, 0, late, 6] = np.nan if kind == "q8" else -np.inf
            v[0, 0, L - 1] = np.nan

    got = run(gpu, kind, 1, S, 4, 2, D, [pos], None, window, sinks, edit=edit)
    assert np.isfinite(got[0, 0].astype(np.float64)).all()
    if late is not None:
        assert np.isfinite(got[0, :late - pos].astype(np.float64)).all()


@KINDS
def test_a_nan_query_stays_in_its_row(gpu, kind):
    rng = np.random.default_rng(6)
    cache = lc.Cache(gpu, rng, kind, 1, 1, 64, 64, [40])
    q = rng.standard_normal((1, 40, 2, 64)).astype(F16).astype(np.float64)
    clean = call(gpu, kind, q, cache, [0], None, 0, 0, 40, 0.125)
    q[0, 7, 1, 3] = np.nan
    got = call(gpu, kind, q, cache, [0], None, 0, 0, 40, 0.125)
    assert np.isnan(got[0, 7, 1]).all()
    got[0, 7, 1] = clean[0, 7, 1]
    assert np.array_equal(got.view(np.uint16), clean.view(np.uint16))


@KINDS
@pytest.mark.parametrize("S,window", [(1, 0), (1, 700), (900, 0), (900, 333)])
def test_long(gpu, kind, S, window):
    rows = [0, 1, S // 2, S - 1]
    run(gpu, kind, 1, S, 8, 2, 128, [4100], None, window, 4 if window else 0, rows=rows)


@KINDS
def test_tiny_weights_add_up(gpu, kind):
    """One key far above 4000 others whose weights are 2^-18 to 2^-22 of it."""
    def edit(k, v):
        k[:] = 0
        v[:, :, 1:] = 1
        v[:, :, 0] = -1
        k[0, 0, 0, 0] = 16.0
        k[0, 0, 1:, 1] = np.linspace(-1, 1, k.shape[2] - 1)
    rng = np.random.default_rng(0)
    cache = lc.Cache(gpu, rng, kind, 1, 1, 4096, 64, [4096], edit=edit)
    for S in (1, 64):
        q = np.zeros((1, S, 1, 64))
        q[..., 0], q[..., 1] = 20 * np.log(2) / 16, np.log(2)
        q = q.astype(F16).astype(np.float64)
        got = call(gpu, kind, q, cache, [4096 - S], None, 0, 0, 4096, 1.0)
        lc.check(got, lc.window64(q, cache, [4096 - S], None, 0, 0, 4096, 1.0), "tiny weights")


@KINDS
@pytest.mark.parametrize("S", [1, 48])
def test_the_same_bits_on_streams_and_in_replays(gpu, kind, S):
    """Eager on the null stream and on another, and captured once and replayed with
    positions that advance, between eager calls of another shape on the same stream."""
    rng = np.random.default_rng(S)
    B, H, G, D, room = 2, 4, 2, 64, 600
    cache = lc.Cache(gpu, rng, kind, B, G, room, D, [room, room])
    q = rng.standard_normal((B, S, H, D)).astype(F16)
    dq, do = gpu.upload(q.view(np.uint16)), gpu.empty(q.shape, np.uint16)
    dp = gpu.upload(np.array([0, 0], np.int32))
    big = gpu.empty((4, 60, H, D), np.uint16)
    big.fill_bytes(0)
    dbig = gpu.upload(np.array([500, 17, 3, -1], np.int32)[:2])

    def step(stream, split):
        gpu.call("eng_attention_window_" + kind, dq.ptr, *cache.ptrs, do.ptr, dp.ptr, None, B, S, H, G, D,
                 200, 4, room, room, 0.125, split, stream)

    for split in (1, 4):
        with gpu.stream() as s:
            step(s.handle, split)
            s.sync()
            graph = gpu.graph(s)
            with graph:
                step(s.handle, split)
            for pos in ([0, 10], [300, 500], [552, -1]):
                dp.upload(np.array(pos, np.int32))
                do.fill_bytes(0)
                gpu.sync()
                step(None, split)
                gpu.sync()
                want = do.download()
                for _ in range(2):
                    do.fill_bytes(0)
                    gpu.sync()
                    graph.launch()
                    gpu.call("eng_attention_window_" + kind, big.ptr, *cache.ptrs, big.ptr + 2 * B * 60 * H * D,
                             dbig.ptr, None, B, 60, H, G, D, 0, 0, room, room, 0.125, 3, s.handle)
                    s.sync()
                    assert np.array_equal(do.download(), want)
            graph.destroy()


@KINDS
@pytest.mark.parametrize("S", [1, 33])
def test_positions_far_past_the_cache(gpu, kind, S):
    """Positions near 2^31: only the sinks are left below the bound, or nothing."""
    rng = np.random.default_rng(S)
    cache = lc.Cache(gpu, rng, kind, 2, 1, 64, 64, [64, 64])
    q = rng.standard_normal((2, S, 2, 64)).astype(F16).astype(np.float64)
    pos = [2**31 - 1, 2**31 - 40]
    for window, sinks in ((0, 0), (50, 3), (50, 0), (2**40, 1), (2**62, 2)):
        got = call(gpu, kind, q, cache, pos, None, window, sinks, 64, 0.125)
        want = {}
        for b in range(2):
            for i in range(S):
                p = pos[b] + i
                j = np.arange(64)
                j = j if window == 0 else j[(j > p - window) | (j < sinks)]
                for h in range(2):
                    want[b, i, h] = lc.attend_rows(q[b, i, h], cache.values[0][b, 0, j], cache.values[1][b, 0, j],
                                                   cache.vmax[b, 0], 0.125)
        lc.check(got, want, f"window {window}, sinks {sinks}")


@KINDS
def test_two_streams_at_once(gpu, kind):
    """Calls with scratch that overlap on two streams, against the same calls one by one."""
    rng = np.random.default_rng(1)
    B, H, G, D, room = 2, 8, 2, 128, 3000
    jobs = []
    for n, S in enumerate((1, 30)):
        cache = lc.Cache(gpu, rng, kind, B, G, room, D, [room] * B)
        q = rng.standard_normal((B, S, H, D)).astype(F16)
        jobs.append((cache, gpu.upload(q.view(np.uint16)), gpu.empty(q.shape, np.uint16),
                     gpu.upload(np.array([room - S, 1000 + n], np.int32)), S))

    def issue(job, stream):
        cache, dq, do, dp, S = job
        gpu.call("eng_attention_window_" + kind, dq.ptr, *cache.ptrs, do.ptr, dp.ptr, None, B, S, H, G, D, 0, 0, room,
                 room, 0.09, 8, stream)

    want = []
    for job in jobs:
        issue(job, None)
        gpu.sync()
        want.append(job[2].download())
    with gpu.stream() as one, gpu.stream() as two:
        for job in jobs:
            job[2].fill_bytes(0)
        gpu.sync()
        for _ in range(20):
            issue(jobs[0], one.handle)
            issue(jobs[1], two.handle)
        one.sync()
        two.sync()
        for job, w in zip(jobs, want):
            assert np.array_equal(job[2].download(), w)


@pytest.mark.parametrize("S", [1, 40])
def test_keys_of_minus_infinity(gpu, S):
    """A visible key whose score is -inf has no weight (e4m3 has no infinity)."""
    kind = "f16"

    def edit(k, v):
        k[..., :] = np.abs(k)
        k[0, :, 7, 0] = -np.inf

    rng = np.random.default_rng(8)
    cache = lc.Cache(gpu, rng, kind, 1, 1, 80, 64, [80], edit=edit)
    q = np.abs(rng.standard_normal((1, S, 2, 64))).astype(F16).astype(np.float64) + 0.5
    q = q.astype(F16).astype(np.float64)
    got = call(gpu, kind, q, cache, [80 - S], None, 0, 0, 80, 0.125)
    want = {}
    for i in range(S):
        j = np.setdiff1d(np.arange(80 - S + i + 1), [7])
        for h in range(2):
            want[0, i, h] = lc.attend_rows(q[0, i, h], cache.values[0][0, 0, j], cache.values[1][0, 0, j],
                                           cache.vmax[0, 0], 0.125)
    lc.check(got, want, "-inf")


@KINDS
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("longest,window,sinks", [(32, 0, 0), (64, 0, 0), (128, 0, 0),
                                                  (129, 0, 0), (300, 50, 3), (300, 20, 0)])
def test_many_short_sequences(gpu, kind, D, longest, window, sinks):
    # enough of them for a workgroup of one wave each, up to four blocks of keys
    pos = [(37 * b) % (longest + 1) - 1 for b in range(130)]
    run(gpu, kind, 130, 1, 8, 8, D, pos, None, window, sinks, max_len=longest)
