"""GPU tests of eng_beam_select_* and eng_kv_cache_reorder_*: choices equal to those of the
float64 scores, scores within their bound, and caches moved byte for byte."""

from __future__ import annotations

import numpy as np
import pytest

import long_context as lc
from helpers import U32

pytestmark = pytest.mark.gpu
KINDS = pytest.mark.parametrize("kind", ["f32", "f16"])


def select(gpu, kind, x, scores, finished, n_out, eos, ld=None, shift=0, vocab=None, stream=None):
    """x [groups, beams, V] float32 / float16; vocab: how much of a row counts."""
    groups, beams, V = x.shape
    ld = ld or V
    vocab = vocab or V
    host = np.full(groups * beams * ld + shift, np.nan, x.dtype)
    host[shift:].reshape(groups * beams, ld)[:, :vocab] = x.reshape(-1, V)[:, :vocab]
    dx = gpu.upload(host)
    ds = gpu.upload(scores.astype(np.float32))
    df = None if finished is None else gpu.upload(finished.astype(np.uint8))
    outs = [gpu.upload(np.full(groups * n_out + 1, 77, t)) for t in (np.float32, np.int32, np.int32, np.uint8)]
    gpu.call("eng_beam_select_" + kind, dx.ptr + shift * x.itemsize, ld, ds.ptr, None if df is None else df.ptr,
             *[o.ptr for o in outs], groups, beams, n_out, vocab, eos, stream)
    gpu.sync()
    got = [o.download() for o in outs]
    assert all(g[-1] == 77 for g in got)
    return [g[:-1].reshape(groups, n_out) for g in got]


def check(got, x, scores, finished, n_out, eos):
    """Choices exactly; scores to fp32's rounding and that of L = log sum exp: its sum's
    terms are off by 8 u each (exp and its argument, |x - max| under 64) and the sum of a
    lane by another 16 + V / 4096 additions, so L by (24 + V / 4096) u, u = 2^-24."""
    V = x.shape[2]
    for g in range(x.shape[0]):
        s, p, t, f = lc.select64(x[g].astype(np.float64), scores[g].astype(np.float32).astype(np.float64),
                                 None if finished is None else finished[g], n_out, eos)
        assert np.array_equal(got[1][g], p), f"group {g}: parents {got[1][g]} for {p}"
        assert np.array_equal(got[2][g], t), f"group {g}: tokens {got[2][g]} for {t}"
        assert np.array_equal(got[3][g] != 0, f), f"group {g}: finished"
        fin = np.isfinite(s)
        assert np.array_equal(got[0][g][~fin], s[~fin])
        assert (np.abs(got[0][g][fin] - s[fin]) <= U32 * np.abs(s[fin]) + (88 + V / 4096) * U32).all()


def inputs(rng, kind, groups, beams, V, ties=False):
    x = (3 * rng.standard_normal((groups, beams, V))).astype(np.float32)
    if ties:
        x = np.round(x)
    scores = (-10 - 4 * rng.random((groups, beams))).astype(np.float32)
    return x.astype(np.float16 if kind == "f16" else np.float32), scores


@KINDS
@pytest.mark.parametrize("groups,beams,n_out,V", [
    (1, 1, 1, 1), (1, 1, 1, 2), (1, 2, 4, 2), (3, 3, 5, 7), (1, 4, 8, 1000), (2, 4, 8, 4096), (2, 4, 8, 4097),
    (1, 1, 64, 64), (1, 1, 64, 5000), (2, 32, 64, 300), (5, 5, 10, 8191), (1, 4, 8, 32000), (3, 1, 2, 50257),
    (2, 10, 20, 20011), (1, 32, 64, 2),
])
@pytest.mark.parametrize("ties", [False, True])
def test_select(gpu, kind, groups, beams, n_out, V, ties):
    rng = np.random.default_rng(groups + beams + n_out + V)
    x, scores = inputs(rng, kind, groups, beams, V, ties)
    check(select(gpu, kind, x, scores, None, n_out, -1), x, scores, None, n_out, -1)
    finished = rng.random((groups, beams)) < 0.4
    eos = int(rng.integers(0, V))
    check(select(gpu, kind, x, scores, finished, n_out, eos), x, scores, finished, n_out, eos)


@KINDS
@pytest.mark.parametrize("ld,shift", [(1003, 0), (1001, 0), (1024, 0), (1024, 1), (1008, 8), (1002, 3)])
def test_strides_and_alignment(gpu, kind, ld, shift):
    rng = np.random.default_rng(ld + shift)
    x, scores = inputs(rng, kind, 2, 3, 1001)
    check(select(gpu, kind, x, scores, None, 6, 5, ld, shift), x, scores, None, 6, 5)


@KINDS
@pytest.mark.parametrize("order", ["rising", "falling", "equal", "one piece"])
@pytest.mark.parametrize("k", [3, 64])
def test_orders(gpu, kind, order, k):
    """Rows whose best tokens lie where a pass finds most to do."""
    V = 30000
    base = {"rising": np.arange(V), "falling": -np.arange(V), "equal": np.zeros(V),
            "one piece": np.where(np.abs(np.arange(V) - 9000) < 40, 5 + np.arange(V) % 7, 0)}[order]
    x = np.stack([base / 2048.0, base / 2048.0 + 1])[None].astype(np.float16 if kind == "f16" else np.float32)
    scores = np.array([[-1.0, -1.5]], np.float32)
    check(select(gpu, kind, x, scores, None, k, -1), x, scores, None, k, -1)


@KINDS
def test_masked_and_special_values(gpu, kind):
    rng = np.random.default_rng(1)
    x, scores = inputs(rng, kind, 6, 4, 500)
    inf = np.inf
    x[0, 1, 5:] = -inf                      # a constrained beam: five tokens left
    x[0, 2] = -inf                          # none left
    x[1, 0, 7] = np.nan                     # not a row of numbers
    x[1, 1, 9] = inf
    x[2, :, 3:] = -inf                      # fewer live candidates than asked for
    x[2, 0, 0] = np.finfo(x.dtype).max
    x[2, 1, 1] = np.finfo(x.dtype).min      # the type's lowest value as a mask
    scores[3] = [0, -inf, -inf, -inf]       # the first step
    scores[4] = [-inf, np.nan, inf, -5]
    scores[5] = -inf                        # nothing lives
    x[5, 3] = np.nan
    x[0, 0, :50] = 0.0
    x[0, 0, ::2] = np.where(x[0, 0, ::2] == 0, -0.0, x[0, 0, ::2])  # -0 and 0 tie
    for n_out in (4, 20, 64):
        check(select(gpu, kind, x, scores, None, n_out, 2), x, scores, None, n_out, 2)
    finished = np.zeros((6, 4), bool)
    finished[:, 1] = finished[4, 0] = finished[2, 3] = True
    for n_out, eos in ((4, 2), (20, 499), (64, 0), (5, 30)):
        check(select(gpu, kind, x, scores, finished, n_out, eos), x, scores, finished, n_out, eos)


def test_large_vocabulary(gpu):
    rng = np.random.default_rng(2)
    x, scores = inputs(rng, "f32", 3, 4, 152064)
    check(select(gpu, "f32", x, scores, None, 8, 2), x, scores, None, 8, 2)


def test_out_finished_may_be_null_and_calls_repeat(gpu):
    rng = np.random.default_rng(4)
    x, scores = inputs(rng, "f32", 2, 4, 9000)
    want = select(gpu, "f32", x, scores, None, 8, 3)
    dx, ds = gpu.upload(x), gpu.upload(scores)
    outs = [gpu.empty((2, 8), t) for t in (np.float32, np.int32, np.int32)]

    def step(stream):
        gpu.call("eng_beam_select_f32", dx.ptr, 9000, ds.ptr, None, *[o.ptr for o in outs], None, 2, 4, 8, 9000, 3,
                 stream)

    with gpu.stream() as s:
        step(s.handle)
        s.sync()
        graph = gpu.graph(s)
        with graph:
            step(s.handle)
        for i in range(3):
            for o in outs:
                o.fill_bytes(0)
            gpu.sync()
            graph.launch()
            select(gpu, "f32", x[::-1].copy(), scores, None, 64, 3, stream=s.handle)  # more scratch, between replays
            s.sync()
            for o, w in zip(outs, want):
                assert np.array_equal(o.download(), w), f"replay {i}"
        graph.destroy()


# -------------------------------------------------------------------- reorder
def reorder(gpu, kind, groups, beams, G, D, room, lens, parent, max_len, in_place, seed=0):
    rng = np.random.default_rng(seed + beams + room)
    B, nb = groups * beams, -(-room // 32)
    dt = np.uint8 if kind == "q8" else np.uint16
    draw = lambda: [rng.integers(0, np.iinfo(dt).max, (B, G, room, D), dtype=dt) for _ in range(2)] + (  # noqa: E731
        [rng.random((B, G, nb), dtype=np.float32) for _ in range(2)] if kind == "q8" else [])
    src = draw()
    old = [a.copy() for a in (src if in_place else draw())]
    want = [a.copy() for a in old]
    for g in range(groups):
        for j in range(beams):
            p = int(parent[g][j])
            if not 0 <= p < beams:
                continue
            n = max(0, min(int(lens[g * beams + p]), max_len))
            for i, a in enumerate(want):
                m = n if i < 2 else -(-n // 32)
                a[g * beams + j, :, :m] = src[i][g * beams + p, :, :m]
    ds = [gpu.upload(a) for a in src]
    dd = ds if in_place else [gpu.upload(a) for a in old]
    dp, dl = gpu.upload(np.asarray(parent, np.int32)), gpu.upload(np.asarray(lens, np.int32))
    gpu.call("eng_kv_cache_reorder_" + kind, *[d.ptr for d in ds], *[d.ptr for d in dd], dp.ptr, dl.ptr, groups,
             beams, G, D, max_len, room, None)
    gpu.sync()
    for i, (d, w) in enumerate(zip(dd, want)):
        assert np.array_equal(d.download(), w), f"buffer {i}"
    if not in_place:
        for d, w in zip(ds, src):
            assert np.array_equal(d.download(), w), "a source was written"


@pytest.mark.parametrize("kind", ["f16", "q8"])
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("groups,beams,G,D,room,parent", [
    (1, 1, 1, 64, 1, [[0]]),
    (1, 2, 1, 64, 33, [[1, 0]]),                       # an exchange
    (2, 3, 2, 128, 70, [[1, 2, 0], [2, 2, 2]]),        # a rotation; one survivor
    (1, 4, 3, 64, 500, [[3, -1, 4, 0]]),               # two left as they are
    (3, 5, 1, 128, 40, [[0, 1, 2, 3, 4], [4, 3, 2, 1, 0], [0, 0, 3, 3, 1]]),
    (1, 9, 2, 64, 100, [[8, 7, 6, 5, 4, 3, 2, 1, 0]]),
    (1, 17, 1, 64, 65, [list(range(1, 17)) + [0]]),
    (1, 32, 1, 128, 35, [[(5 * j) % 32 for j in range(32)]]),
])
def test_reorder(gpu, kind, in_place, groups, beams, G, D, room, parent):
    rng = np.random.default_rng(room)
    B = groups * beams
    reorder(gpu, kind, groups, beams, G, D, room, [room] * B, parent, room, in_place)
    lens = rng.integers(-1, room + 9, B)
    reorder(gpu, kind, groups, beams, G, D, room, lens, parent, room, in_place)
    reorder(gpu, kind, groups, beams, G, D, room, lens, parent, (room + 1) // 2, in_place)


@pytest.mark.parametrize("kind", ["f16", "q8"])
def test_reorder_long(gpu, kind):
    rng = np.random.default_rng(0)
    reorder(gpu, kind, 4, 6, 4, 128, 1500, rng.integers(0, 1500, 24), rng.integers(0, 6, (4, 6)), 1500, True)
