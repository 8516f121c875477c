"""GPU tests of infinities and NaN in V rows that single tokens see (the formula's result:
an infinity's weight is above zero, so it stays that infinity; two of unlike signs, or a
NaN, give NaN), over one cache, in splits, and over a shared prefix of few and of many rows."""

from __future__ import annotations

import numpy as np
import pytest

import long_context as lc
import test_gpu_attention_prefix as prefix
import test_gpu_attention_window as window

pytestmark = pytest.mark.gpu
KINDS = pytest.mark.parametrize("kind", ["f16", "q8"])


def special(v, b, keys, kind):
    """Dims 1 to 6 of the first, middle and last of `keys` in sequence b's caches."""
    first, mid, last = keys[0], keys[len(keys) // 2], keys[-1]
    inf = np.nan if kind == "q8" else np.inf  # (e4m3 has no infinity)
    v[b, :, first, 1] = inf
    v[b, :, mid, 2] = -inf
    v[b, :, last, 3] = inf
    v[b, :, first, 4], v[b, :, last, 4] = inf, inf
    v[b, 0, mid, 5] = np.nan
    if len(keys) > 1:
        v[b, :, first, 6], v[b, :, last, 6] = inf, -inf


@KINDS
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,G", [(2, 2), (8, 2), (20, 1)])
@pytest.mark.parametrize("pos,win,sinks,split", [
    (0, 0, 0, 0), (1, 0, 0, 0), (31, 0, 0, 0), (32, 0, 0, 0), (200, 0, 0, 0), (700, 0, 0, 0), (700, 0, 0, 1),
    (700, 0, 0, 7), (700, 100, 0, 0), (700, 100, 40, 3), (3000, 1500, 4, 0)])
def test_single_tokens(gpu, kind, D, H, G, pos, win, sinks, split):
    keys = lc.seen_keys(pos, win, sinks, pos + 1)
    hidden = np.setdiff1d(np.arange(pos), keys)

    def edit(k, v):
        special(v, 0, keys, kind)
        v[0, :, hidden[::3], ::2] = np.inf
        v[0, :, hidden[1::3]] = np.nan

    got = window.run(gpu, kind, 2, 1, H, G, D, [pos, max(pos - 1, 0)], None, win, sinks, split=split, edit=edit)
    assert np.isfinite(got[1].astype(np.float64)).all()
    assert np.isfinite(got[0, 0][:, 7:].astype(np.float64)).all()


@KINDS
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [20, 100])
def test_many_sequences(gpu, kind, D, n):
    """Workgroups of one wave; every second sequence holds them."""
    keys = np.arange(n)

    def edit(k, v):
        for b in range(0, 130, 2):
            special(v, b, keys, kind)

    got = window.run(gpu, kind, 130, 1, 8, 8, D, [n - 1] * 130, edit=edit)
    assert np.isfinite(got[1::2].astype(np.float64)).all()


@KINDS
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("per,H,G,plen,split", [
    (2, 4, 2, [100, 80], 0), (4, 8, 2, [1, 500], 3), (40, 8, 2, [300], 0),
    (70, 8, 2, [200, 3], 0), (33, 4, 1, [900], 2), (130, 2, 2, [129], 1)])  # the last three: tiles of many rows
def test_shared_prefixes(gpu, kind, D, per, H, G, plen, split):
    def edit(k, v):
        special(v, 0, np.arange(plen[0]), kind)

    lens = [(3 * b) % 11 for b in range(per * len(plen))]
    got = prefix.run(gpu, kind, per, H, G, D, plen, lens, split=split, edit=edit)
    assert np.isfinite(got[per:].astype(np.float64)).all()
    assert np.isfinite(got[:per, :, 7:].astype(np.float64)).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,split", [(1, 0), (1, 1), (1, 5), (40, 1), (40, 5)])
def test_weights_far_below_the_largest(gpu, D, S, split):
    """Keys whose weights no fp32 number holds (2^-150 of the largest and less) still count."""
    def edit(k, v):
        k[0, :, :, 0] = np.where(np.arange(k.shape[2]) % 97 == 5, 100, -100)
        special(v, 0, np.arange(600), "f16")

    rng = np.random.default_rng(4)
    cache = lc.Cache(gpu, rng, "f16", 1, 2, 640, D, [640], edit=edit)
    q = rng.standard_normal((1, S, 4, D)).astype(np.float16)
    q[..., 0] = 8
    q = q.astype(np.float64)
    got = window.call(gpu, "f16", q, cache, [640 - S], None, 0, 0, 640, 0.125, split)
    lc.check(got, lc.window64(q, cache, [640 - S], None, 0, 0, 640, 0.125), "far below")
    assert np.isinf(got[0, 0, 0, 1:5].astype(np.float64)).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,split", [(1, 1), (1, 4), (40, 1), (40, 4)])
def test_rows_without_a_score(gpu, D, S, split):
    """Where all scores that a row sees are -inf it gets zeros, infinities in V or not, and such
    keys in one of several splits leave the others' result as it is."""
    def edit(k, v):
        k[0, 0, :, 0] = -np.inf       # the first KV head: no score at all
        k[0, 1, :128, 0] = -np.inf    # the second: from the 129th key on
        v[0, :, 5, 3], v[0, :, 70, 4] = np.inf, -np.inf

    rng = np.random.default_rng(12)
    cache = lc.Cache(gpu, rng, "f16", 1, 2, 400, D, [400], edit=edit)
    q = rng.standard_normal((1, S, 4, D)).astype(np.float16)
    q[..., 0] = np.abs(q[..., 0]) + np.float16(0.5)
    q = q.astype(np.float64)
    got = window.call(gpu, "f16", q, cache, [400 - S], None, 0, 0, 400, 0.125, split)
    assert (got[0, :, :2] == 0).all()
    want = {}
    for i in range(S):
        j = np.arange(128, 400 - S + i + 1)
        for h in (2, 3):
            y, bound = lc.attend_rows(q[0, i, h], cache.values[0][0, 1, j], cache.values[1][0, 1, j],
                                      cache.vmax[0, 1], 0.125)
            rest = np.delete(np.arange(D), (3, 4))  # (weights of 0 times an infinity: left open)
            assert (np.abs(got[0, i, h].astype(np.float64) - y) <= bound)[rest].all()
