"""GPU tests of eng_attention_prefix_*: single tokens of sequences that share prefixes,
against the float64 formula within long_context.attend_rows' bound."""

from __future__ import annotations

import numpy as np
import pytest

import long_context as lc

pytestmark = pytest.mark.gpu
F16 = np.float16
KINDS = pytest.mark.parametrize("kind", ["f16", "q8"])


def call(gpu, kind, q, prefix, plen, own, lens, max_prefix, max_len, scale, split=0, stream=None):
    B, H, D = q.shape
    G = own.raw[0].shape[1]
    dq, do = gpu.upload(q.astype(F16).view(np.uint16)), gpu.upload(np.full(q.size + 8, 0x7777, np.uint16))
    dp, dl = gpu.upload(np.asarray(plen, np.int32)), gpu.upload(np.asarray(lens, np.int32))
    gpu.call("eng_attention_prefix_" + kind, dq.ptr, *prefix.ptrs, dp.ptr, *own.ptrs, dl.ptr, do.ptr,
             len(plen), B, H, G, D, max_prefix, prefix.room, max_len, own.room, scale, split, stream)
    gpu.sync()
    raw = do.download()
    assert (raw[q.size:] == 0x7777).all()
    return raw[:q.size].view(F16).reshape(q.shape)


def run(gpu, kind, per, H, G, D, plen, lens, max_prefix=None, max_len=None, scale=None, split=0, edit=None,
        sigma=1.0):
    B = per * len(plen)
    assert len(lens) == B
    rng = np.random.default_rng(B + 10 * H + D + sum(plen))
    max_prefix = max(max(plen), 0) if max_prefix is None else max_prefix
    max_len = max(max(lens), 0) if max_len is None else max_len
    cut = [min(n, max_prefix) for n in plen], [min(n, max_len) for n in lens]
    prefix = lc.Cache(gpu, rng, kind, len(plen), G, max_prefix + 3, D, cut[0], sigma, edit)
    own = lc.Cache(gpu, rng, kind, B, G, max_len + 1, D, cut[1], sigma)
    q = (sigma * rng.standard_normal((B, H, D))).astype(F16).astype(np.float64)
    scale = 1 / np.sqrt(D) if scale is None else scale
    got = call(gpu, kind, q, prefix, plen, own, lens, max_prefix, max_len, scale, split)
    lc.check(got, lc.prefix64(q, prefix, cut[0], own, cut[1], float(np.float32(scale))), f"{kind} prefix")
    return got


@KINDS
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("per,H,G,plen,lens", [
    (1, 1, 1, [1], [1]),
    (1, 4, 2, [33], [0]),
    (2, 4, 2, [0], [5, 0]),                       # no prefix; a sequence without a key gets zeros
    (2, 2, 1, [64, 65], [1, 31, 32, 33]),
    (4, 8, 2, [300], [0, 1, 64, 100]),
    (4, 4, 4, [700, 1, 128], [3] * 12),
    (5, 6, 2, [97], [1, 2, 3, 4, 5]),
    (40, 8, 2, [200], list(range(40))),           # more rows than a tile
    (3, 40, 1, [150], [7, 70, 170]),              # 120 rows of one KV head
    (33, 4, 1, [257], [2] * 33),                  # 132
    (2, 4, 2, [-1, 40], [4, -3, 0, 2]),           # lengths below zero are zero
])
def test_prefix(gpu, kind, D, per, H, G, plen, lens):
    run(gpu, kind, per, H, G, D, plen, lens)


@KINDS
@pytest.mark.parametrize("split", [1, 2, 7, 1000])
def test_splits(gpu, kind, split):
    run(gpu, kind, 3, 4, 2, 64, [900, 40], [0, 3, 200, 500, 33, 1], split=split)
    run(gpu, kind, 3, 4, 2, 128, [90, 40], [0, 3, 20, 50, 33, 1], split=split)


@KINDS
def test_bounds_cut_lengths(gpu, kind):
    run(gpu, kind, 2, 4, 2, 64, [500, 20], [50, 3, 10, 11], max_prefix=100, max_len=10)
    run(gpu, kind, 2, 4, 2, 64, [500, 20], [50, 3, 10, 11], max_prefix=0, max_len=10)
    run(gpu, kind, 2, 4, 2, 64, [500, 20], [50, 3, 10, 11], max_prefix=100, max_len=0)
    run(gpu, kind, 2, 4, 2, 64, [500, 20], [50, 3, 10, 11], max_prefix=0, max_len=0)


@KINDS
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.5])
def test_scales(gpu, kind, scale):
    run(gpu, kind, 2, 4, 2, 64, [100], [50, 3], scale=scale)


@KINDS
def test_long(gpu, kind):
    run(gpu, kind, 4, 8, 2, 128, [5000], [600, 1, 0, 99])


@KINDS
def test_a_nan_value_in_a_prefix_reaches_its_group_only(gpu, kind):
    def edit(k, v):
        v[0, 0, 17, 5] = np.nan
    got = run(gpu, kind, 2, 4, 2, 64, [100, 80], [5, 6, 7, 8], edit=edit)
    assert np.isnan(got[:2, :2, 5]).all() and np.isnan(got.astype(np.float64)).sum() == 4


@KINDS
def test_as_one_cache(gpu, kind):
    """A prefix and own tokens give what one cache that holds both gives."""
    rng = np.random.default_rng(3)
    B, H, G, D, P, n = 3, 4, 2, 64, 96, 40
    prefix = lc.Cache(gpu, rng, kind, 1, G, P, D, [P])
    own = lc.Cache(gpu, rng, kind, B, G, n, D, [n] * B)
    q = rng.standard_normal((B, H, D)).astype(F16).astype(np.float64)
    got = call(gpu, kind, q, prefix, [P], own, [n] * B, P, n, 0.125)
    want = {}
    for b in range(B):
        for h in range(H):
            k, v = (np.concatenate((prefix.values[i][0, h // 2], own.values[i][b, h // 2])) for i in (0, 1))
            want[b, h] = lc.attend_rows(q[b, h], k, v, max(prefix.vmax.max(), own.vmax.max()), 0.125)
    lc.check(got, want, "one cache")


@KINDS
def test_replayed_with_lengths_that_grow(gpu, kind):
    rng = np.random.default_rng(9)
    per, H, G, D, P, room = 4, 4, 2, 64, 300, 80
    prefix = lc.Cache(gpu, rng, kind, 2, G, P, D, [P, P])
    own = lc.Cache(gpu, rng, kind, 2 * per, G, room, D, [room] * 2 * per)
    q = rng.standard_normal((2 * per, H, D)).astype(F16)
    dq, do = gpu.upload(q.view(np.uint16)), gpu.empty(q.shape, np.uint16)
    dp, dl = gpu.upload(np.array([P, 250], np.int32)), gpu.upload(np.zeros(2 * per, np.int32))

    def step(stream):
        gpu.call("eng_attention_prefix_" + kind, dq.ptr, *prefix.ptrs, dp.ptr, *own.ptrs, dl.ptr, do.ptr, 2,
                 2 * per, H, G, D, P, P, room, room, 0.125, 0, stream)

    with gpu.stream() as s:
        step(s.handle)
        s.sync()
        graph = gpu.graph(s)
        with graph:
            step(s.handle)
        for t in (0, 1, 33, 80):
            dl.upload(np.full(2 * per, t, np.int32))
            gpu.sync()
            step(None)
            gpu.sync()
            want = do.download()
            lc.check(want.view(F16), lc.prefix64(q.astype(np.float64), prefix, [P, 250], own, [t] * 2 * per, 0.125),
                     f"token {t}")
            do.fill_bytes(0)
            gpu.sync()
            graph.launch()
            step(s.handle)  # eager work on the capture's stream beside it
            s.sync()
            assert np.array_equal(do.download(), want)
        graph.destroy()


@KINDS
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("prefix,longest", [(15, 5), (32, 32), (33, 128), (129, 40)])
def test_many_short_sequences(gpu, kind, D, prefix, longest):
    # enough of them for a workgroup of one wave each, up to four blocks of keys
    run(gpu, kind, 10, 8, 8, D, [(5 * g) % (prefix + 1) for g in range(12)] + [prefix],
        [(37 * b) % (longest + 1) for b in range(130)], max_prefix=prefix, max_len=longest)
