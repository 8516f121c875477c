"""GPU tests of the tiles of 256 rows (eight waves, three LDS buffers) that long-context
attention takes at head_dim 128 where they leave a workgroup for every CU: prompts with
windows, sinks, splits and ragged counts, values that are not finite, and shared prefixes.
Rows are picked and checked as in test_gpu_attention_window."""

from __future__ import annotations

import numpy as np
import pytest

import long_context as lc
import test_gpu_attention_prefix as prefix
import test_gpu_attention_window as window

pytestmark = pytest.mark.gpu
KINDS = pytest.mark.parametrize("kind", ["f16", "q8"])
B, G, D = 32, 8, 128  # 256 pairs of a sequence and a KV head


def is_wide(gpu, units, rows):
    """The launcher's rule: tiles of 256 rows where there is one for every CU."""
    return units * -(-rows // 256) >= gpu.cu_count()


def run(gpu, kind, S, H, **kw):
    assert is_wide(gpu, B * G, S * H // G)
    return window.run(gpu, kind, B, S, H, G, D, rows=[0, S // 2, S - 1], **kw)


def positions(most):
    return [(29 * b) % (most + 1) for b in range(B)]


@KINDS
@pytest.mark.parametrize("win,sinks", [(0, 0), (40, 4), (30, 70), (1, 0)])
def test_prompts(gpu, kind, win, sinks):
    # 280 rows a pair: a full tile and one of 24 rows
    run(gpu, kind, 70, 32, pos=positions(150), window=win, sinks=sinks)


@KINDS
@pytest.mark.parametrize("win,sinks", [(0, 0), (33, 65)])
def test_ragged_counts(gpu, kind, win, sinks):
    pos = positions(100)
    pos[3] = pos[17] = -1
    n = [(31 * b) % 90 - 5 for b in range(B)]
    run(gpu, kind, 70, 32, pos=pos, n_new=n, window=win, sinks=sinks)


@KINDS
@pytest.mark.parametrize("split", [3, 100])
@pytest.mark.parametrize("win,sinks", [(0, 0), (90, 5)])
def test_splits(gpu, kind, split, win, sinks):
    run(gpu, kind, 40, 32, pos=positions(180), window=win, sinks=sinks, split=split)


@KINDS
@pytest.mark.parametrize("win,sinks", [(20, 3), (64, 64)])
def test_windows_that_waves_of_a_tile_do_not_share(gpu, kind, win, sinks):
    """One head a pair: 256 tokens to a tile, most key tiles seen by one or two waves."""
    run(gpu, kind, 300, 8, pos=[0] * B, window=win, sinks=sinks)


@KINDS
@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_scales(gpu, kind, scale):
    run(gpu, kind, 40, 32, pos=positions(60), window=50, sinks=4, scale=scale)


@KINDS
def test_rows_at_any_alignment(gpu, kind):
    run(gpu, kind, 33, 32, pos=positions(70), q_shift=1)


@KINDS
def test_large_scores(gpu, kind):
    run(gpu, kind, 33, 32, pos=positions(150), sigma=6.0)


@KINDS
def test_lengths_past_the_bound(gpu, kind):
    run(gpu, kind, 40, 32, pos=positions(150), window=30, sinks=2, max_len=100)


@KINDS
@pytest.mark.parametrize("split", [1, 3])
@pytest.mark.parametrize("win,sinks", [(0, 0), (40, 70)])
def test_values_that_are_not_finite(gpu, kind, win, sinks, split):
    """In sequence 1: NaN behind its window, infinities and a NaN that its later queries see."""
    S, pos = 70, positions(150)
    pos[1] = p = 120
    hidden = np.setdiff1d(np.arange(p), lc.seen_keys(p, win, sinks, p + S))
    inf = np.nan if kind == "q8" else np.inf

    def edit(k, v):
        for j in hidden[::7]:
            k[1, :, j] = np.nan
            v[1, :, j, ::2] = np.inf
            v[1, :, j, 1::2] = np.nan
        late = p + S // 2
        v[1, 0, late, 3] = np.nan
        v[1, 0, late, 5] = inf
        v[1, 0, late, 6] = -inf
        v[1, :, p + S - 1, 100] = inf

    got = run(gpu, kind, S, 32, pos=pos, window=win, sinks=sinks, split=split, edit=edit).astype(np.float64)
    assert np.isfinite(got[0]).all() and np.isfinite(got[2:]).all()
    assert np.isfinite(got[1, :S // 2]).all()


# ------------------------------------------------------------- shared prefixes
def run_prefix(gpu, kind, per, H, plen, longest, split=0, edit=None):
    groups = len(plen)
    n = groups * per
    assert per * H // G > 128
    rng = np.random.default_rng(per + H)
    lens = [(7 * b) % (longest + 1) for b in range(n)]
    cache = lc.Cache(gpu, rng, kind, groups, G, max(plen) + 3, D, plen, 1.0, edit)
    own = lc.Cache(gpu, rng, kind, n, G, longest + 1, D, lens)
    q = rng.standard_normal((n, H, D)).astype(np.float16).astype(np.float64)
    scale = float(np.float32(1 / np.sqrt(D)))
    got = prefix.call(gpu, kind, q, cache, plen, own, lens, max(plen), longest, scale, split)
    rest = H // G
    for b in {0, 1, per // 2, per - 1, per % n, n // 2 + 1, n - per, n - 1}:
        p = b // per
        want = {}
        for h in range(H):
            g = h // rest
            k, v = (np.concatenate((cache.values[i][p, g, :plen[p]], own.values[i][b, g, :lens[b]])) for i in (0, 1))
            want[b, h] = lc.attend_rows(q[b, h], k, v, max(cache.vmax[p, g], own.vmax[b, g]), scale)
        lc.check(got, want, f"sequence {b}")
    return got.astype(np.float64)


@KINDS
@pytest.mark.parametrize("per,H,longest,split", [(20, 64, 3, 0), (70, 32, 2, 2)])
def test_prefixes(gpu, kind, per, H, longest, split):
    plen = [(53 * g) % 200 + 1 for g in range(32)]
    assert is_wide(gpu, 32 * G, per * H // G)
    run_prefix(gpu, kind, per, H, plen, longest, split)


@KINDS
@pytest.mark.parametrize("groups,per,H", [(32, 20, 64), (2, 20, 64), (1, 70, 32)])  # 256 and 128 rows a tile
def test_prefix_values_that_are_not_finite(gpu, kind, groups, per, H):
    assert is_wide(gpu, groups * G, per * H // G) == (groups == 32)
    plen = [150 - g for g in range(groups)]
    inf = np.nan if kind == "q8" else np.inf

    def edit(k, v):
        v[0, 0, 17, 5] = np.nan
        v[0, :, 40, 7], v[0, 1, 99, 9] = inf, -inf
        v[0, 2, 3, 11], v[0, 2, 149, 11] = inf, -inf

    got = run_prefix(gpu, kind, per, H, plen, 3, edit=edit)
    assert np.isfinite(got[per:]).all()
    bad = ~np.isfinite(got[:per]).all(0)
    assert set(np.flatnonzero(bad.any(0))) == {5, 7, 9, 11}
