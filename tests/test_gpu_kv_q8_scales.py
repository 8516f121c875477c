"""Decode attention over 8-bit caches whose V scales lie far apart or far below what
the append makes: blocks of zeros with the least scale that a writer's floor leaves, and
codes whose scale was set to zero."""

from __future__ import annotations

import numpy as np
import pytest

import helpers
import narrow
from test_gpu_kv_q8 import Cache, attend

pytestmark = pytest.mark.gpu
TINY = [0.0, 2.0**-149, 1e-40, 2.0**-126, 1e-36, 2.0**-120, 2.0**-60, 2.0**-41, 2.0**-40, 2.0**-39]


def foreign(gpu, rng, L, D, vs=2.0**-8, B=1, G=2):
    """A cache of any finite codes, K scales that keep scores within a few units."""
    c = Cache(gpu, rng, B, G, L, D)
    finite = lambda: (rng.integers(0, 2, (B, G, L, D)) * 128 + rng.integers(0, 127, (B, G, L, D))).astype(np.uint8)  # noqa: E731
    c.k, c.v = finite(), finite()
    c.ks[:] = 0.05 / np.sqrt(D)
    c.vs[:] = vs
    return c, (0.3 * rng.standard_normal((B, 2 * G, D))).astype(np.float16)


def check(gpu, c, q, split):
    """Scales below 2^-40 may count as 2^-40: that moves a value by at most 448 2^-40 <
    2^-31, and with it the weighted mean, on top of narrow.attend64's bound."""
    c.dev = [gpu.upload(a) for a in (c.k, c.v, c.ks, c.vs)]
    L, scale = c.shape[2], 1.0
    y, bound = narrow.attend64(q.astype(np.float64), c.k, c.v, c.ks, c.vs, [L], scale)
    got = attend(gpu, c, q, [L], L, scale, split)
    helpers.assert_within(got, y, bound + 2.0**-31, f"split {split}")
    return y, bound


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tiny", TINY)
def test_tiny_v_scales_beside_ordinary_ones(gpu, tiny, D):
    """In the first blocks of the waves, the middle ones, the last ones, alone and in all
    but one: the keys count in the denominator whatever their values are."""
    rng = np.random.default_rng(int(np.float32(tiny).view(np.uint32)) + D)
    for at in ([0, 1, 2, 3], [5], [8, 9, 10, 11], [0, 6, 11], list(range(11)), [12]):
        c, q = foreign(gpu, rng, 32 * 12 + 5, D)
        c.vs[..., at] = tiny
        for split in (1, 3, 0):
            y, bound = check(gpu, c, q, split)
            assert bound.max() < 0.02 * np.abs(y).max()


@pytest.mark.parametrize("tiny", TINY)
def test_nothing_but_tiny_v_scales(gpu, tiny):
    rng = np.random.default_rng(3)
    c, q = foreign(gpu, rng, 300, 64, vs=tiny)
    for split in (1, 3):
        check(gpu, c, q, split)


@pytest.mark.parametrize("high", [-6.0, 6.0])
def test_tiny_scales_where_the_scores_differ(gpu, high):
    """Keys of the tiny-scale blocks above, and below, the others."""
    rng = np.random.default_rng(4)
    for tiny in (0.0, 2.0**-126, 2.0**-44):
        c, q = foreign(gpu, rng, 32 * 10, 128)
        c.vs[..., ::2] = tiny
        # one dim of K and q carries a score of its own: +-high 2 / 2 per block
        q[..., 0] = 1.0
        c.ks[..., ::2] = 2.0**-4
        c.k[:, :, :, 0] = 0
        c.k[:, :, :, 1:] &= 0x87  # the least exponents: small scores beside dim 0's
        for j in range(0, 10, 2):
            c.k[:, :, 32 * j:32 * j + 32, 0] = narrow.e4m3_encode(np.array([high * 16]))[0]
        for split in (1, 2):
            check(gpu, c, q, split)


def test_zero_scales_do_not_cost_the_other_blocks_precision(gpu):
    """Values of 128 to 240 times 2^-25, a hundred of fp16's least steps, beside blocks
    whose scale is zero: the bound, with the largest scale 2^-25, allows little more than
    half such a step."""
    rng = np.random.default_rng(5)
    c, q = foreign(gpu, rng, 32 * 12, 128, vs=2.0**-25)
    c.vs[..., [0, 5, 10, 11]] = 0
    c.v[...] = (c.v & 7) | 0x70  # one sign: no cancellation
    for split in (1, 3):
        y, bound = check(gpu, c, q, split)
        assert bound.max() < 2.0**-24 < np.abs(y).max() / 64


def test_nan_codes_count_under_a_zero_scale(gpu):
    """A value is its code times its block's scale: NaN, also where the scale is zero."""
    rng = np.random.default_rng(6)
    c, q = foreign(gpu, rng, 100, 64)
    c.vs[0, 1, 1] = 0
    c.v[0, 1, 40, 9] = 0x7F
    c.dev = [gpu.upload(a) for a in (c.k, c.v, c.ks, c.vs)]
    for split in (1, 3):
        got = attend(gpu, c, q, [100], 100, 1.0, split)
        assert np.isnan(got[0, 2:, 9]).all()
        assert np.isfinite(got[0, :2]).all() and np.isfinite(np.delete(got[0, 2:], 9, axis=1)).all()


@pytest.mark.parametrize("top,code", [(1.0, 0x38), (2.0**12, 0x38), (2.0**24, 0x01)])
def test_zero_codes_under_a_large_v_scale(gpu, top, code):
    """Blocks of zeros under the largest scales beside blocks under 2^-40 and zero; the
    last block's values are all the same. Numerator and denominator are then sums of the
    same weights, each held to 2^-22 (the last block's are among the largest), so the
    output's rounding, 2^-11, is nearly all of the error."""
    rng = np.random.default_rng(7)
    c, q = foreign(gpu, rng, 32 * 12, 128, vs=top)
    c.vs[..., 1::3] = 2.0**-40
    c.vs[..., 2::3] = 0
    c.v[...] = 0
    c.v[:, :, 32 * 11:, :] = code
    c.vs[..., 11] = top
    y, _ = narrow.attend64(q.astype(np.float64), c.k, c.v, c.ks, c.vs, [384], 1.0)
    assert 0.01 < y.min() and y.max() < 60000
    c.dev = [gpu.upload(a) for a in (c.k, c.v, c.ks, c.vs)]
    for split in (1, 3):
        got = attend(gpu, c, q, [384], 384, 1.0, split)
        helpers.assert_within(got, y, 2.0**-10.9 * y, f"split {split}")
