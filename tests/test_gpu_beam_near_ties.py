"""GPU tests of eng_beam_select_* where beams' candidates lie closer than fp32 sums tell
apart: their order is that of the scores in 64 bits.

Bounds of L = log sum exp, u = 2^-24. Of the sum of fp32 exponentials, relative: a term's
argument, x - max in the end, by 1.22 |x - max| u (one rounding, log2 e as an fp32 number) and
half a u, whose mean over the row's weights is 1.22 log V u at the most (an entropy less log
of the sum, and that is 1 at least); an exponential 2 u, a lane's additions 6 u, the rest in
64 bits: wide(V). Candidates of unlike beams closer than twice that are compared by sums in 64 bits, v =
2^-53: an exponential to 2e-14 and its argument's rounding, |x - L| log2 e v, under 2e-14
for |x - L| < 100 and times its weight beyond; V / 256 + 20 additions of v: 6e-14 for V <
60000, and the few roundings of scores under 1000 another 4e-13. EPS = 1e-12."""

from __future__ import annotations

import numpy as np
import pytest

import long_context as lc
from helpers import U32
from test_gpu_beam import select

pytestmark = pytest.mark.gpu
KINDS = pytest.mark.parametrize("kind", ["f32", "f16"])
EPS = 1e-12


def wide(V):
    return (1.22 * np.log(V) + 10) * U32


def lse64(x):
    return x.max(-1) + np.log(np.exp(x - x.max(-1, keepdims=True)).sum(-1))


@KINDS
@pytest.mark.parametrize("V", [300, 4096, 9001, 50257])
@pytest.mark.parametrize("spread", [0.5, 3.0, 20.0])
def test_beams_a_hair_apart(gpu, kind, V, spread):
    """Beam 1's score is set so that its best candidate meets beam 0's as nearly as an fp32
    score can: the gaps are roundings of it, 1e-6 to nothing."""
    rng = np.random.default_rng(V + int(10 * spread))
    groups = 40
    x = (spread * rng.standard_normal((groups, 2, V))).astype(np.float16 if kind == "f16" else np.float32)
    lse = lse64(x.astype(np.float64))
    top = x.astype(np.float64).max(2)
    scores = np.zeros((groups, 2), np.float32)
    scores[:, 0] = -rng.random(groups)
    scores[:, 1] = (scores[:, 0].astype(np.float64) + (top[:, 0] - lse[:, 0])) - (top[:, 1] - lse[:, 1])
    best = scores.astype(np.float64) + (top - lse)
    apart = np.abs(best[:, 0] - best[:, 1]) > 2 * EPS
    assert apart.sum() > 30 and (np.abs(best[:, 0] - best[:, 1]) < 1e-5).all()
    got = select(gpu, kind, x, scores, None, 2, -1)
    first = np.where(best[:, 0] > best[:, 1], 0, 1)
    wrong = np.flatnonzero(apart & (got[1][:, 0] != first))
    assert not len(wrong), f"groups {wrong}: gaps {(best[wrong, 0] - best[wrong, 1])}"


@KINDS
@pytest.mark.parametrize("V", [1, 63, 5000, 33000])
@pytest.mark.parametrize("spread", [0.0, 2.0, 12.0])
def test_scores_and_their_order(gpu, kind, V, spread):
    rng = np.random.default_rng(V + 7)
    x = (spread * rng.standard_normal((6, 3, V))).astype(np.float16 if kind == "f16" else np.float32)
    scores = (-2 * rng.random((6, 3))).astype(np.float32)
    n_out = min(6, 3 * V)
    got = select(gpu, kind, x, scores, None, n_out, -1)
    for g in range(6):
        s = scores[g].astype(np.float64)[:, None] + (x[g].astype(np.float64) - lse64(x[g].astype(np.float64))[:, None])
        at = s[got[1][g], got[2][g]]
        assert (np.abs(got[0][g] - at) <= U32 * np.abs(at) + wide(V)).all()
        assert (at >= np.sort(s.reshape(-1))[::-1][:n_out] - 2 * EPS).all()


@KINDS
def test_equal_rows_of_all_beams_tie_to_the_lower(gpu, kind):
    """The same logits and scores in every beam: every token ties, in beams' order, however
    the sums come out."""
    rng = np.random.default_rng(0)
    row = (2 * rng.standard_normal(20011)).astype(np.float16 if kind == "f16" else np.float32)
    x = np.broadcast_to(row, (3, 5, 20011)).copy()
    scores = np.full((3, 5), -1.25, np.float32)
    got = select(gpu, kind, x, scores, None, 15, -1)
    for g in range(3):
        _, p, t, _ = lc.select64(x[g].astype(np.float64), scores[g].astype(np.float64), None, 15, -1)
        assert np.array_equal(got[1][g], p) and np.array_equal(got[2][g], t)


@KINDS
def test_large_and_far_apart_logits(gpu, kind):
    """Terms that vanish beside the largest, and rows far from zero, where exponents of x
    itself would leave every range."""
    rng = np.random.default_rng(2)
    dt = np.float16 if kind == "f16" else np.float32
    x = (3 * rng.standard_normal((4, 2, 3000))).astype(dt)
    x[0] = (x[0] + (60000 if kind == "f16" else 1e30)).astype(dt)
    x[1] = (x[1] - (60000 if kind == "f16" else 1e6)).astype(dt)
    x[2, :, ::2] = -np.inf
    x[2, :, 1::4] = np.finfo(dt).min
    x[3] *= 100
    scores = np.array([[-1, -1.5]] * 4, np.float32)
    got = select(gpu, kind, x, scores, None, 4, -1)
    for g in range(4):
        s, p, t, _ = lc.select64(x[g].astype(np.float64), scores[g].astype(np.float64), None, 4, -1)
        assert np.array_equal(got[1][g], p) and np.array_equal(got[2][g], t)
        # (a score is formed from x and L, half a step of 64 bits of either each)
        far = 4 * 2.0**-53 * np.abs(x[g].astype(np.float64)[np.isfinite(x[g])]).max()
        assert (np.abs(got[0][g] - s) <= U32 * np.abs(s) + wide(3000) + far).all()


@pytest.mark.parametrize("base", [300.0, -5000.0, 2.0**21, 1e7, -3e7, 3e8, -1e30])
def test_rows_far_from_zero(gpu, base):
    """Logits whose differences count though the numbers are large: L less the row's largest
    logit is compared, in which nothing is lost; and NaN, infinities and masks among them."""
    rng = np.random.default_rng(3)
    V, step = 5000, float(np.spacing(np.float32(abs(base))))
    x = (base + step * rng.integers(0, 4, (5, 2, V))).astype(np.float32)
    x[1, 0, 4321] = np.nan
    x[1, 1, 17] = np.inf
    x[2, 0, 1::2] = -np.inf
    x[2, 1] = -np.inf
    x[3, 0, 5] = np.finfo(np.float32).min
    scores = (-rng.random((5, 2))).astype(np.float32)
    got = select(gpu, "f32", x, scores, None, 3, -1)
    for g in range(5):
        want = []
        for b in range(2):
            row = x[g, b].astype(np.float64)
            top = row.max()
            if not np.isfinite(top):
                want += [(-np.inf, -b, -t) for t in range(3)]
                continue
            more = np.log(np.exp(row - top).sum())
            want += [(float(scores[g, b]) - more + (row[t] - top), -b, -t)
                     for t in np.lexsort((np.arange(V), -row))[:3]]
        want = sorted(want, reverse=True)[:3]
        assert [(-b, -t) for _, b, t in want] == list(zip(got[1][g], got[2][g]))
        for s, y in zip(want, got[0][g]):
            assert y == s[0] or abs(y - s[0]) <= U32 * abs(s[0]) + wide(V)


@KINDS
def test_masked_rows(gpu, kind):
    """Rows of -inf alone, in all beams but one: the others' order is the live beam's."""
    rng = np.random.default_rng(4)
    x = (3 * rng.standard_normal((3, 4, 9000))).astype(np.float16 if kind == "f16" else np.float32)
    x[:, 1:] = -np.inf
    got = select(gpu, kind, x, np.full((3, 4), -1, np.float32), None, 8, -1)
    for g in range(3):
        assert (got[1][g] == 0).all()
        assert np.array_equal(got[2][g], np.lexsort((np.arange(9000), -x[g, 0].astype(np.float64)))[:8])


@KINDS
@pytest.mark.parametrize("V", [700, 20011])
def test_equal_beams_beside_one_a_hair_apart(gpu, kind, V):
    """Beams 1 and 3 are equal, beam 0 or 2 comes as near to them as an fp32 score can."""
    rng = np.random.default_rng(V)
    groups, dt = 30, np.float16 if kind == "f16" else np.float32
    x = (3 * rng.standard_normal((groups, 4, V))).astype(dt)
    x[:, 3] = x[:, 1]
    lse, top = lse64(x.astype(np.float64)), x.astype(np.float64).max(2)
    scores = np.full((groups, 4), -40, np.float32)
    scores[:, 1] = scores[:, 3] = -rng.random(groups)
    near = 2 * (np.arange(groups) % 2)
    g = np.arange(groups)
    scores[g, near] = (scores[:, 1].astype(np.float64) + (top[:, 1] - lse[:, 1])) - (top[g, near] - lse[g, near])
    best = scores.astype(np.float64) + (top - lse)
    got = select(gpu, kind, x, scores, None, 3, -1)
    for i in range(groups):
        if abs(best[i, near[i]] - best[i, 1]) <= 2 * EPS:
            continue
        _, p, t, _ = lc.select64(x[i].astype(np.float64), scores[i].astype(np.float64), None, 3, -1)
        assert np.array_equal(got[1][i], p) and np.array_equal(got[2][i], t), f"group {i}: {got[1][i]} for {p}"
