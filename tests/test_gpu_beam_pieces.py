"""GPU tests of eng_beam_select_* in pieces of two and of four steps of 4096 logits, which
many rows take: rows that end inside each step, lists that grow over steps, NaN and -inf in a
later step."""

from __future__ import annotations

import numpy as np
import pytest

from helpers import U32
from test_gpu_beam import select

pytestmark = pytest.mark.gpu
KINDS = pytest.mark.parametrize("kind", ["f32", "f16"])
STEP = 4096


def steps_of(cus, rows, n_out, V):
    """The launcher's rule for the steps of a piece."""
    pieces = lambda n: -(-(-(-V // STEP)) // n)  # noqa: E731
    per = 4
    while per > 1 and rows * pieces(per) < 2 * cus:
        per //= 2
    while per < 4 and pieces(per) * n_out > 256 and rows * pieces(2 * per) >= cus:
        per *= 2
    return per


def expected(x, scores, n_out):
    """(scores, parent, token) of one group of live beams, in 64 bits: the n_out best of each
    beam by (logit, lowest token), then those by (score, beam)."""
    x = x.astype(np.float64)
    score, parent, token = [], [], []
    for b, row in enumerate(x):
        at = np.lexsort((np.arange(len(row)), -row))[:n_out]
        live = not np.isnan(row).any() and np.isfinite(row.max())
        lse = row.max() + np.log(np.exp(row - row.max()).sum()) if live else 0.0
        score.append(float(scores[b]) + (row[at] - lse) if live else np.full(len(at), -np.inf))
        parent.append(np.full(len(at), b))
        token.append(at if live else np.arange(len(at)))
    score, parent, token = (np.concatenate(a) for a in (score, parent, token))
    rank = np.concatenate([np.arange(c) for c in np.bincount(parent)])
    at = np.lexsort((rank, parent, -score))[:n_out]
    return score[at], parent[at], token[at]


def check(gpu, kind, per, groups, beams, n_out, V, x=None, scores=None, ld=None, shift=0):
    assert steps_of(gpu.cu_count(), groups * beams, n_out, V) == per
    rng = np.random.default_rng(V + n_out)
    dt = np.float16 if kind == "f16" else np.float32
    x = (3 * rng.standard_normal((groups, beams, V), np.float32)).astype(dt) if x is None else x.astype(dt)
    scores = (-10 - 4 * rng.random((groups, beams))).astype(np.float32) if scores is None else scores
    got = select(gpu, kind, x, scores, None, n_out, -1, ld, shift)
    # fp32 sums, as derived in test_gpu_beam_near_ties
    wide = (1.22 * np.log(V) + 10) * U32
    for g in range(groups):
        s, p, t = expected(x[g], scores[g], n_out)
        assert np.array_equal(got[1][g], p), f"group {g}: parents"
        assert np.array_equal(got[2][g], t), f"group {g}: tokens"
        fin = np.isfinite(s)
        assert np.array_equal(got[0][g][~fin], s[~fin])
        assert (np.abs(got[0][g][fin] - s[fin]) <= U32 * np.abs(s[fin]) + wide).all()


# a piece of four steps is 16384 logits: rows end in the second one's first to fourth step
FOUR = [(32, 8, 16384 + 7), (8, 32, 16384 + STEP + 100), (256, 1, 16384 + 2 * STEP + 5), (16, 16, 16384 + 3 * STEP + 77),
        (32, 8, 32768)]
# of two steps 8192, in the fourth one
TWO = [(16, 8, 3 * 8192 + 1), (4, 32, 3 * 8192 + STEP + 9), (128, 1, 32768)]


@KINDS
@pytest.mark.parametrize("groups,beams,V,per", [(*c, 4) for c in FOUR] + [(*c, 2) for c in TWO])
@pytest.mark.parametrize("n_out", [1, 12])
def test_rows_that_end_in_each_step(gpu, kind, groups, beams, V, per, n_out):
    check(gpu, kind, per, groups, beams, n_out, V)


@KINDS
@pytest.mark.parametrize("groups,beams,V,per", [(*FOUR[1], 4), (*FOUR[3], 4), (*TWO[1], 2)])
def test_64_of_them(gpu, kind, groups, beams, V, per):
    check(gpu, kind, per, groups, beams, 64, V)


def test_a_large_vocabulary_and_many_candidates(gpu):
    check(gpu, "f32", 4, 8, 4, 20, 152064)  # pieces doubled for the join's sake
    check(gpu, "f16", 2, 8, 4, 8, 152064)


@KINDS
@pytest.mark.parametrize("groups,beams,V,per", [(*FOUR[2], 4), (*FOUR[1], 4), (*TWO[0], 2)])
@pytest.mark.parametrize("ld,shift", [(1, 0), (64, 3)])
def test_rows_without_alignment(gpu, kind, groups, beams, V, per, ld, shift):
    check(gpu, kind, per, groups, beams, 9, V, ld=(V + ld) | 1, shift=shift)


@KINDS
@pytest.mark.parametrize("groups,beams,V,per", [(*FOUR[1], 4), (*FOUR[4], 4), (*TWO[1], 2)])
@pytest.mark.parametrize("order", ["equal", "rising", "falling", "few values", "late"])
@pytest.mark.parametrize("n_out", [5, 64])
def test_lists_that_grow_over_the_steps(gpu, kind, groups, beams, V, per, order, n_out):
    i = np.arange(V)
    row = {"equal": np.zeros(V), "rising": i / 4096.0, "falling": -i / 4096.0, "few values": (i * 7919) % 5,
           "late": np.where(i >= V - 200, 3.0, (i * 31) % 97 / 97)}[order]
    x = np.broadcast_to(row.astype(np.float32), (groups, beams, V))
    rng = np.random.default_rng(V)
    # (beams half a unit apart: none tie)
    scores = np.stack([rng.permutation(beams) for _ in range(groups)]).astype(np.float32) * -0.5
    check(gpu, kind, per, groups, beams, n_out, V, x, scores)


@KINDS
@pytest.mark.parametrize("groups,beams,V,per", [(*FOUR[1], 4), (*FOUR[3], 4), (*TWO[1], 2)])
def test_special_values_in_later_steps(gpu, kind, groups, beams, V, per):
    rng = np.random.default_rng(3)
    x = (3 * rng.standard_normal((groups, beams, V), np.float32))
    x[0, 0, STEP + 5] = np.nan
    x[0, 1, V - 1] = np.nan
    x[0, 2, 2 * STEP + 3] = np.inf
    x[0, 3, :STEP] = -np.inf           # nothing in the first step
    x[1, :, STEP + 50:] = -np.inf      # nothing behind the second
    x[1, 1] = -np.inf
    x[2, 0, :V - 3] = -np.inf          # three left, at the end
    x[3, :, ::2] = np.finfo(np.float16).min
    check(gpu, kind, per, groups, beams, 12, V, x)
