"""GPU tests of eng_attention_window_* with counts of new queries below zero: no row is there,
whatever the count times a group of query heads comes to in 32 bits."""

from __future__ import annotations

import numpy as np
import pytest

import long_context as lc
import test_gpu_attention_window as window

GPU = pytest.mark.gpu
COUNTS = [-1, -(2**31), -(2**31) + 1, -(2**30), -715827883, -1431655766, -858993460, -429496730]


def test_some_of_the_counts_wrap_to_a_number_of_rows():
    """What the counts are chosen for: -715827883 x 3 is 2^31 - 1 modulo 2^32."""
    wrapped = [int(np.int64(n * g).astype(np.int32)) for n in COUNTS for g in (3, 5)]
    assert (2**31 - 1) in wrapped and sum(w > 0 for w in wrapped) >= 4


@GPU
@pytest.mark.parametrize("kind", ["f16", "q8"])
@pytest.mark.parametrize("group", [3, 5])
@pytest.mark.parametrize("S,split", [(1, 1), (1, 3), (40, 1), (40, 3)])
def test_counts_below_zero(gpu, kind, group, S, split):
    rng = np.random.default_rng(group + S)
    B, G, D = len(COUNTS) + 1, 2, 64
    cache = lc.Cache(gpu, rng, kind, B, G, 128, D, [128] * B)
    q = rng.standard_normal((B, S, group * G, D)).astype(np.float16).astype(np.float64)
    pos = [60] * B
    n_new = [*COUNTS, S]  # the last sequence is there
    got = window.call(gpu, kind, q, cache, pos, n_new, 0, 0, 128, 0.125, split)
    assert (got.view(np.uint16)[:-1] == 0x7777).all()
    want = lc.window64(q, cache, pos, [max(n, 0) for n in n_new], 0, 0, 128, 0.125, rows=[0, S - 1])
    assert len(want) == group * G * len({0, S - 1})
    lc.check(got, want, "counts")
