"""GPU test of a step of beams that are not equally long: caches reordered, the lengths
gathered by parent, the next token appended and attended over, as the integration guide has it.
Tokens behind a length hold NaN codes, and their blocks other beams' scales."""

from __future__ import annotations

import numpy as np
import pytest

import long_context as lc
import narrow

pytestmark = pytest.mark.gpu


class View:
    def __init__(self, values, vmax):
        self.values, self.vmax = values, vmax


@pytest.mark.parametrize("kind", ["f16", "q8"])
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("lens,parent", [
    ([7, 33, 40, 64], [2, 0, 0, 3]),     # a shorter one over a longer one, in one block
    ([95, 1, 31, 32], [1, 2, 3, 1]),
    ([50, 40, 45], [1, 2, 0]),           # a rotation, lengths of one block
    ([0, 20], [1, 0]),                   # an empty one
])
def test_the_next_step_sees_its_parent_and_its_token(gpu, kind, in_place, lens, parent):
    rng = np.random.default_rng(sum(lens))
    B, H, G, D, room = len(lens), 4, 2, 64, 96
    src = lc.Cache(gpu, rng, kind, B, G, room, D, lens)
    dst = src if in_place else lc.Cache(gpu, rng, kind, B, G, room, D, [0] * B)
    dp, dl = gpu.upload(np.array(parent, np.int32)), gpu.upload(np.array(lens, np.int32))
    gpu.call("eng_kv_cache_reorder_" + kind, *src.ptrs, *dst.ptrs, dp.ptr, dl.ptr, 1, B, G, D, room, room, None)
    pos = np.array(lens)[parent]
    k, v = rng.standard_normal((2, B, 1, G, D)).astype(np.float16)
    # a parent of no token leaves its place as it was: nothing there counts
    values = [np.where((np.arange(room) < pos[:, None])[:, None, :, None], a[parent], np.nan) for a in src.values]
    dk, dv, dpos = gpu.upload(k.view(np.uint16)), gpu.upload(v.view(np.uint16)), gpu.upload(pos.astype(np.int32))
    if kind == "q8":
        gpu.call("eng_kv_cache_write_q8", dk.ptr, dv.ptr, *dst.ptrs, dpos.ptr, None, B, 1, G, D, room, None)
        raw, scales = [a[parent].copy() for a in src.raw], [a[parent].copy() for a in src.scales]
        for x, c, s in zip((k, v), raw, scales):
            narrow.kv_write(x.astype(np.float64), c, s, pos, None)
        values = [narrow.kv_values(c, s) for c, s in zip(raw, scales)]
        vmax = 448 * np.nanmax(np.where(np.isnan(scales[1]), 0, scales[1]), 2)
    else:
        for b in range(B):
            at, row = b * G * room * D * 2, b * G * D * 2
            gpu.call("eng_kv_cache_write_f16", dk.ptr + row, dv.ptr + row, dst.ptrs[0] + at, dst.ptrs[1] + at, 1, G, D,
                     int(pos[b]), room, None)
            for x, a in zip((k, v), values):
                a[b, :, pos[b]] = x[b, 0]
        vmax = np.nanmax(np.abs(values[1]), (2, 3))
    q = rng.standard_normal((B, 1, H, D)).astype(np.float16)
    dq, do = gpu.upload(q.view(np.uint16)), gpu.empty(q.shape, np.uint16)
    gpu.call("eng_attention_window_" + kind, dq.ptr, *dst.ptrs, do.ptr, dpos.ptr, None, B, 1, H, G, D, 0, 0, room,
             room, 0.125, 0, None)
    gpu.sync()
    want = lc.window64(q.astype(np.float64), View(values, vmax), pos, None, 0, 0, room, 0.125)
    lc.check(do.download().view(np.float16), want, "next step")
    assert all(np.isfinite(y).all() for y, _ in want.values())
