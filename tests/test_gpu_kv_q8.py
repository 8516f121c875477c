"""GPU tests of the 8-bit KV cache: the append, compared code for code with the
definition, and the decode attention over it, within narrow.attend64's bound."""

from __future__ import annotations

import numpy as np
import pytest

import helpers
import narrow

pytestmark = pytest.mark.gpu


class Cache:
    """Host and device copies of K and V caches, written in step."""

    def __init__(self, gpu, rng, B, G, L, D):
        self.gpu, self.shape = gpu, (B, G, L, D)
        nb = -(-L // 32)
        fill = lambda: rng.integers(0, 256, (B, G, L, D)).astype(np.uint8)  # noqa: E731
        self.k, self.v = fill(), fill()
        self.ks = np.exp2(rng.integers(-15, 9, (B, G, nb))).astype(np.float32)
        self.vs = np.exp2(rng.integers(-15, 9, (B, G, nb))).astype(np.float32)
        self.dev = [gpu.upload(a) for a in (self.k, self.v, self.ks, self.vs)]

    def write(self, kn, vn, pos, n_new=None, stream=None):
        """kn, vn [B, S, G, D] float16."""
        gpu = self.gpu
        B, S, G, D = kn.shape
        dk, dv = gpu.upload(kn.view(np.uint16)), gpu.upload(vn.view(np.uint16))
        dp = gpu.upload(np.asarray(pos, np.int32))
        dn = None if n_new is None else gpu.upload(np.asarray(n_new, np.int32))
        gpu.call("eng_kv_cache_write_q8", dk.ptr, dv.ptr, *[d.ptr for d in self.dev], dp.ptr,
                 None if dn is None else dn.ptr, B, S, G, D, self.shape[2], stream)
        gpu.sync()
        narrow.kv_write(kn.astype(np.float64), self.k, self.ks, pos, n_new)
        narrow.kv_write(vn.astype(np.float64), self.v, self.vs, pos, n_new)

    def check(self):
        k, v, ks, vs = (d.download() for d in self.dev)
        assert np.array_equal(ks, self.ks) and np.array_equal(vs, self.vs)
        assert narrow.same_codes(k, self.k), "K codes"
        assert narrow.same_codes(v, self.v), "V codes"


def rows(rng, B, S, G, D, sigma=1.0):
    return (sigma * rng.standard_normal((B, S, G, D))).astype(np.float16)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,S,G,L,pos,n_new", [
    (1, 1, 1, 1, [0], None),
    (1, 1, 3, 40, [31], None),
    (1, 1, 2, 40, [32], None),
    (3, 1, 2, 100, [0, 50, 99], None),
    (2, 5, 1, 70, [30, 65], None),
    (2, 33, 3, 128, [0, 31], None),
    (2, 64, 1, 64, [0, 0], None),
    (3, 70, 2, 200, [17, 100, 0], [70, 1, 33]),
    (4, 9, 2, 64, [0, 5, 60, -1], [0, 9, 9, 9]),        # nothing, all, past the end, inactive
    (3, 4, 1, 33, [31, 32, 33], [4, 3, 2]),             # runs past the cache's end
    (2, 6, 2, 96, [10, 20], [99, -3]),                  # counts past s_new and below zero
])
def test_write_equals_the_definition(gpu, D, B, S, G, L, pos, n_new):
    rng = np.random.default_rng(B * 100 + S + G + L + D)
    c = Cache(gpu, rng, B, G, L, D)
    c.write(rows(rng, B, S, G, D), rows(rng, B, S, G, D, 30.0), pos, n_new)
    c.check()


@pytest.mark.parametrize("D", [64, 128])
def test_write_token_by_token_with_growing_scales(gpu, D):
    """70 tokens one at a time, magnitudes from 2^-20 to 2^15 and back: scales grow
    inside a block, earlier codes are brought to them, and a new block starts afresh."""
    rng = np.random.default_rng(D)
    B, G = 2, 2
    c = Cache(gpu, rng, B, G, 100, D)
    pos = np.array([0, 13])
    for t in range(70):
        sigma = 2.0 ** rng.integers(-20, 14)
        c.write(rows(rng, B, 1, G, D, sigma), rows(rng, B, 1, G, D, 2.0 ** (t % 9)), pos + t)
    c.check()
    # rewound: the block's scale stays at least what its earlier tokens need
    c.write(rows(rng, B, 3, G, D), rows(rng, B, 3, G, D), [40, 7])
    c.check()


def test_write_special_values(gpu):
    rng = np.random.default_rng(5)
    B, S, G, D = 1, 8, 1, 64
    c = Cache(gpu, rng, B, G, 64, D)
    x = rows(rng, B, S, G, D)
    x[0, 1, 0, :4] = [np.nan, np.inf, -np.inf, -0.0]
    x[0, 2, 0, :] = np.finfo(np.float16).max
    x[0, 3, 0, :] = np.finfo(np.float16).smallest_subnormal
    y = np.full_like(x, np.inf)  # a block with no finite value
    c.write(x, y, [3])
    c.check()
    c.write(np.zeros_like(x), x[:, ::-1].copy(), [32])
    c.check()
    c.write(x[:, :1] * 0, x[:, 1:2], [40])
    c.check()


def test_write_every_half(gpu):
    bits = np.arange(65536, dtype=np.uint32).astype(np.uint16)
    rng = np.random.default_rng(6)
    a = rng.permutation(bits).view(np.float16).reshape(1, 512, 1, 128)
    b = np.sort(np.where(np.isfinite(a), a, 0).reshape(-1)).reshape(1, 512, 1, 128)  # narrow ranges
    c = Cache(gpu, rng, 1, 1, 512, 128)
    c.write(a, b, [0])
    c.check()


# ---------------------------------------------------------------- attention
def filled(gpu, rng, B, H, G, D, L, room=None):
    room = room or L
    c = Cache(gpu, rng, B, G, room, D)
    if L:
        c.write(rows(rng, B, L, G, D), rows(rng, B, L, G, D), [0] * B)
    q = rng.standard_normal((B, H, D)).astype(np.float16)
    return c, q


def attend(gpu, c, q, lens, max_len, scale=None, split=0, stream=None, skew=0):
    B, H, D = q.shape
    G, room = c.shape[1], c.shape[2]
    scale = 1 / np.sqrt(D) if scale is None else scale
    dq = gpu.upload(np.concatenate([np.zeros(skew, np.uint16), q.view(np.uint16).reshape(-1)]))
    dl = gpu.upload(np.asarray(lens, np.int32))
    out = gpu.empty(B * H * D + 32 + skew, np.uint16)
    out.fill_bytes(0x5A)
    k, v, ks, vs = (d.ptr for d in c.dev)
    gpu.call("eng_attention_decode_q8", dq.ptr + 2 * skew, k, v, ks, vs, out.ptr + 2 * skew, dl.ptr,
             B, H, G, D, max_len, room, scale, split, stream)
    gpu.sync()
    o = out.download()
    assert (o[skew + B * H * D:] == 0x5A5A).all() and (o[:skew] == 0x5A5A).all(), "written outside out"
    return o[skew:skew + B * H * D].view(np.float16).reshape(B, H, D)


def check_attend(gpu, c, q, lens, max_len, scale=None, split=0, skew=0):
    D = q.shape[2]
    scale = 1 / np.sqrt(D) if scale is None else scale
    got = attend(gpu, c, q, lens, max_len, scale, split, skew=skew)
    used = np.clip(lens, 0, max_len)
    y, bound = narrow.attend64(q.astype(np.float64), c.k, c.v, c.ks, c.vs, used, scale)
    helpers.assert_within(got, y, bound, f"lens {list(lens)[:6]} split {split}")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("L", [1, 2, 31, 32, 33, 63, 65, 127, 129, 255, 300, 513, 1025])
def test_attention_lengths(gpu, L, D):
    rng = np.random.default_rng(L + D)
    c, q = filled(gpu, rng, 1, 8, 2, D, L, L + 7)
    check_attend(gpu, c, q, [L], L)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 5, 8, 15, 16, 17, 33])
def test_attention_groups(gpu, group, D):
    rng = np.random.default_rng(group)
    c, q = filled(gpu, rng, 2, 3 * group, 3, D, 150)
    check_attend(gpu, c, q, [150, 77], 150)


@pytest.mark.parametrize("split", [0, 1, 2, 3, 7, 16, 40, 256, 100000])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_splits(gpu, split, D):
    rng = np.random.default_rng(split % 97)
    c, q = filled(gpu, rng, 4, 8, 4, D, 1300)
    check_attend(gpu, c, q, [1300, 0, 1, 640], 1300, split=split)


def test_attention_ragged_and_clamped_lengths(gpu):
    rng = np.random.default_rng(9)
    c, q = filled(gpu, rng, 7, 12, 4, 64, 400, 500)
    check_attend(gpu, c, q, [0, 1, 32, 399, 400, -5, 250], 400)
    check_attend(gpu, c, q, [0, 1, 32, 399, 400, -5, 250], 100)  # longer ones are taken as 100
    assert (attend(gpu, c, q, [3] * 7, 0) == 0).all()


@pytest.mark.parametrize("split", [1, 5])
def test_attention_ignores_what_lies_behind_a_sequence(gpu, split):
    """NaN codes and scales behind the last token must not reach the result."""
    rng = np.random.default_rng(10)
    c, q = filled(gpu, rng, 2, 4, 2, 128, 320)
    lens = [45, 257]
    c.k[0, :, 45:] = 0x7F
    c.v[0, :, 45:] = 0xFF
    c.k[1, :, 257:] = 0x7F
    c.v[1, :, 257:] = 0x7F
    for s in (c.ks, c.vs):
        s[0, :, 2:] = np.nan
        s[1, :, 9:] = np.nan
    c.dev = [gpu.upload(a) for a in (c.k, c.v, c.ks, c.vs)]
    check_attend(gpu, c, q, lens, 320, split=split)


def test_attention_propagates_nan_of_its_own_tokens(gpu):
    rng = np.random.default_rng(11)
    c, q = filled(gpu, rng, 1, 4, 2, 64, 100)
    c.k[0, 0, 50, 3] = 0x7F      # one K value of head 0: both its query heads
    c.v[0, 1, 99, 7] = 0xFF      # one V value of head 1: dim 7 of its query heads
    c.dev = [gpu.upload(a) for a in (c.k, c.v, c.ks, c.vs)]
    for split in (1, 2, 0):
        got = attend(gpu, c, q, [100], 100, split=split)
        assert np.isnan(got[0, :2]).all()
        assert np.isnan(got[0, 2:, 7]).all()
        assert np.isfinite(np.delete(got[0, 2:], 7, axis=1)).all()


@pytest.mark.parametrize("scale", [0.0, -0.5, 4.0])
def test_attention_scales(gpu, scale):
    rng = np.random.default_rng(12)
    c, q = filled(gpu, rng, 1, 4, 4, 64, 200)
    check_attend(gpu, c, q, [200], 200, scale=scale)


def test_attention_unlike_block_scales(gpu):
    """Blocks whose magnitudes run from 2^-15 to 2^9, and one key that takes nearly
    all of the weight."""
    rng = np.random.default_rng(13)
    B, H, G, D, L = 1, 6, 2, 128, 600
    c = Cache(gpu, rng, B, G, L, D)
    mag = np.exp2(rng.integers(-15, 10, L // 32 + 1)).repeat(32)[:L, None, None]
    kn = rng.standard_normal((L, G, D)).astype(np.float16)
    kn[400] *= 4
    vn = (rng.standard_normal((L, G, D)) * mag).astype(np.float16)
    c.write(kn[None], vn[None], [0])
    q = rng.standard_normal((B, H, D)).astype(np.float16)
    for split in (0, 1, 4):
        check_attend(gpu, c, q, [L], L, split=split)


def test_attention_over_a_cache_written_elsewhere(gpu):
    """Scales that are no powers of two, and zero for blocks of K, of V and of both."""
    rng = np.random.default_rng(17)
    B, H, G, D, L = 2, 6, 2, 64, 300
    c = Cache(gpu, rng, B, G, L, D)
    finite = lambda: (rng.integers(0, 2, (B, G, L, D)) * 128 + rng.integers(0, 127, (B, G, L, D))).astype(np.uint8)  # noqa: E731
    c.k, c.v = finite(), finite()
    c.ks = (0.002 * rng.random(c.ks.shape)).astype(np.float32)
    c.vs = (0.01 * rng.random(c.vs.shape)).astype(np.float32)
    c.ks[0, 0, 2:4] = 0
    c.vs[0, 0, 3:5] = 0
    c.vs[1, 1, :] = 0
    c.dev = [gpu.upload(a) for a in (c.k, c.v, c.ks, c.vs)]
    q = (0.3 * rng.standard_normal((B, H, D))).astype(np.float16)
    for split in (0, 1, 3):
        check_attend(gpu, c, q, [L, 217], L, split=split)


@pytest.mark.parametrize("skew", [1, 4])
def test_attention_unaligned_q_and_out(gpu, skew):
    rng = np.random.default_rng(14)
    c, q = filled(gpu, rng, 2, 4, 2, 64, 90)
    check_attend(gpu, c, q, [90, 33], 90, skew=skew)


def test_offsets_past_32_bits(gpu):
    """Two sequences of 17 million tokens' room: the second one's cache begins past
    2^31 bytes, and its tokens at the end of the room past 2^32."""
    rng = np.random.default_rng(15)
    B, H, G, D, room = 2, 4, 1, 128, 17 << 20
    nb = room // 32
    kc, vc = gpu.empty(B * room * D, np.uint8), gpu.empty(B * room * D, np.uint8)
    ks, vs = gpu.empty(B * nb, np.float32), gpu.empty(B * nb, np.float32)
    S = 40
    kn, vn = rows(rng, B, S, G, D), rows(rng, B, S, G, D)
    dk, dv = gpu.upload(kn.view(np.uint16)), gpu.upload(vn.view(np.uint16))
    dp = gpu.upload(np.array([-1, 0], np.int32))
    args = [kc.ptr, vc.ptr, ks.ptr, vs.ptr]
    gpu.call("eng_kv_cache_write_q8", dk.ptr, dv.ptr, *args, dp.ptr, None, B, S, G, D, room, None)
    at = room - 32  # eight of the forty are past the end
    dp2 = gpu.upload(np.array([-1, at], np.int32))
    gpu.call("eng_kv_cache_write_q8", dk.ptr, dv.ptr, *args, dp2.ptr, None, B, S, G, D, room, None)
    gpu.sync()
    small = np.zeros((1, G, 64, D), np.uint8)
    smalls = np.zeros((1, G, 2), np.float32)
    narrow.kv_write(kn[1:].astype(np.float64), small, smalls, [32], None)
    got = np.empty(64 * D, np.uint8)
    gpu.call("eng_memcpy_d2h", got.ctypes.data, kc.ptr + (2 * room - 64) * D, got.nbytes)
    assert narrow.same_codes(got.reshape(64, D)[32:], small[0, 0, 32:])
    q = rng.standard_normal((B, H, D)).astype(np.float16)
    dq, dl = gpu.upload(q.view(np.uint16)), gpu.upload(np.array([0, S], np.int32))
    out = gpu.empty((B, H, D), np.uint16)
    gpu.call("eng_attention_decode_q8", dq.ptr, *args, out.ptr, dl.ptr, B, H, G, D, S, room,
             1 / np.sqrt(D), 0, None)
    gpu.sync()
    o = out.download().view(np.float16)
    assert (o[0] == 0).all()
    k8, v8 = np.zeros((1, G, 64, D), np.uint8), np.zeros((1, G, 64, D), np.uint8)
    k8s, v8s = np.ones((1, G, 2), np.float32), np.ones((1, G, 2), np.float32)
    narrow.kv_write(kn[1:].astype(np.float64), k8, k8s, [0], None)
    narrow.kv_write(vn[1:].astype(np.float64), v8, v8s, [0], None)
    y, bound = narrow.attend64(q[1:].astype(np.float64), k8, v8, k8s, v8s, [S], 1 / np.sqrt(D))
    helpers.assert_within(o[1:], y, bound, "second sequence")
    for d in (kc, vc, ks, vs):
        d.free()


def test_two_streams_with_splits_at_once(gpu):
    """Each stream has its own scratch for the splits' states."""
    rng = np.random.default_rng(16)
    c, q = filled(gpu, rng, 2, 8, 2, 128, 900)
    q2 = rng.standard_normal(q.shape).astype(np.float16)
    want = attend(gpu, c, q, [900, 512], 900, split=9), attend(gpu, c, q2, [900, 512], 900, split=9)
    with gpu.stream() as s1, gpu.stream() as s2:
        B, H, D = q.shape
        dl = gpu.upload(np.array([900, 512], np.int32))
        dq = [gpu.upload(x.view(np.uint16)) for x in (q, q2)]
        out = [gpu.empty((B, H, D), np.uint16) for _ in range(2)]
        gpu.sync()
        for _ in range(20):
            for i, s in enumerate((s1, s2)):
                gpu.call("eng_attention_decode_q8", dq[i].ptr, *[d.ptr for d in c.dev], out[i].ptr,
                         dl.ptr, B, H, 2, D, 900, 900, 1 / np.sqrt(D), 9, s.handle)
        s1.sync()
        s2.sync()
        for i in range(2):
            assert np.array_equal(out[i].download().view(np.float16), want[i])
