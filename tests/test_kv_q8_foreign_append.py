"""Appending to blocks whose scale is no power of two (a cache written elsewhere): the
codes are those nearest to x / s, and to the old values over the new scale, with the
inputs a rounding of 2^-24 away from the middle between two codes."""

from __future__ import annotations

import numpy as np
import pytest

import narrow
from test_gpu_kv_q8 import Cache

N = 600  # blocks
F = np.float32


def middles(rng, n):
    """Values half-way between two e4m3 codes, 8.5 to 15.5."""
    return rng.integers(8, 16, n) + 0.5


def steps(n):
    """Signs and powers of two of a row: the same distance from a middle each."""
    d = np.arange(n)
    return np.where(d & 1, -1.0, 1.0) * np.exp2(-(d // 2 % 8))


def kept_scales(rng, D):
    """(x [N, D] float16, s [N] float32): x / s next to a middle, s above every scale
    that x needs."""
    x = rng.uniform(1, 2, N).astype(np.float16).astype(np.float64) * np.exp2(rng.integers(-3, 4, N))
    s = (x / middles(rng, N)).astype(F)
    s = np.nextafter(s, s * rng.integers(0, 3, N).astype(F))  # to zero, to itself, up
    return (x[:, None] * steps(D)).astype(np.float16), s


def grown_scales(rng, D):
    """(old codes [N, D], s_old [N] float32, new [N] powers of two): old values over the
    new scale next to a middle."""
    m = rng.integers(8, 15, N) + 0.5
    a = np.array([rng.integers(int(v + 1), 16) for v in m], np.float64)
    new = np.exp2(rng.integers(-6, 6, N))
    s = (m / a * new).astype(F)
    s = np.nextafter(s, s * rng.integers(0, 3, N).astype(F))
    return narrow.e4m3_encode(a[:, None] * steps(D)), s, new


def test_these_inputs_tell_the_roundings_apart():
    """A quotient or product rounded to fp32 first gives other codes, as does x (1 / s)."""
    rng = np.random.default_rng(1)
    x, s = kept_scales(rng, 64)
    want = narrow.e4m3_encode(x.astype(np.float64) / s[:, None].astype(np.float64))
    assert ((s.view(np.uint32) & 0x7FFFFF) != 0).mean() > 0.99  # hardly a power of two
    assert (narrow.e4m3_encode(x.astype(F) * (F(1) / s[:, None])) != want).mean() > 0.1
    assert (narrow.e4m3_encode(x.astype(F) / s[:, None]) != want).mean() > 0.1
    c, s, new = grown_scales(rng, 64)
    r = (s / new).astype(F)[:, None]
    want = narrow.e4m3_encode(narrow.e4m3_decode(c) * r.astype(np.float64))
    assert (narrow.e4m3_encode(narrow.e4m3_decode(c).astype(F) * r) != want).mean() > 0.1


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S", [1, 3])
def test_new_rows_under_a_kept_scale(gpu, D, S):
    rng = np.random.default_rng(D + S)
    c = Cache(gpu, rng, N, 1, 64, D)
    (xk, c.ks[:, 0, 1]), (xv, c.vs[:, 0, 1]) = kept_scales(rng, D), kept_scales(rng, D)
    for dev, host in zip(c.dev, (c.k, c.v, c.ks, c.vs)):
        dev.upload(host)
    rows = lambda x: np.repeat(x[:, None, None, :], S, 1)  # noqa: E731
    c.write(rows(xk), rows(xv), rng.integers(33, 60, N))
    c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_old_codes_under_a_grown_scale(gpu, D):
    rng = np.random.default_rng(D)
    c = Cache(gpu, rng, N, 1, 32, D)
    new = []
    for codes, scales in ((c.k, c.ks), (c.v, c.vs)):
        old, scales[:, 0, 0], top = grown_scales(rng, D)
        codes[:, 0, :9] = old[:, None]
        new.append(np.broadcast_to(400 * top[:, None, None, None], (N, 1, 1, D)).astype(np.float16))
    for dev, host in zip(c.dev, (c.k, c.v, c.ks, c.vs)):
        dev.upload(host)
    c.write(*new, np.full(N, 9))
    c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_any_scale_of_zero_or_more(gpu, D):
    """Scales from zero and the least subnormal to 2^24 and 1e30, infinities and NaN among
    the new rows and the old codes."""
    rng = np.random.default_rng(D + 9)
    s = np.concatenate([[0, 2.0**-149, 1e-42, 2.0**-126, 1e-30, 2.0**24, 1e30],
                        np.exp(rng.uniform(np.log(1e-6), np.log(3e3), 120))]).astype(F)
    B = s.size
    c = Cache(gpu, rng, B, 1, 32, D)
    c.ks[:, 0, 0], c.vs[:, 0, 0] = s, s[::-1]
    for dev, host in zip(c.dev, (c.k, c.v, c.ks, c.vs)):
        dev.upload(host)
    kn, vn = ((rng.standard_normal((B, 2, 1, D)) * np.exp2(rng.integers(-20, 12, (B, 1, 1, 1))))
              .astype(np.float16) for _ in range(2))
    kn[:, 1, 0, :3] = [np.nan, np.inf, -np.inf]
    c.write(kn, vn, np.full(B, 17))
    c.check()
