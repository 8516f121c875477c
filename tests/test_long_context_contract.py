"""Refusals of the long-context entries, decided on the host before any device call."""

from __future__ import annotations

import pytest

P = 0x1000  # dummy 16-byte aligned "device" pointer; never dereferenced here
PU = 0x1008  # and one that is not 16-byte aligned
BIG = 1 << 31


def _window(kind="q8", i=None, v=None, dims=(2, 3, 8, 2, 64), window=0, sinks=0, lens=(100, 128), scale=0.125,
            split=0):
    a = [P] * (6 if kind == "f16" else 8)
    if i is not None:
        a[i] = v
    return ("eng_attention_window_" + kind, *a, *dims, window, sinks, *lens, scale, split, None)


def _prefix(kind="q8", i=None, v=None, dims=(2, 4, 8, 2, 64), lens=(100, 128, 50, 64), scale=0.125, split=0):
    a = [P] * (8 if kind == "f16" else 12)
    if i is not None:
        a[i] = v
    return ("eng_attention_prefix_" + kind, *a, *dims, *lens, scale, split, None)


REFUSALS = [
    *[(_window("f16", i, None), f"attention_window: {n} is null")
      for i, n in enumerate(("q", "k_cache", "v_cache", "out", "pos")) if i != 5],
    *[(_window("q8", i, None), f"attention_window: {n} is null")
      for i, n in enumerate(("q", "k_cache", "v_cache", "k_scale/v_scale", "k_scale/v_scale", "out", "pos"))],
    (_window("f16", 1, PU), "caches must be 16-byte aligned"),
    (_window("q8", 2, PU), "caches must be 16-byte aligned"),
    (_window(dims=(-1, 3, 8, 2, 64)), "batch must be non-negative"),
    (_window(dims=(2, -3, 8, 2, 64)), "s_new must be non-negative"),
    (_window(dims=(2, 3, 0, 2, 64)), "n_heads must be positive"),
    (_window(dims=(2, 3, 8, 0, 64)), "n_kv_heads must be positive"),
    (_window(dims=(2, 3, 8, 3, 64)), "divisible by n_kv_heads"),
    (_window(dims=(2, 3, 8, 2, 96)), "head_dim must be 64 or 128"),
    (_window(window=-1), "window must be non-negative"),
    (_window(sinks=-1), "sinks must be non-negative"),
    (_window(lens=(-1, 128)), "max_kv_len must be non-negative"),
    (_window(lens=(129, 128)), "kv_max_seq_len < max_kv_len"),
    (_window(lens=(100, BIG)), "kv_max_seq_len must be below"),
    (_window(scale=float("nan")), "scale must be finite"),
    (_window(split=-1), "split_kv must be non-negative"),
    (_window(dims=(BIG, 3, 8, 2, 64)), "too many"),
    (_window(dims=(1 << 20, 1 << 20, 8, 2, 64)), "too many"),
    (_window(dims=(1, 1 << 29, 8, 2, 64)), "too many"),
    (_window(dims=(1 << 25, 1, 8, 8, 64)), "too many"),
    *[(_prefix("q8", i, None), f"attention_prefix: {n} is null") for i, n in enumerate(
        ("q", "k_prefix/v_prefix", "k_prefix/v_prefix", "k_prefix_scale/v_prefix_scale",
         "k_prefix_scale/v_prefix_scale", "prefix_len", "k_cache/v_cache", "k_cache/v_cache",
         "k_scale/v_scale", "k_scale/v_scale", "kv_len", "out"))],
    *[(_prefix("f16", i, None), f"attention_prefix: {n} is null") for i, n in enumerate(
        ("q", "k_prefix/v_prefix", "k_prefix/v_prefix", "prefix_len", "k_cache/v_cache", "k_cache/v_cache",
         "kv_len", "out"))],
    *[(_prefix("f16", i, PU), "caches must be 16-byte aligned") for i in (1, 2, 4, 5)],
    (_prefix(dims=(2, -4, 8, 2, 64)), "batch must be non-negative"),
    (_prefix(dims=(0, 4, 8, 2, 64)), "n_prefix must be positive"),
    (_prefix(dims=(2, 5, 8, 2, 64)), "batch must be divisible by n_prefix"),
    (_prefix(dims=(2, 4, 0, 2, 64)), "n_heads must be positive"),
    (_prefix(dims=(2, 4, 8, -2, 64)), "n_kv_heads must be positive"),
    (_prefix(dims=(2, 4, 9, 2, 64)), "divisible by n_kv_heads"),
    (_prefix(dims=(2, 4, 8, 2, 32)), "head_dim must be 64 or 128"),
    (_prefix(lens=(-1, 128, 50, 64)), "max_prefix_len must be non-negative"),
    (_prefix(lens=(100, 128, -50, 64)), "max_kv_len must be non-negative"),
    (_prefix(lens=(100, 99, 50, 64)), "prefix_max_seq_len < max_prefix_len"),
    (_prefix(lens=(100, 128, 50, 49)), "kv_max_seq_len < max_kv_len"),
    (_prefix(lens=(100, BIG, 50, 64)), "must be below"),
    (_prefix(lens=(100, 128, 50, BIG)), "must be below"),
    (_prefix(scale=float("inf")), "scale must be finite"),
    (_prefix(split=-2), "split_kv must be non-negative"),
    (_prefix(dims=(1, 1 << 30, 8, 2, 64)), "too many"),
    (_prefix(dims=(1, 1 << 25, 8, 8, 64)), "too many"),
]


@pytest.mark.parametrize("call,substr", REFUSALS, ids=[f"{i}-{c[0][4:]}" for i, (c, _) in enumerate(REFUSALS)])
def test_refusals(eng, call, substr):
    assert eng.status(*call) == 1
    assert substr in eng.last_error()


@pytest.mark.parametrize("call", [
    _window(dims=(0, 3, 8, 2, 64)),
    _window("f16", dims=(2, 0, 8, 2, 64)),
    _prefix(dims=(3, 0, 8, 2, 64)),
])
def test_nothing_to_do(eng, call):
    assert eng.status(*call) == 0
