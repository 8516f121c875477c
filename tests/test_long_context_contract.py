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


# ---------------------------------------------------------------- beam search
def _select(kind="f32", i=None, v=None, ld=100, dims=(2, 4, 8, 100, 2)):
    a = [P] * 7
    if i is not None:
        a[i] = v
    return ("eng_beam_select_" + kind, a[0], ld, *a[1:], *dims, None)


def _reorder(kind="q8", change=(), dims=(2, 4, 2, 64, 100, 128)):
    n = 3 if kind == "f16" else 5
    a = [P + 4096 * i for i in range(4 * (n // 2))] + [P, P]  # (sources, destinations), parent, lengths
    for i, v in change:
        a[i] = v
    return ("eng_kv_cache_reorder_" + kind, *a, *dims, None)


BEAM_REFUSALS = [
    (_select("f32", 0, None), "logits is null"),
    (_select("f16", 1, None), "scores is null"),
    (_select("f32", 3, None), "out_scores/out_parent/out_token is null"),
    (_select("f32", 4, None), "out_scores/out_parent/out_token is null"),
    (_select("f32", 5, None), "out_scores/out_parent/out_token is null"),
    (_select("f32", 0, P + 2), "aligned to their type"),
    (_select("f16", 0, P + 1), "aligned to their type"),
    (_select(dims=(-1, 4, 8, 100, 2)), "batch must be non-negative"),
    (_select(dims=(2, 0, 8, 100, 2)), "beams must be 1 to 32"),
    (_select(dims=(2, 33, 8, 100, 2)), "beams must be 1 to 32"),
    (_select(dims=(2, 4, 0, 100, 2)), "n_out must be 1 to 64"),
    (_select(dims=(2, 4, 65, 100, 2)), "n_out must be 1 to 64"),
    (_select(dims=(2, 4, 8, 0, 2)), "vocab must be positive"),
    (_select(ld=BIG, dims=(2, 4, 8, BIG - 4097, 2)), "vocab must be positive and below"),
    (_select(dims=(2, 2, 8, 3, 2)), "n_out > beams * vocab"),
    (_select(ld=99), "ld < vocab"),
    (_select(dims=(2, 4, 8, 100, 100)), "eos >= vocab"),
    (_select(dims=(2, 4, 8, 100, -1)), "finished beams need eos"),
    (_select(dims=(1 << 22, 4, 8, 100, 2)), "too many logits"),
    *[(_reorder("q8", [(i, None)]), n) for i, n in enumerate(
        ["k_src/v_src is null"] * 2 + ["a scale buffer is null"] * 2 + ["k_dst/v_dst is null"] * 2
        + ["a scale buffer is null"] * 2 + ["parent is null", "kv_len is null"])],
    *[(_reorder("f16", [(i, None)]), n) for i, n in enumerate(
        ["k_src/v_src is null"] * 2 + ["k_dst/v_dst is null"] * 2 + ["parent is null", "kv_len is null"])],
    *[(_reorder("f16", [(i, PU)]), "16-byte aligned") for i in range(4)],
    (_reorder("f16", [(2, P)]), "all buffers in place, or none"),
    (_reorder("q8", [(4, P), (5, P + 4096)]), "all buffers in place, or none"),
    (_reorder(dims=(-2, 4, 2, 64, 100, 128)), "batch must be non-negative"),
    (_reorder(dims=(2, 0, 2, 64, 100, 128)), "beams must be 1 to 32"),
    (_reorder(dims=(2, 33, 2, 64, 100, 128)), "beams must be 1 to 32"),
    (_reorder(dims=(2, 4, 0, 64, 100, 128)), "n_kv_heads must be positive"),
    (_reorder(dims=(2, 4, 2, 80, 100, 128)), "head_dim must be 64 or 128"),
    (_reorder(dims=(2, 4, 2, 64, -1, 128)), "max_kv_len must be non-negative"),
    (_reorder(dims=(2, 4, 2, 64, 129, 128)), "kv_max_seq_len < max_kv_len"),
    (_reorder(dims=(2, 4, 2, 64, 100, BIG)), "kv_max_seq_len must be below"),
    (_reorder(dims=(1 << 23, 4, 2, 64, 100, 128)), "too many"),
]


@pytest.mark.parametrize("call,substr", BEAM_REFUSALS,
                         ids=[f"{i}-{c[0][4:]}" for i, (c, _) in enumerate(BEAM_REFUSALS)])
def test_beam_refusals(eng, call, substr):
    assert eng.status(*call) == 1
    assert substr in eng.last_error()


@pytest.mark.parametrize("call", [
    _select(dims=(0, 4, 8, 100, 2)),
    _reorder(dims=(0, 4, 2, 64, 100, 128)),
    _reorder("f16", dims=(2, 4, 2, 64, 0, 128)),
])
def test_beam_nothing_to_do(eng, call):
    assert eng.status(*call) == 0
