"""The 4-bit weight and 8-bit cache entries' refusals (decided on the host, before
any device call), and the tests' own statements of the formats."""

from __future__ import annotations

import numpy as np
import pytest

import narrow

P = 0x1000  # dummy 16-byte aligned "device" pointer; never dereferenced here
PU = 0x1008  # and one that is not 16-byte aligned
W8 = (P, P, P, P, P, P, P, None)  # k_new, v_new, caches, scales, pos, n_new


def _write(i=None, v=None, dims=(2, 3, 4, 64, 128)):
    a = list(W8)
    if i is not None:
        a[i] = v
    return ("eng_kv_cache_write_q8", *a, *dims, None)


def _attend(i=None, v=None, dims=(2, 8, 2, 64, 100, 128), scale=0.125, split=0):
    a = [P] * 7
    if i is not None:
        a[i] = v
    return ("eng_attention_decode_q8", *a, *dims, scale, split, None)


REFUSALS = [
    (("eng_mx4_quantize_f32", None, P, P, 4, 4, None), "null device pointer"),
    (("eng_mx4_quantize_f32", P, None, P, 4, 4, None), "null"),
    (("eng_mx4_quantize_f16", P, P, None, 4, 4, None), "null"),
    (("eng_mx4_quantize_f16", P, P, P, -1, 4, None), "negative dimension"),
    (("eng_mx4_quantize_f32", P, P, P, 4, -1, None), "negative dimension"),
    (("eng_mx4_quantize_f32", P, PU, P, 4, 4, None), "codes must be 16-byte aligned"),
    (("eng_mx4_quantize_f32", P, P, P, 1 << 40, 1 << 30, None), "too large"),
    (("eng_mx4_dequantize_f32", None, P, P, 4, 4, None), "null"),
    (("eng_mx4_dequantize_f16", P, P, None, 4, 4, None), "null"),
    (("eng_mx4_dequantize_f16", P, P, P, 4, -4, None), "negative dimension"),
    (("eng_mx4_dequantize_f32", PU, P, P, 4, 4, None), "aligned"),
    (("eng_linear_mx4w_nk", None, P, P, P, 1, 4, 4, None), "linear_mx4w: null device pointer"),
    (("eng_linear_mx4w_nk", P, None, P, P, 1, 4, 4, None), "null"),
    (("eng_linear_mx4w_nk", P, P, None, P, 1, 4, 4, None), "null"),
    (("eng_linear_mx4w_nk", P, P, P, None, 1, 4, 4, None), "null"),
    (("eng_linear_mx4w_nk", P, P, P, P, -1, 4, 4, None), "negative dimension"),
    (("eng_linear_mx4w_nk", P, P, P, P, 1, -4, 4, None), "negative dimension"),
    (("eng_linear_mx4w_nk", P, P, P, P, 1, 4, -4, None), "negative dimension"),
    (("eng_linear_mx4w_nk", P, PU, P, P, 1, 4, 4, None), "codes must be 16-byte aligned"),
    (("eng_linear_mx4w_nk", P, P, P, P, 1, 4, 1 << 31, None), "K too large"),
    (("eng_rmsnorm_linear_mx4w_nk", None, P, P, P, P, 1, 4, 4, 1e-5, None), "null"),
    (("eng_rmsnorm_linear_mx4w_nk", P, None, P, P, None, 1, 4, 4, 1e-5, None), "null"),
    (("eng_rmsnorm_linear_mx4w_nk", P, P, P, P, P, 1, -4, 4, 1e-5, None), "negative dimension"),
    (("eng_rmsnorm_linear_mx4w_nk", P, P, P, P, P, 1, 4, 4, -1.0, None), "eps must be non-negative"),
    (("eng_rmsnorm_linear_mx4w_nk", P, P, P, P, P, 1, 4, 4, float("nan"), None), "eps"),
    (_write(0, None), "k_new/v_new is null"),
    (_write(1, None), "k_new/v_new is null"),
    (_write(2, None), "k_cache/v_cache is null"),
    (_write(3, None), "k_cache/v_cache is null"),
    (_write(4, None), "k_scale/v_scale is null"),
    (_write(5, None), "k_scale/v_scale is null"),
    (_write(6, None), "pos is null"),
    (_write(0, PU), "aligned"),
    (_write(1, PU), "aligned"),
    (_write(2, PU), "aligned"),
    (_write(3, PU), "aligned"),
    (_write(dims=(-1, 3, 4, 64, 128)), "batch must be non-negative"),
    (_write(dims=(2, -3, 4, 64, 128)), "s_new must be non-negative"),
    (_write(dims=(2, 3, 0, 64, 128)), "n_kv_heads must be positive"),
    (_write(dims=(2, 3, 4, 32, 128)), "head_dim must be 64 or 128"),
    (_write(dims=(2, 3, 4, 64, -1)), "kv_max_seq_len"),
    (_write(dims=(2, 3, 4, 64, 1 << 31)), "kv_max_seq_len"),
    (_write(dims=(2, 129, 4, 64, 128)), "kv_max_seq_len < s_new"),
    (_write(dims=(1 << 30, 3, 4, 64, 128)), "too many"),
    (_attend(0, None), "q is null"),
    (_attend(1, None), "k_cache is null"),
    (_attend(2, None), "v_cache is null"),
    (_attend(3, None), "k_scale/v_scale is null"),
    (_attend(4, None), "k_scale/v_scale is null"),
    (_attend(5, None), "out is null"),
    (_attend(6, None), "kv_len is null"),
    (_attend(1, PU), "aligned"),
    (_attend(2, PU), "aligned"),
    (_attend(dims=(-1, 8, 2, 64, 100, 128)), "batch must be non-negative"),
    (_attend(dims=(2, 0, 2, 64, 100, 128)), "n_heads must be positive"),
    (_attend(dims=(2, 8, 0, 64, 100, 128)), "n_kv_heads must be positive"),
    (_attend(dims=(2, 8, 3, 64, 100, 128)), "divisible by n_kv_heads"),
    (_attend(dims=(2, 8, 2, 80, 100, 128)), "head_dim must be 64 or 128"),
    (_attend(dims=(2, 8, 2, 64, -1, 128)), "max_kv_len must be non-negative"),
    (_attend(dims=(2, 8, 2, 64, 129, 128)), "kv_max_seq_len < max_kv_len"),
    (_attend(dims=(2, 8, 2, 64, 100, 1 << 31)), "kv_max_seq_len must be below"),
    (_attend(dims=(1 << 30, 8, 2, 64, 100, 128)), "too many"),
    (_attend(scale=float("inf")), "scale must be finite"),
    (_attend(scale=float("nan")), "scale must be finite"),
    (_attend(split=-1), "split_kv must be non-negative"),
]


@pytest.mark.parametrize("call,substr", REFUSALS, ids=[f"{i}-{c[0][4:]}" for i, (c, _) in enumerate(REFUSALS)])
def test_refusals(eng, call, substr):
    assert eng.status(*call) == 1
    assert substr in eng.last_error()


@pytest.mark.parametrize("call", [
    ("eng_mx4_quantize_f32", None, None, None, 0, 4, None),
    ("eng_mx4_dequantize_f16", None, None, None, 4, 0, None),
    ("eng_linear_mx4w_nk", P, P, P, P, 0, 4, 4, None),
    ("eng_linear_mx4w_nk", P, P, P, P, 4, 0, 4, None),
    ("eng_rmsnorm_linear_mx4w_nk", P, None, P, P, P, 4, 4, 0, 1e-5, None),
    _write(dims=(0, 3, 4, 64, 128)),
    _write(dims=(2, 0, 4, 64, 128)),
    _attend(dims=(0, 8, 2, 64, 100, 128)),
])
def test_nothing_to_do(eng, call):
    assert eng.status(*call) == 0


def test_e4m3_statement_agrees_with_torch():
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(3)
    x = np.concatenate([rng.uniform(-448, 448, 4000), rng.standard_normal(4000) * 0.01,
                        narrow.E4M3, -narrow.E4M3, (narrow.E4M3[1:] + narrow.E4M3[:-1]) / 2,
                        [np.inf, -np.inf, np.nan, -0.0]]).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert narrow.same_codes(narrow.e4m3_encode(x), want)
    back = torch.from_numpy(want).view(torch.float8_e4m3fn).to(torch.float32).numpy()
    assert np.array_equal(narrow.e4m3_decode(want), back, equal_nan=True)


def test_mx4_statement_rounds_to_the_nearest_code():
    rng = np.random.default_rng(4)
    W = rng.standard_normal((5, 100)) * np.exp2(rng.integers(-30, 30, (5, 1)))
    codes, scales = narrow.mx4_encode(W)
    assert codes.shape == (5, 64) and scales.shape == (5, 4)
    v = narrow.mx4_decode(codes, scales, 100)
    s = np.repeat(np.exp2(scales.astype(np.float64) - 127), 32, 1)[:, :100]
    # half a step of the grid (1 from 4 up), 2 past 6 where values saturate below 8
    assert (np.abs(v - W) <= np.where(np.abs(W) > 6 * s, 2 * s, np.where(np.abs(W) > 4 * s, s, s / 2))).all()
