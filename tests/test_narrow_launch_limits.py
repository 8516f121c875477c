"""Calls of the 4-bit and 8-bit entries that need 2^32 threads or more in one launch, which
HIP does not take, are refused on the host, before any device call."""

from __future__ import annotations

import pytest

P = 0x1000  # dummy 16-byte aligned "device" pointer; never dereferenced here


@pytest.mark.parametrize("call,substr", [
    # 2 batch heads blocks units of a wave each
    (("eng_kv_cache_write_q8", *[P] * 7, None, 1 << 20, 1, 32, 64, 64, None), "kv_cache_write_q8: too many"),
    (("eng_kv_cache_write_q8", *[P] * 7, None, 1 << 10, 1 << 15, 32, 64, 1 << 15, None), "too many"),
    # batch heads workgroups of up to 256 threads
    (("eng_attention_decode_q8", *[P] * 7, 1 << 23, 4, 2, 64, 100, 128, 0.125, 1, None),
     "attention_decode_q8: too many"),
    # the merge's wave for each of batch heads
    (("eng_attention_decode_q8", *[P] * 7, 1 << 22, 16, 1, 64, 100, 128, 0.125, 2, None), "too many"),
    # 48 tiles of 16 columns to 1024 threads; 384 columns to 512
    (("eng_linear_mx4w_nk", P, P, P, P, 1, 768 << 22, 32, None), "linear_mx4w: N too large"),
    (("eng_rmsnorm_linear_mx4w_nk", P, P, P, P, P, 4, 1 << 40, 32, 1e-5, None), "N too large"),
    (("eng_linear_mx4w_nk", P, P, P, P, 5, 384 << 23, 32, None), "N too large"),
    (("eng_linear_mx4w_nk", P, P, P, P, 64, 1 << 40, 32, None), "N too large"),
])
def test_refusals(eng, call, substr):
    assert eng.status(*call) == 1
    assert substr in eng.last_error()
