"""The packed and int8-cache ops without a device: the library exports them, refuses a null suite, and the plain forms
that the GPU tests compare with hold to their definitions."""
from __future__ import annotations

import numpy as np
import pytest
import seq_oracle as so


def test_null_suite_is_refused(lz):
    L = lz.load_library()
    calls = [L.l0b_attention_execute_packed(*[None] * 8, 64, 4, 2, 1, 1, 1, 0, 0, 0, 0),
             L.l0b_attention_execute_q8(*[None] * 10, 64, 4, 2, 32, 64, 1, 1, 0, 0),
             L.l0b_kv_cache_q8_store(*[None] * 10, 2, 64, 32, 64, 1, 1, 0, 0),
             L.l0b_kv_cache_q8_load(*[None] * 10, 2, 64, 32, 64, 1, 1, 0, 0)]
    assert calls == [1] * 4
    with pytest.raises(lz.ArgumentException):
        lz.check(calls[0])


def test_codes_round_the_real_quotient_to_even():
    scale = np.float32(0.1)  # not a dyadic number
    h = np.arange(-126, 126) + 0.5
    x = h * np.float64(scale)
    want = np.where(np.floor(h).astype(int) % 2 == 0, np.floor(h), np.ceil(h))
    np.testing.assert_array_equal(so.codes_of(x, scale), want)
    np.testing.assert_array_equal(so.codes_of(np.nextafter(x, np.inf), scale), np.ceil(h))
    assert not so.codes_of(x, np.float32(0)).any() and not so.codes_of(x, np.float32(np.nan)).any()


@pytest.mark.parametrize("block", [32, 64])
def test_store_keeps_values_within_half_a_step_of_each_store(block):
    rng = np.random.default_rng(0)
    x = rng.standard_normal((200, 2, 64))
    codes, scales = np.zeros((200, 2, 64), np.int8), np.zeros((-(-200 // block), 2), np.float32)
    for start, n in [(0, 70), (70, 1), (71, 1), (72, 60), (132, 68)]:
        so.store(x[start:start + n], codes, scales, start, block)
        before = codes.copy(), scales.copy()
        so.store(x[start:start + n], codes, scales, start, block)
        np.testing.assert_array_equal(codes, before[0])
        np.testing.assert_array_equal(scales, before[1])
    # at most three stores met one block here: three half steps of its last scale
    assert np.all(np.abs(so.values(codes, scales, block) - x) <= 1.5 * np.repeat(scales, block, 0)[:200, :, None] * 1.001)


def test_attention_with_nothing_to_see_is_zero():
    rng = np.random.default_rng(1)
    q, k = rng.standard_normal((5, 4 * 64)), rng.standard_normal((3, 2 * 64))
    out, spread, *_ = so.attention(q, k, k, np.arange(-2, 3), 4, 2)
    assert not out[:2].any() and np.all(out[2] == k[0].reshape(2, 64).repeat(2, 0))
    np.testing.assert_allclose(spread[2], np.abs(out[2]))
