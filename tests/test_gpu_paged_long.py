"""Attention in tiles over more keys than a wave holds pages of (1024), in one piece: 512 K/V
heads of 8 fill the card, so that keys are not split over workgroups."""
from __future__ import annotations

import numpy as np
import pytest

import paged_model as M
from test_gpu_paged import attention_case, rng

pytestmark = pytest.mark.gpu

H, HD, SCALE = 512, 8, 0.35
HEADS = np.r_[0:8, 250:262, 500:512]  # those compared
COLS = (HEADS[:, None] * HD + np.arange(HD)).ravel()


def compare(kind, q, bits, table, kv, cu, o, P, bad=0, zeroed=None):
    """zeroed: the table with pages that count as zeros at the number past the last one."""
    k, v = (np.concatenate([M.from_bits(b, kind)[..., COLS], np.zeros((1, P, len(COLS)), np.float32)]).astype(np.float64)
            for b in bits)
    want, tol = M.attention(q[:, COLS], k, v, table if zeroed is None else zeroed, kv, cu, P, len(HEADS), len(HEADS),
                            SCALE, o[:, COLS])
    got, found = M.call_attention(q, *bits, kind, table, kv, cu, P, H, H, SCALE, o)
    assert found == bad and np.isfinite(got).all()
    np.testing.assert_array_less(np.abs(got[:, COLS] - want), np.maximum(tol, 1e-30))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("P", [8, 16, 64])
@pytest.mark.parametrize("lens", [[1023, 1024, 1025], [1100, 2049], [2100, 40]])
def test_keys_past_the_pages_of_a_wave(kind, P, lens):
    # what lies behind the last token, in the same page too, is NaN
    r = rng(50, P, *lens)
    news = [20, 17, 33][:len(lens)]
    q, bits, table, kv, cu, o = attention_case(r, kind, lens, news, P, H, H, HD, pad=2)
    used = np.zeros(len(bits[0]) * P, bool)
    for b, m in enumerate(lens):
        at = np.arange(m)
        used[table[b, at // P] * P + at % P] = True
    for x in bits:
        x.reshape(-1, H * HD)[~used] = M.to_bits(np.full(1, np.nan), kind)[0]
    compare(kind, q, bits, table, kv, cu, o, P)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("P", [8, 16, 64])
@pytest.mark.parametrize("key", [1023, 1024, 1090, 2048, 2099])
def test_bad_pages_past_the_pages_of_a_wave(kind, P, key):
    r = rng(51, P, key)
    q, bits, table, kv, cu, o = attention_case(r, kind, [2100], [17], P, H, H, HD)
    broken, zeroed = table.copy(), table.copy()
    broken[0, key // P] = -3 if key % 2 else len(bits[0])
    zeroed[0, key // P] = len(bits[0])
    compare(kind, q, bits, broken, kv, cu, o, P, bad=1, zeroed=zeroed)
