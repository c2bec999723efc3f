"""Attention over shared prefixes at sizes that all run shared: chunks whose shared and own tokens go in tiles, on every
cache type, and single tokens of wide groups.  Against float64 as in test_gpu_paged_shared.py, whose helper runs a call
unshared, and says nothing, where no length of a prefix is worth sharing: here that fails."""
from __future__ import annotations

import numpy as np
import pytest

import paged_q8_model as Q
from test_gpu_paged import rng
from test_gpu_paged_shared import KINDS, case_of, check

pytestmark = pytest.mark.gpu


def shares(case, H):
    """The case, which the entry shares by its estimate (Q.forced) and which the tables then prove."""
    _, c, table, kv, cu, groups, _ = case
    assert Q.forced(c, table, kv, cu, groups, H) is not None
    return case


def chunks(r, kind, H, HK, hd, P, most, groups=(0, 12, 14, 30), prefix=(70, 200, 700)):
    """Ragged chunks of up to `most` new tokens, some requests idle, some of one token."""
    B = groups[-1]
    news = r.integers(1, most + 1, B)
    news[[0, B - 1]], news[[1, 13, B - 2]], news[[2, 20]] = most, 1, 0
    tails = np.maximum(news, r.integers(0, 150, B))
    tails[3] = news[3]
    pages = [max(1, n // P) for n in prefix]
    return case_of(r, kind, list(groups), pages, list(tails), list(news), P, H, HK, hd)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,HK,hd,P,most", [
    (2, 2, 32, 16, 20), (2, 2, 32, 16, 140), (4, 1, 64, 8, 5), (4, 2, 64, 16, 20), (4, 2, 64, 16, 70), (3, 1, 128, 64, 5),
    (3, 1, 128, 64, 45), (2, 2, 128, 16, 20), (2, 2, 128, 16, 70), (2, 2, 50, 1, 20), (2, 2, 50, 1, 70), (3, 1, 7, 4, 45),
    (8, 2, 96, 32, 5), (6, 1, 40, 2, 5), (34, 2, 24, 16, 2)])
def test_chunks(kind, H, HK, hd, P, most):
    check(*shares(chunks(rng(101, hd, most), kind, H, HK, hd, P, most), H), H)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,HK,hd,P", [(4, 4, 16, 16), (7, 1, 128, 32), (1, 1, 7, 4), (4, 2, 104, 8), (5, 1, 64, 1)])
def test_single_tokens_of_wide_groups(kind, H, HK, hd, P):
    r = rng(102, hd)
    tails, news = r.integers(1, 60, 110), [1] * 110
    news[2] = news[105] = 0
    check(*shares(case_of(r, kind, [0, 101, 110], [max(1, n // P) for n in (300, 75)], tails, news, P, H, HK, hd), H), H)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,P", [(64, 16), (128, 16), (128, 8)])
def test_chunks_do_not_see_other_slots(kind, hd, P):
    case = chunks(rng(103, hd), kind, 2, 2, hd, P, 70)
    Q.unseen_filth(case[1], case[2], case[3])
    check(*shares(case, 2), 2)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
def test_a_nan_in_what_chunks_share(kind, hd):
    r = rng(104, hd)
    q, c, table, kv, cu, g, o = chunks(r, kind, 2, 2, hd, 16, 70, prefix=(70, 200, 320))
    x = r.standard_normal((len(c["k"]), 16, 2, hd)).astype(np.float32)
    x[table[14, 7], 3, 1, 5] = np.nan
    Q.put(c, "v", x)
    got, _ = check(*shares((q, c, table, kv, cu, g, o), 2), 2)
    broken = np.isnan(got).reshape(len(got), 2, hd).any(2)
    assert broken[cu[14]:cu[30], 1].all() and broken.sum() == cu[30] - cu[14]
