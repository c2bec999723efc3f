"""Attention over shared prefixes where a wave takes a (request, K/V head): from 1024 of these on, with at most four
rows each and few tokens of their own, in 8-bit and bf16 caches.  Against float64 (paged_model.py) as in
test_gpu_paged_shared.py, with tables that only let a call that shares be right."""
from __future__ import annotations

import numpy as np
import pytest

import paged_model as M
import paged_q8_model as Q
from test_gpu_paged import rng
from test_gpu_paged_attn_q8 import compare, normal_rows, underflow
from test_gpu_paged_shared import case_of

pytestmark = pytest.mark.gpu

KINDS = ["bf16", "i8", "f8"]
# heads, K/V heads, head dim, page size, requests
SHAPES = [(5, 5, 64, 16, 210), (4, 4, 16, 2, 260), (14, 7, 40, 8, 150), (12, 3, 128, 16, 345), (1, 1, 8, 4, 1030),
          (2, 2, 128, 1, 520), (9, 9, 24, 64, 130), (8, 4, 96, 32, 258)]


def call(monkeypatch, case, H, tail, want=None):
    """The entry with bounds for which it shares, of `tail` tokens behind what is shared: (o, shared, bad)."""
    q, c, table, kv, cu, groups, o = case
    assert tail >= np.max(kv - Q.shared(table, kv, cu, groups, c["P"], len(c["k"])))
    forced = Q.forced
    assert forced(c, table, kv, cu, groups, H) is not None

    def bounds(*a):
        t, (members, new, prefix, _) = forced(*a)
        more = max(0, -(-tail // c["P"]) - t.shape[1])  # (bounds lie within the table)
        return np.concatenate([t, np.full((len(t), more), -1, np.int32)], 1), (members, new, prefix, tail)
    scale = float(np.float32(1) / np.sqrt(np.float32(c["hd"])))
    if want is None:
        want = M.attention(q, c["kx"], c["vx"], table, kv, cu, c["P"], H, c["heads"], scale, o)
    with monkeypatch.context() as m:
        m.setattr(Q, "forced", bounds)
        got, found, bad = Q.call_attention_shared(q, c, table, kv, cu, groups, H, scale, o, force=True)
    np.testing.assert_array_equal(found, Q.shared(table, kv, cu, groups, c["P"], len(c["k"])))
    compare(got, want[0], want[1] + underflow(c, kv))
    return got, found, bad


def check(monkeypatch, case, H, tail, want=None):
    """The same at sizes that give a wave to a (request, K/V head)."""
    c, pairs, new = case[1], len(case[3]) * case[1]["heads"], int(np.max(np.diff(case[4])))
    assert pairs >= 1024 and 4 * tail <= pairs and new * (H // c["heads"]) <= 4 and c["hd"] <= 128 and c["hd"] % 8 == 0
    return call(monkeypatch, case, H, tail, want)


def crowd(r, kind, shape, prefix=(40, 17, 90), news=1, most=70):
    """Three groups, a request alone and four of no group; tails of `most` tokens and fewer, some requests idle."""
    H, HK, hd, P, B = shape
    groups = [2, B // 3, B // 3 + 1, B - 30, B - 2]
    pages = [max(1, n // P) for n in (prefix[0], 3, *prefix[1:])]
    tails = r.integers(news, most + 1, B)
    tails[[3, 9, B - 5]] = news
    tails[[4, B - 6]] = most
    new = [news] * B
    new[5] = new[B - 7] = 0
    return case_of(r, kind, groups, pages, tails, new, P, H, HK, hd, batch=B, outside=[50, 3, 33, 64])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", SHAPES)
def test_a_wave_to_a_head(monkeypatch, kind, shape):
    case = crowd(rng(91, shape[2]), kind, shape)
    _, found, bad = check(monkeypatch, case, shape[0], 200)
    assert bad == 0 and (found[2:shape[4] // 3] > 0).all() and (found[-30:-2] > 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape,news", [((14, 7, 40, 8, 150), 2), ((5, 5, 64, 16, 210), 4), ((6, 6, 128, 2, 180), 3)])
def test_several_new_tokens(monkeypatch, kind, shape, news):
    # up to four rows, of which each sees one token more than the one before
    case = crowd(rng(92, news), kind, shape, news=news)
    assert check(monkeypatch, case, shape[0], 96)[2] == 0


@pytest.mark.parametrize("kind", KINDS)
def test_tails_of_one_token_and_of_many(monkeypatch, kind):
    for most, tail in ((1, 64), (240, 256)):
        case = crowd(rng(93, most), kind, (5, 5, 64, 16, 210), most=most)
        assert check(monkeypatch, case, 5, tail)[2] == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("P", [2, 8, 16])
def test_what_is_not_seen_does_not_matter(monkeypatch, kind, P):
    case = crowd(rng(94, P), kind, (5, 5, 40, P, 210))
    Q.unseen_filth(case[1], case[2], case[3])
    assert check(monkeypatch, case, 5, 96)[2] == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("P", [4, 8, 16])
def test_a_nan_reaches_the_rows_that_see_it(monkeypatch, kind, P):
    # in a tail, and in what a group shares
    r = rng(95, P)
    q, c, table, kv, cu, g, o = crowd(r, kind, (5, 5, 64, P, 210), most=40)
    x = normal_rows(r, len(c["k"]), P, 5, 64)
    x[table[6, (kv[6] - 1) // P], (kv[6] - 1) % P, 2, 9] = np.nan
    x[table[g[3], 0], 1, 4, 3] = np.nan
    Q.put(c, "v", x)
    got, _, bad = check(monkeypatch, (q, c, table, kv, cu, g, o), 5, 80)
    broken = np.isnan(got[:cu[-1]]).reshape(-1, 5, 64).any(2)
    rows = np.diff(cu) > 0
    members = np.arange(g[3], g[4])
    assert bad == 0 and broken[cu[6], 2] and broken[:, 4].sum() == rows[members].sum() and broken[:, [0, 1, 3]].sum() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("P", [4, 8, 16])
def test_pages_that_are_none(monkeypatch, kind, P):
    # of a tail: its tokens count as zeros
    r = rng(96, P)
    q, c, table, kv, cu, g, o = crowd(r, kind, (5, 5, 64, P, 210), most=40)
    n = len(c["k"])
    table[[4, 40], (kv[[4, 40]] - 1) // P] = -3, n
    zeros = np.where((table >= 0) & (table < n), table, n)
    k, v = (np.concatenate([c[s], np.zeros((1, P, 5 * 64))]) for s in ("kx", "vx"))
    want = M.attention(q, k, v, zeros, kv, cu, P, 5, 5, 0.125, o)
    assert check(monkeypatch, (q, c, table, kv, cu, g, o), 5, 80, want)[2] == 1


@pytest.mark.parametrize("kind", KINDS)
def test_scores_and_values_far_apart(monkeypatch, kind):
    # the maximum in the prefix, then in the tails; values of the one 1000 times the other's
    r = rng(97)
    for turn in range(4):
        q, c, table, kv, cu, g, o = crowd(r, kind, (5, 5, 64, 16, 210), most=30)
        x = {s: normal_rows(r, len(c["k"]), 16, 5, 64) for s in "kv"}
        own = np.unique(table[np.arange(210), (kv - 1) // 16])
        pages = np.unique(table[[g[0], g[3]], 0]) if turn % 2 else own
        x["kv"[turn // 2]][pages] *= np.float32(30 if turn < 2 else 1000)
        for s in "kv":
            Q.put(c, s, x[s])
        assert check(monkeypatch, (q, c, table, kv, cu, g, o), 5, 80)[2] == 0


def test_results_do_not_depend_on_the_form(monkeypatch):
    """The same call with a bound of the tails that gives a workgroup to a K/V head: as near as two sums of the same
    values in another order (both lie within the bound of float64, so twice that apart)."""
    shape = (5, 5, 64, 16, 210)
    for kind in KINDS:
        case = crowd(rng(98), kind, shape)
        q, c, table, kv, cu, _, o = case
        want, tol = M.attention(q, c["kx"], c["vx"], table, kv, cu, 16, 5, 5, 0.125, o)
        one = check(monkeypatch, case, 5, 96, (want, tol))[0]
        four = call(monkeypatch, case, 5, 300, (want, tol))[0]
        assert (np.abs(one.astype(np.float64) - four) <= 2 * (tol + underflow(c, kv))).all()
