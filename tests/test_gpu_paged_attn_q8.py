"""Attention over 8-bit paged caches on the GPU against float64 (paged_model.py), within the bound that it
derives: the products with a key's scales are two of its spare roundings.  A column in which the heavy keys hold
exact zeros (code 0) shows what fp32 cannot hold of the others: an exponential below 2^-126 comes out as 0, relative
to a reference that lies up to 2^32 below the row's sum, so T keys lose 2^-94 T max |v| at most."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import paged_model as M
import paged_q8_model as Q
from abi_ops import down, stream, up
from cdml import native as N
from test_gpu_paged import pool, rng

pytestmark = pytest.mark.gpu

KINDS = ["i8", "f8"]


def normal_rows(r, pages, P, heads, hd):
    """N(0, 1) rows of which every sixteenth channel is eight times as large."""
    x = r.standard_normal((pages, P, heads, hd))
    x[..., 3::16] *= 4
    return x.astype(np.float32)


def case_of(r, kind, lens, news, P, H, HK, hd, pad=0, blocks=None, rows=normal_rows):
    """(q, cache, table, kv, cu, o)."""
    B = len(lens)
    blocks = blocks or max(1, -(-max(max(lens), 1) // P)) + 1
    _, table = pool(r, B, blocks, P, lens, held=0)
    c = {"kind": kind, "P": P, "heads": HK, "hd": hd}
    for side in "kv":
        Q.put(c, side, rows(r, B * blocks, P, HK, hd))
    n = sum(news) + pad
    q, o = (r.standard_normal((n, H * hd)).astype(np.float32) for _ in range(2))
    return q, c, table, np.array(lens, np.int32), np.concatenate([[0], np.cumsum(news)]).astype(np.int32), o


def compare(got, want, tol):
    fine = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    worst = np.max(np.abs(got[fine] - want[fine]) - tol[fine], initial=-1)
    assert worst <= 0, f"off by {np.abs(got[fine] - want[fine]).max():.3g}, {worst:.3g} over the bound"


def check(q, c, table, kv, cu, o, H, scale=None, **more):
    if scale is None:
        scale = float(np.float32(1) / np.sqrt(np.float32(c["hd"])))
    want, tol = M.attention(q, c["kx"], c["vx"], table, kv, cu, c["P"], H, c["heads"], scale, o)
    got, bad = Q.call_attention(q, c, table, kv, cu, H, scale, o, **more)
    assert bad == 0
    compare(got, want, tol + underflow(c, kv))
    return got


def underflow(c, kv):
    v = np.abs(c["vx"])
    return 2.0 ** -94 * np.max(kv) * np.max(v[np.isfinite(v)])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,HK,hd", [(1, 1, 8), (4, 4, 16), (5, 5, 40), (2, 1, 64), (8, 2, 32), (7, 1, 128), (3, 3, 96),
                                     (4, 2, 7), (2, 2, 256), (3, 1, 200), (2, 1, 72), (1, 1, 1), (17, 1, 24), (34, 2, 136)])
@pytest.mark.parametrize("P", [16, 8, 2])
def test_one_new_token(kind, H, HK, hd, P):
    r = rng(50, H, hd, P)
    lens = [1, 16, 17, 255, 256, 257, 700, 0]
    check(*case_of(r, kind, lens, [1] * 8, P, H, HK, hd), H)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,HK,hd,P", [(2, 2, 64, 16), (4, 1, 32, 8), (2, 1, 128, 64), (3, 3, 24, 1), (1, 1, 100, 32),
                                       (6, 2, 64, 128), (2, 1, 160, 16), (3, 1, 50, 4), (2, 2, 256, 4), (1, 1, 5, 16)])
def test_ragged_chunks(kind, H, HK, hd, P):
    r = rng(51, H, hd, P)
    lens = [1, 40, 129, 333, 64, 65, 200, 0, 31, 400]
    news = [1, 40, 2, 130, 0, 33, 128, 0, 4, 1]
    case = case_of(r, kind, lens, news, P, H, HK, hd, pad=5)
    got = check(*case, H)
    np.testing.assert_array_equal(got[-5:], case[-1][-5:])  # rows of no request stay


@pytest.mark.parametrize("kind", KINDS)
def test_keys_split_over_workgroups_and_long_ones(kind):
    r = rng(52)
    check(*case_of(r, kind, [2900, 1111, 9], [9, 70, 5], 16, 2, 1, 64), 2)
    check(*case_of(r, kind, [2900, 1], [1, 1], 32, 4, 2, 128), 4)
    # one chunk of more keys than a wave holds places of: 300 requests fill the device
    check(*case_of(r, kind, [5000, 4200] + [3] * 298, [1] * 300, 64, 1, 1, 32, blocks=79), 1)


@pytest.mark.parametrize("kind", KINDS)
def test_rows_without_a_key_are_zero(kind):
    r = rng(53)
    for lens, news in (([3, 0, 2], [5, 2, 1]), ([3, 0, 400], [40, 20, 401]), ([700, 2], [1, 4])):
        case = case_of(r, kind, lens, news, 16, 2, 2, 32)
        got = check(*case, 2)
        for first, n, m in zip(case[4], news, lens):
            assert not got[first:first + max(0, n - m)].any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,P", [(64, 16), (128, 8), (40, 1), (256, 32)])
@pytest.mark.parametrize("news", [[1, 1], [3, 2], [60, 200]])
def test_what_is_not_seen_does_not_matter(kind, news, hd, P):
    r = rng(54, hd)
    lens = [70, 300]
    q, c, table, kv, cu, o = case_of(r, kind, lens, news, P, 4, 2, hd)
    Q.unseen_filth(c, table, lens)
    check(q, c, table, kv, cu, o, 4)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [4, 60])
@pytest.mark.parametrize("side", ["k", "v"])
def test_a_token_with_an_infinity_stays_in_its_rows(kind, n, side):
    r = rng(55, n)
    lens = [90]
    q, c, table, kv, cu, o = case_of(r, kind, lens, [n], 16, 2, 2, 64)
    x = normal_rows(r, len(c["k"]), 16, 2, 64)
    x[table[0, 88 // 16], 88 % 16, 1, 5] = np.inf
    Q.put(c, side, x)
    got = check(q, c, table, kv, cu, o, 2)
    assert np.isfinite(got[:n - 2]).all() and np.isfinite(got[:, :64]).all() and np.isnan(got[n - 2:, 64:]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("news", [[1, 1], [50, 3]])
@pytest.mark.parametrize("P", [16, 4, 1])
def test_pages_out_of_range_count_as_zeros(kind, news, P):
    r = rng(56, P)
    H, hd = 2, 64
    q, c, table, kv, cu, o = case_of(r, kind, [100, 60], news, P, H, H, hd)
    n = len(c["k"])
    table[0, 32 // P], table[1, 1] = n + 3, -5
    zeros = np.where((table >= 0) & (table < n), table, n)
    k, v = (np.concatenate([c[s], np.zeros((1, P, H * hd))]) for s in ("kx", "vx"))
    want, tol = M.attention(q, k, v, zeros, kv, cu, P, H, H, 0.125, o)
    for s in "kv":  # (page 0, which is read in their place)
        c[s + "s"][0] = np.nan if 0 not in table else c[s + "s"][0]
    got, bad = Q.call_attention(q, c, table, kv, cu, H, 0.125, o)
    assert bad == 1
    compare(got, want, tol)


@pytest.mark.parametrize("kind", KINDS)
def test_bounds_cut_lengths(kind):
    r = rng(57)
    q, c, table, kv, cu, o = case_of(r, kind, [100, 60], [6, 2], 16, 2, 2, 32, blocks=7)
    want, tol = M.attention(q, c["kx"], c["vx"], table, np.array([80, 60]), cu, 16, 2, 2, 0.125, o)
    got, _ = Q.call_attention(q, c, table, kv, cu, 2, 0.125, o, max_len=80)
    compare(got, want, tol)
    got, _ = Q.call_attention(q, c, table, kv, cu, 2, 0.125, o, max_new=2)
    np.testing.assert_array_equal(got[2:6], o[2:6])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("news", [[30, 1], [3, 1], [1, 1]])
def test_strided_rows(kind, news):
    r = rng(58)
    for ldq, ldo in ((130, 128), (132, 140), (128, 129)):
        check(*case_of(r, kind, [100, 60], news, 16, 2, 1, 64), 2, ldq=ldq, ldo=ldo)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("news", [[1, 1], [7, 2], [50, 1]])
@pytest.mark.parametrize("scale", [0.0, -0.3, 40.0])
def test_scales(kind, news, scale):
    r = rng(59)
    check(*case_of(r, kind, [100, 60], news, 16, 2, 1, 32), 2, scale=scale)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 4, 60])
@pytest.mark.parametrize("ek,ev", [(0, -100), (0, 60), (0, 100), (-100, 0), (90, 0)])
def test_keys_and_values_of_any_size(kind, n, ek, ev):
    # scales far from 1; Q makes up for K's
    r = rng(60, n)

    def rows(power):
        return lambda *size: normal_rows(*size) * np.float32(2.0 ** power)
    q, c, table, kv, cu, o = case_of(r, kind, [240, 30], [n, 1], 16, 2, 2, 64)
    for side, power in (("k", ek), ("v", ev)):
        Q.put(c, side, rows(power)(r, len(c["k"]), 16, 2, 64))
    check(q * np.float32(2.0 ** -ek), c, table, kv, cu, o, 2)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [2, 60])
@pytest.mark.parametrize("e", [24, 40])
def test_values_that_grow_as_scores_fall(kind, n, e):
    # keys whose V is larger by 2^e and whose probability is smaller by as much
    r = rng(61, n, e)
    hd, lens = 64, [96, 70]
    scale = float(np.float32(1) / np.sqrt(np.float32(hd)))
    q, c, table, kv, cu, o = case_of(r, kind, lens, [n, n], 16, 1, 1, hd)
    q *= np.float32(0.1)
    q[:, 0] = 1 / scale
    k, v = (r.standard_normal((len(c["k"]), 16, 1, hd)).astype(np.float32) * np.float32(0.1) for _ in range(2))
    for b, m in enumerate(lens):
        at = np.arange(m)
        far = at * 7 % 3 == 0
        k[table[b, at // 16], at % 16, 0, 0] = np.where(far, -e * np.log(2), 0)
        v[table[b, at // 16], at % 16, 0] *= np.where(far, 2.0 ** e, 1)[:, None].astype(np.float32)
    Q.put(c, "k", k)
    Q.put(c, "v", v)
    check(q, c, table, kv, cu, o, 1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [3, 40])
@pytest.mark.parametrize("value", [np.nan, np.inf, 1e33, 2.0 ** -120])
def test_queries_out_of_the_ordinary(kind, n, value):
    # 1e33 and 2^-120 beside ordinary dims; the keys are 0 where Q is large
    r = rng(62, n)
    q, c, table, kv, cu, o = case_of(r, kind, [90], [n], 16, 2, 2, 64)
    q[1, 70] = value
    if value == 1e33:
        k = normal_rows(r, len(c["k"]), 16, 2, 64)
        k[:, :, 1, 6] = 0
        Q.put(c, "k", k)
    got = check(q, c, table, kv, cu, o, 2)
    assert np.isfinite(got[:1]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_every_score_minus_infinity(kind):
    r = rng(63)
    for n in (2, 40):
        q, c, table, kv, cu, o = case_of(r, kind, [60], [n], 16, 1, 1, 32)
        Q.put(c, "k", np.full((len(c["k"]), 16, 1, 32), 3e38, np.float32))
        q[:] = -3e38
        got, _ = Q.call_attention(q, c, table, kv, cu, 1, 1.0, o)
        assert not got.any()


@pytest.mark.parametrize("kind", KINDS)
def test_the_same_bits_again_and_in_a_graph(kind):
    """Recorded once, replayed with other queries and lengths, eager calls in the same workspace between."""
    r = rng(64)
    lens, news, H, HK, hd, P = [900, 700, 333, 65], [1, 30, 1, 2], 4, 2, 64, 16
    q, c, table, kv, cu, o = case_of(r, kind, lens, news, P, H, HK, hd)
    rows, B, L, st = len(q), len(lens), N.lib(), stream()
    size = (rows, B, 30, 912, H, HK, hd)
    d = Q.upload(c)
    dt, dc, bad = M.ints(table), M.ints(cu), M.ints(np.zeros(1))
    dq, dl, do = up(q), M.ints(kv), up(o)
    w, n = M.ws("cdml_paged_attn_q8_workspace_size", *size)

    def call():
        N.check(L.cdml_paged_attn_q8(dq.ptr, H * hd, *(b.ptr for b in d), N.CACHE[kind], len(c["k"]), P, dt.ptr,
                                     table.shape[1], dl.ptr, dc.ptr, do.ptr, H * hd, *size, 0.125, bad.ptr,
                                     w.ptr, n, st.handle))
    call()
    eager = down(do, o.shape)
    graph = C.c_void_p()
    N.check(L.cdml_graph_capture_begin(st.handle))
    call()
    N.check(L.cdml_graph_capture_end(st.handle, C.byref(graph)))
    for turn in range(4):
        x = r.standard_normal(q.shape).astype(np.float32) if turn else q
        m = kv - turn * 11
        dq.upload(x, st)
        dl.upload(m.astype(np.int32), st)
        do.upload(o, st)
        N.check(L.cdml_graph_launch(graph, st.handle))
        got = down(do, o.shape)
        if turn == 0:
            np.testing.assert_array_equal(got, eager)
        want, tol = M.attention(x, c["kx"], c["vx"], table, m, cu, P, H, HK, 0.125, o)
        compare(got, want, tol)
        do.upload(o, st)
        call()
        np.testing.assert_array_equal(down(do, o.shape), got)
    N.check(L.cdml_graph_destroy(graph))
