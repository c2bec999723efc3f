"""The paged K/V cache on the GPU: plans, appends, attention, reordering and copies
against plain numpy and float64 restatements (paged_model.py)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import paged_model as M
from abi_ops import down, stream, up
from cdml import native as N

pytestmark = pytest.mark.gpu


def rng(*key):
    return np.random.default_rng([*key])


def pool(r, B, blocks, P, lens, extra=0, held=0.25):
    """Random pages for requests of the given lengths: (refs, table); unused entries are -1."""
    n = B * blocks + extra
    refs = (r.random(n) < held).astype(np.int32)
    table, order, at = np.full((B, blocks), -1, np.int32), r.permutation(n), 0
    for b, m in enumerate(lens):
        used = -(-int(m) // P)
        table[b, :used] = order[at:at + used]
        refs[table[b, :used]] = 1
        at += used
    return refs, table


def same(got, want):
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g, w)


# ---- plan ------------------------------------------------------------------------

@pytest.mark.parametrize("B,P,blocks,most_new,extra_rows", [
    (1, 16, 4, 1, 0), (3, 1, 9, 4, 2), (7, 16, 6, 40, 0), (64, 16, 8, 1, 3), (250, 8, 12, 50, 1), (1100, 4, 3, 5, 0),
    (5, 4096, 2, 3000, 7), (4096, 2, 2, 2, 0)])
def test_plan_takes_the_lowest_free_pages(B, P, blocks, most_new, extra_rows):
    r = rng(1, B, P)
    kv = r.integers(0, blocks * P // 2 + 1, B).astype(np.int32)
    new = np.minimum(r.integers(0, most_new + 1, B), blocks * P - kv).astype(np.int32)
    refs, table = pool(r, B, blocks, P, kv, extra=B * 2)
    rows = int(new.sum()) + extra_rows
    want = M.plan(refs, table, kv, new, P, rows)
    assert want[-1][0] in (0, 1)
    same(M.call_plan(refs, table, kv, new, P, rows), want)


def test_plan_scans_large_and_full_pools():
    r = rng(2)
    refs = np.ones(100_003, np.int32)
    refs[[99_990, 16_384, 5]] = 0
    kv, new = np.array([16, 0], np.int32), np.array([17, 16], np.int32)
    table = np.full((2, 4), -1, np.int32)
    table[0, 0] = 7
    same(M.call_plan(refs, table, kv, new, 16, 33), M.plan(refs, table, kv, new, 16, 33))
    new = np.array([33, 16], np.int32)  # four pages of three
    want = M.plan(refs, table, kv, new, 16, 60)
    assert want[-1][0] == 1
    same(M.call_plan(refs, table, kv, new, 16, 60), want)


@pytest.mark.parametrize("kv,new,rows,code", [
    ([0, 3], [5, 1], 6, 0), ([0, 3], [5, 1], 5, 4), ([0, -1], [5, 1], 9, 2), ([0, 3], [5, -2], 9, 2),
    ([0, 3], [5, 30], 60, 2), ([0, 3], [32, 29], 61, 1), ([0, 3], [40, 29], 1, 2 + 4),
    ([2 ** 31 - 1, 3], [2 ** 31 - 1, 1], 9, 2), ([0, 0], [0, 0], 3, 0), ([0, 0], [0, 0], 0, 0)])
def test_plan_takes_all_or_nothing(kv, new, rows, code):
    refs, table = np.zeros(14, np.int32), np.full((2, 8), -1, np.int32)
    table[1, 0], refs[0], refs[3] = 3, 2, 1
    kv, new = np.array(kv, np.int64).astype(np.int32), np.array(new, np.int64).astype(np.int32)
    got = M.call_plan(refs, table, kv, new, 4, rows)
    assert got[-1][0] == code
    same(got, M.plan(refs, table, kv.astype(np.int64), new.astype(np.int64), 4, rows))


def test_plan_without_requests():
    got = M.call_plan(np.zeros(3, np.int32), np.zeros((0, 2), np.int32), np.zeros(0, np.int32), np.zeros(0, np.int32),
                      16, 4)
    assert list(got[3]) == [0] and list(got[4]) == [-1] * 4 and list(got[6]) == [0, 0, 0]


# ---- append ------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,dim,ldk,ldv,P", [(1, 8, 8, 8, 16), (33, 64, 64, 64, 16), (7, 5, 9, 5, 4),
                                                (65, 40, 44, 41, 8), (300, 256, 256, 512, 1)])
def test_append(kind, rows, dim, ldk, ldv, P):
    r = rng(3, rows, dim)
    pages = -(-rows * 2 // P)
    k, v = (r.standard_normal((rows, n)).astype(np.float32) * 10.0 ** r.integers(-9, 6, (rows, 1)) for n in (ldk, ldv))
    k, v = k.astype(np.float32), v.astype(np.float32)
    k[0, 0], k[0, 1], v[0, 0] = np.inf, -0.0, np.nan
    slots = r.permutation(pages * P)[:rows].astype(np.int32)
    slots[1::3] = r.choice([-1, -7, pages * P, 2 ** 31 - 1], len(slots[1::3]))
    first = [r.integers(-2 ** 15, 2 ** 15, (pages * P, dim)).astype(M.raw_dtype(kind)) for _ in range(2)]
    want = [f.copy() for f in first]
    for w, new in zip(want, (k, v)):
        for i, s in enumerate(slots):
            if 0 <= s < pages * P:
                w[s] = M.to_bits(new[i, :dim], kind)
    d = [up(a, a.dtype) for a in (k, v, first[0], first[1], slots)]
    N.check(N.lib().cdml_paged_append(d[0].ptr, ldk, d[1].ptr, ldv, d[2].ptr, d[3].ptr, N.CACHE[kind], d[4].ptr, rows,
                                      pages, P, dim, stream().handle))
    for buf, w in zip(d[2:4], want):
        got = M.from_bits(down(buf, w.shape, w.dtype), kind)
        np.testing.assert_array_equal(got, M.from_bits(w, kind))  # (NaN equals NaN, whatever its payload)


# ---- attention -----------------------------------------------------------------------

def attention_case(r, kind, lens, news, P, H, HK, hd, pad=0, blocks=None):
    B = len(lens)
    blocks = blocks or max(1, -(-max(max(lens), 1) // P)) + 1
    _, table = pool(r, B, blocks, P, lens, held=0)
    n_pages = B * blocks
    rows = sum(news) + pad
    q = r.standard_normal((rows, H * hd)).astype(np.float32)
    o = r.standard_normal((rows, H * hd)).astype(np.float32)
    bits = [M.to_bits(r.standard_normal((n_pages, P, HK * hd)), kind) for _ in range(2)]
    cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    return q, bits, table, np.array(lens, np.int32), cu, o


def check_attention(kind, q, bits, table, kv, cu, o, P, H, HK, scale=None, **more):
    if scale is None:
        scale = float(np.float32(1) / np.sqrt(np.float32(q.shape[1] // H)))
    k, v = (M.from_bits(b, kind).astype(np.float64) for b in bits)
    want, tol = M.attention(q, k, v, table, kv, cu, P, H, HK, scale, o)
    got, bad = M.call_attention(q, *bits, kind, table, kv, cu, P, H, HK, scale, o, **more)
    assert bad == 0
    fine = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    worst = np.max(np.abs(got[fine] - want[fine]) - tol[fine], initial=-1)
    assert worst <= 0, f"off by {np.abs(got[fine] - want[fine]).max():.3g}, {worst:.3g} over the bound"
    return got


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,HK,hd", [(1, 1, 8), (4, 4, 16), (5, 5, 40), (2, 1, 64), (8, 2, 32), (7, 1, 128), (3, 3, 96),
                                     (4, 2, 7), (2, 2, 256), (3, 1, 200)])
def test_one_new_token(kind, H, HK, hd):
    r = rng(4, H, hd)
    lens = [1, 16, 17, 255, 256, 257, 700, 0]
    case = attention_case(r, kind, lens, [1] * 8, 16, H, HK, hd)
    check_attention(kind, *case, 16, H, HK)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,HK,hd,P", [(2, 2, 64, 16), (4, 1, 32, 8), (2, 1, 128, 64), (3, 3, 24, 1), (1, 1, 100, 32),
                                       (6, 2, 64, 128), (2, 1, 160, 16)])
def test_ragged_chunks(kind, H, HK, hd, P):
    r = rng(5, H, hd, P)
    lens = [1, 40, 129, 333, 64, 65, 200, 0, 31, 400]
    news = [1, 40, 2, 130, 0, 33, 128, 0, 4, 1]
    case = attention_case(r, kind, lens, news, P, H, HK, hd, pad=5)
    got = check_attention(kind, *case, P, H, HK)
    np.testing.assert_array_equal(got[-5:], case[-1][-5:])  # rows of no request stay


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_keys_split_over_workgroups(kind):
    r = rng(6)
    case = attention_case(r, kind, [2900, 1111, 9], [9, 70, 5], 16, 2, 1, 64)
    check_attention(kind, *case, 16, 2, 1)
    case = attention_case(r, kind, [2900, 1], [1, 1], 32, 4, 2, 128)
    check_attention(kind, *case, 32, 4, 2)


def test_rows_without_a_key_are_zero():
    # more new tokens than the cache holds: the first of them see nothing
    r = rng(7)
    for lens, news in (([3, 0, 2], [5, 2, 1]), ([3, 0, 400], [40, 20, 401]), ([700, 2], [1, 4])):
        case = attention_case(r, "f32", lens, news, 16, 2, 2, 32)
        got = check_attention("f32", *case, 16, 2, 2)
        for first, n, m in zip(case[4], news, lens):
            assert not got[first:first + max(0, n - m)].any()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("news", [[1, 1], [3, 2], [60, 200]])
@pytest.mark.parametrize("filth", [np.nan, np.inf, -np.inf])
def test_what_is_not_seen_does_not_matter(kind, news, filth):
    r = rng(8)
    lens, P, H, HK, hd = [70, 300], 16, 4, 2, 64
    q, bits, table, kv, cu, o = attention_case(r, kind, lens, news, P, H, HK, hd)
    used = np.zeros(len(bits[0]) * P, bool)
    for b, m in enumerate(lens):
        at = np.arange(m)
        used[table[b, at // P] * P + at % P] = True
    for x in bits:
        x.reshape(-1, HK * hd)[~used] = M.to_bits(np.full(1, filth), kind)[0]
    check_attention(kind, q, bits, table, kv, cu, o, P, H, HK)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_later_tokens_do_not_reach_earlier_rows(kind, value):
    # an infinity or a NaN in V of a token: the rows before it keep finite values
    r = rng(9)
    q, bits, table, kv, cu, o = attention_case(r, kind, [90], [60], 16, 2, 2, 64)
    bits[1].reshape(-1, 128)[table[0, 50 // 16] * 16 + 50 % 16] = M.to_bits(np.full(1, value), kind)[0]
    got = check_attention(kind, q, bits, table, kv, cu, o, 16, 2, 2)
    assert np.isfinite(got[:20]).all() and not np.isfinite(got[20:]).any()


def test_far_scores_and_small_values():
    # scores that rise by hundreds along the keys (the reference has to follow), then values at 2^-120
    r = rng(10)
    for kind in ("f32", "bf16"):
        q, bits, table, kv, cu, o = attention_case(r, kind, [300, 300], [1, 80], 16, 1, 1, 64)
        k = M.from_bits(bits[0], kind)
        for b in range(2):
            at = np.arange(300)
            k[table[b, at // 16], at % 16] *= (1 + at[:, None] / 4)
        bits[0] = M.to_bits(k, kind)
        check_attention(kind, q, bits, table, kv, cu, o, 16, 1, 1)
        bits[1] = M.to_bits(M.from_bits(bits[1], kind) * np.float32(2.0 ** -120), kind)
        check_attention(kind, q, bits, table, kv, cu, o, 16, 1, 1)


def test_contiguous_cache_is_a_paged_one():
    # [batch, t_max, dim] with its pages in a row equals cdml_decode_attn within both bounds
    r = rng(11)
    B, T, H, hd, P = 3, 128, 4, 64, 32
    q, lens = r.standard_normal((B, H * hd)).astype(np.float32), np.array([128, 77, 1], np.int32)
    k, v = (r.standard_normal((B * T // P, P, H * hd)).astype(np.float32) for _ in range(2))
    table = np.arange(B * T // P, dtype=np.int32).reshape(B, -1)
    cu = np.arange(B + 1, dtype=np.int32)
    scale = 0.125
    want, tol = M.attention(q, k.astype(np.float64), v.astype(np.float64), table, lens, cu, P, H, H, scale,
                            np.zeros_like(q))
    got, _ = M.call_attention(q, k, v, "f32", table, lens, cu, P, H, H, scale, np.zeros_like(q))
    import abi_ops
    dense = abi_ops.decode(q, k.reshape(B, T, -1), v.reshape(B, T, -1), lens, H, scale)
    assert (np.abs(got - want) <= tol).all() and (np.abs(dense - want) <= tol).all()


@pytest.mark.parametrize("news", [[1, 1], [50, 3]])
def test_pages_out_of_range_count_as_zeros(news):
    r = rng(12)
    P, H, hd = 16, 2, 64
    q, bits, table, kv, cu, o = attention_case(r, "f32", [100, 60], news, P, H, H, hd)
    broken = table.copy()
    broken[0, 2], broken[1, 1] = len(bits[0]), -5
    k, v = (np.concatenate([b, np.zeros((1, P, H * hd), np.float32)]).astype(np.float64) for b in bits)
    zeros = broken.copy()
    zeros[0, 2] = zeros[1, 1] = len(bits[0])
    want, tol = M.attention(q, k, v, zeros, kv, cu, P, H, H, 0.125, o)
    got, bad = M.call_attention(q, *bits, "f32", broken, kv, cu, P, H, H, 0.125, o)
    assert bad == 1 and (np.abs(got - want) <= tol).all()


def test_bounds_cut_lengths():
    r = rng(13)
    q, bits, table, kv, cu, o = attention_case(r, "f32", [100, 60], [6, 2], 16, 2, 2, 32, blocks=7)
    # kv_len beyond max_len counts as max_len; new tokens past max_new are left alone
    want, tol = M.attention(q, *(b.astype(np.float64) for b in bits), table, np.array([80, 60]), cu, 16, 2, 2, 0.125, o)
    got, _ = M.call_attention(q, *bits, "f32", table, kv, cu, 16, 2, 2, 0.125, o, max_len=80)
    assert (np.abs(got - want) <= tol).all()
    got, _ = M.call_attention(q, *bits, "f32", table, kv, cu, 16, 2, 2, 0.125, o, max_new=2)
    np.testing.assert_array_equal(got[2:6], o[2:6])


@pytest.mark.parametrize("news", [[30, 1], [3, 1], [1, 1]])
def test_strided_rows(news):
    r = rng(14)
    for ldq, ldo in ((130, 128), (132, 140), (128, 129)):
        q, bits, table, kv, cu, o = attention_case(r, "bf16", [100, 60], news, 16, 2, 1, 64)
        check_attention("bf16", q, bits, table, kv, cu, o, 16, 2, 1, ldq=ldq, ldo=ldo)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("news", [[1, 1], [7, 2], [50, 1]])
@pytest.mark.parametrize("scale", [0.0, -0.3, 40.0])
def test_scales(kind, news, scale):
    # no weight on the scores at all, a negative one, and one that leaves a single key
    r = rng(15)
    q, bits, table, kv, cu, o = attention_case(r, kind, [100, 60], news, 16, 2, 1, 32)
    check_attention(kind, q, bits, table, kv, cu, o, 16, 2, 1, scale=scale)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [4, 60, 200])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("where", [5, 239])
def test_a_huge_key_or_value_among_ordinary_ones(kind, n, which, where):
    # one token's K or V is 10^30 in a few dims; the rows that do not see it, or give it no weight, are exact
    r = rng(23)
    q, bits, table, kv, cu, o = attention_case(r, kind, [240, 30], [n, 30], 16, 2, 2, 64)
    x = M.from_bits(bits[which], kind).reshape(-1, 128).copy()
    at = table[0, where // 16] * 16 + where % 16
    x[at, 5:9] = 1e30
    bits[which] = M.to_bits(x, kind).reshape(bits[which].shape)
    if which == 1:
        k = M.from_bits(bits[0], kind).reshape(-1, 128).copy()
        k[at] = -50 * np.sign(q[0])  # the first row's head gives the token no weight
        bits[0] = M.to_bits(k, kind).reshape(bits[0].shape)
    check_attention(kind, q, bits, table, kv, cu, o, 16, 2, 2)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_magnitudes_that_change_along_the_keys(kind):
    # V grows and shrinks by tens along the request, some dims are always small, some keys zero
    r = rng(24)
    q, bits, table, kv, cu, o = attention_case(r, kind, [600, 333], [70, 333], 16, 2, 1, 64)
    k, v = (M.from_bits(b, kind).copy() for b in bits)
    for b, m in enumerate((600, 333)):
        at = np.arange(m)
        v[table[b, at // 16], at % 16] *= (10.0 ** np.sin(at / 40))[:, None].astype(np.float32)
        v[table[b, at[::17] // 16], at[::17] % 16] = 0
        k[table[b, at[::13] // 16], at[::13] % 16] = 0
    v[..., 7:13] *= np.float32(1 / 64)
    k[..., 20:24] *= np.float32(1 / 64)
    bits = [M.to_bits(x, kind) for x in (k, v)]
    check_attention(kind, q, bits, table, kv, cu, o, 16, 2, 1)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [4, 60])
def test_a_broken_key_or_query_stays_in_its_rows(kind, n):
    r = rng(16)
    q, bits, table, kv, cu, o = attention_case(r, kind, [90], [n], 16, 2, 2, 64)
    first_seen = 90 - n
    bits[0].reshape(-1, 128)[table[0, (first_seen + 2) // 16] * 16 + (first_seen + 2) % 16] = M.to_bits(np.full(1, np.nan), kind)[0]
    q[1, :64] = np.inf
    got = check_attention(kind, q, bits, table, kv, cu, o, 16, 2, 2)
    assert np.isfinite(got[0]).all() and np.isfinite(got[1, 64:]).all() and np.isnan(got[1, :64]).all()
    assert np.isnan(got[2:]).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("first", [0.02, 0.021, 0.022])
def test_a_large_key_beside_unseen_infinities(kind, hd, first):
    # K's largest values stand next to infinite ones that the rows do not see
    r = rng(29)
    q, bits, table, kv, cu, o = attention_case(r, kind, [73], [64], 16, 1, 1, hd)
    k = M.from_bits(bits[0], kind).copy()
    k[table[0, 33 // 16], 33 % 16, 0] = -100
    at = np.arange(41, 73)  # row 31 sees keys up to 40
    k[table[0, at // 16], at % 16] = np.inf
    bits[0] = M.to_bits(k, kind)
    q[:, 0] = first
    got = check_attention(kind, q, bits, table, kv, cu, o, 16, 1, 1)
    assert np.isfinite(got[:32]).all()


def test_queries_out_of_the_split_range():
    # components below 2^-110 beside ordinary ones, and large ones against small keys
    r = rng(17)
    for news in ([7], [60]):
        q, bits, table, kv, cu, o = attention_case(r, "f32", [90], news, 16, 1, 1, 64)
        q[:, ::3] *= np.float32(2.0 ** -118)
        check_attention("f32", q, bits, table, kv, cu, o, 16, 1, 1)
        q *= np.float32(2.0 ** 105)
        bits[0] *= np.float32(2.0 ** -105)
        check_attention("f32", q, bits, table, kv, cu, o, 16, 1, 1)


@pytest.mark.parametrize("kind,news", [("f32", 1), ("bf16", 1), ("bf16", 6), ("f32", 40), ("bf16", 40)])
def test_offsets_past_32_bits(kind, news):
    """Pages at the end of a cache of over 2^32 bytes (and, in fp32, 2^31 elements) a tensor: written by
    cdml_paged_append, read back by the attention.  Only the pages in use are ever touched."""
    r = rng(18)
    P, H, hd = 16, 8, 128
    D, n_pages = H * hd, 140_000
    size = n_pages * P * D * (4 if kind == "f32" else 2)
    assert size > 2 ** 32
    lens = np.array([70, 45], np.int32)
    table = np.array([[n_pages - 1, 3, n_pages - 9, n_pages - 2, n_pages // 2 + 1], [n_pages - 5, n_pages - 4, 0, -1, -1]],
                     np.int32)
    k, v = (r.standard_normal((lens.sum(), D)).astype(np.float32) for _ in range(2))
    slots = np.concatenate([table[b, np.arange(m) // P] * P + np.arange(m) % P for b, m in enumerate(lens)])
    kc, vc = N.DeviceBuffer(size), N.DeviceBuffer(size)
    dk, dv, ds = up(k), up(v), M.ints(slots)
    N.check(N.lib().cdml_paged_append(dk.ptr, D, dv.ptr, D, kc.ptr, vc.ptr, N.CACHE[kind], ds.ptr, len(slots), n_pages,
                                      P, D, stream().handle))
    rows = 2 * news
    q, cu = r.standard_normal((rows, D)).astype(np.float32), np.array([0, news, rows], np.int32)
    dq, do, dt, dl, dc, bad = up(q), N.DeviceBuffer(4 * rows * D), M.ints(table), M.ints(lens), M.ints(cu), M.ints([0])
    args = (rows, 2, news, 80, H, H, hd)
    w, n = M.ws("cdml_paged_attn_workspace_size", *args)
    N.check(N.lib().cdml_paged_attn(dq.ptr, D, kc.ptr, vc.ptr, N.CACHE[kind], n_pages, P, dt.ptr, 5, dl.ptr, dc.ptr,
                                    do.ptr, D, *args, 0.09, bad.ptr, w.ptr, n, stream().handle))
    got = down(do, (rows, D))
    small = np.concatenate([[0], np.cumsum(lens)])
    rounded = [M.from_bits(M.to_bits(x, kind), kind).astype(np.float64) for x in (k, v)]
    for b in range(2):
        own = [x[small[b]:small[b + 1]][:, None] for x in rounded]
        want, tol = M.attention(q[b * news:(b + 1) * news], *own, np.arange(lens[b])[None], lens[b:b + 1],
                                np.array([0, news]), 1, H, H, 0.09, np.zeros((news, D)))
        assert (np.abs(got[b * news:(b + 1) * news] - want) <= tol).all()
    assert down(bad, (1,), np.int32)[0] == 0


def test_many_requests():
    r = rng(19)
    B = 700
    lens = r.integers(0, 40, B).tolist()
    news = [min(int(n), m) for n, m in zip(r.integers(0, 4, B), lens)]
    news[333], lens[333] = 30, 37
    case = attention_case(r, "bf16", lens, news, 8, 2, 1, 16, pad=3)
    check_attention("bf16", *case, 8, 2, 1)


@pytest.mark.parametrize("B", [2, 64, 65, 140])
def test_tiles_of_many_ragged_requests(B):
    # every tile of every request is met once, whatever the order: long and short, few rows, none, rows without a key
    r = rng(33, B)
    news = np.where(r.random(B) < 0.2, r.integers(0, 5, B), r.integers(0, 100, B))
    lens = np.where(r.random(B) < 0.3, news, news + r.integers(0, 500, B))
    news[B // 2], lens[B // 2] = 260, 300
    news[1], lens[1] = 70, 10
    case = attention_case(r, "bf16", lens.tolist(), news.tolist(), 16, 4, 1, 16, pad=5, blocks=48)
    check_attention("bf16", *case, 16, 4, 1)


# ---- reorder and copies ------------------------------------------------------------------

@pytest.mark.parametrize("R,P,blocks,steps", [(1, 16, 4, 3), (8, 4, 6, 6), (40, 16, 5, 5), (300, 2, 9, 3),
                                              (2100, 4, 2, 2)])
def test_reorder_follows_the_plain_form(R, P, blocks, steps):
    r = rng(20, R, P)
    lens = r.integers(0, blocks * P - steps, R).astype(np.int32)
    refs, table = pool(r, R, blocks, P, lens, extra=3)
    kv = lens
    for step in range(steps):
        parents = r.integers(0, R, R).astype(np.int32)
        parents[r.random(R) < 0.15] = -1
        if step == 1:
            parents = np.arange(R, dtype=np.int32)  # nothing moves
        if step == 2:
            parents[:] = parents[0] if parents[0] >= 0 else R - 1  # everything from one row
            parents[-1] = R + 5
        want = M.reorder(refs, table, kv, parents, P)
        got = M.call_reorder(refs, table, kv, parents, P)
        same(got, want)
        refs, table, kv = got[:3]
        assert (refs >= 0).all()
        new = np.minimum(1, blocks * P - kv).astype(np.int32)
        want = M.plan(refs, table, kv, new, P, R)
        got = M.call_plan(refs, table, kv, new, P, R)
        same(got, want)
        refs, table, kv = got[:3]


@pytest.mark.parametrize("R", [6, 50])
def test_released_pages_are_taken_again(R):
    r = rng(22, R)
    P, blocks = 4, 6
    lens = r.integers(1, 16, R).astype(np.int32)
    refs, table = pool(r, R, blocks, P, lens, held=0)
    kv = lens
    for turn in range(4):
        parents = np.where(np.arange(R) % 3 == turn % 3, -1, np.arange(R)).astype(np.int32)
        want = M.reorder(refs, table, kv, parents, P)
        got = M.call_reorder(refs, table, kv, parents, P)
        same(got, want)
        refs, table, kv = got[:3]
        assert (kv[parents < 0] == 0).all() and refs.sum() == sum(-(-m // P) for m in kv)
        new = np.where(parents < 0, 9, 0).astype(np.int32)
        want = M.plan(refs, table, kv, new, P, int(new.sum()))
        got = M.call_plan(refs, table, kv, new, P, int(new.sum()))
        assert got[-1][0] == 0
        same(got, want)
        refs, table, kv = got[:3]
    nobody = np.full(R, -1, np.int32)
    assert not M.call_reorder(refs, table, kv, nobody, P)[0].any()


def test_reorder_without_room_cuts_to_full_pages():
    refs, table = np.array([1, 1, 1], np.int32), np.array([[0, 1], [-1, -1], [2, -1]], np.int32)
    kv, parents = np.array([6, 0, 4], np.int32), np.array([0, 0, 2], np.int32)
    want = M.reorder(refs, table, kv, parents, 4)
    assert list(want[-1]) == [1, 0, 0] and list(want[2]) == [6, 4, 4]
    same(M.call_reorder(refs, table, kv, parents, 4), want)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("dim,layers,P", [(64, 3, 16), (5, 1, 8), (1024, 2, 64)])
def test_copies_move_the_open_tokens(kind, dim, layers, P):
    r = rng(21, dim)
    pages, R = 12, 5
    stride = pages * P * dim + (16 if layers > 1 else 0)
    cache = [r.integers(-2 ** 15, 2 ** 15, layers * stride).astype(M.raw_dtype(kind)) for _ in range(2)]
    kv = np.array([P + 1, 2 * P - 1, 3, P // 2, 5], np.int32)
    src, dst = np.array([1, 2, -1, pages, 7], np.int32), np.array([3, 4, 5, 6, -9], np.int32)
    want = [c.copy() for c in cache]
    for w in want:
        for l in range(layers):
            page = w[l * stride:l * stride + pages * P * dim].reshape(pages, P, dim)
            for b in range(2):
                page[dst[b], :kv[b] % P] = page[src[b], :kv[b] % P]
    d = [up(a, a.dtype) for a in cache] + [M.ints(a) for a in (src, dst, kv)]
    N.check(N.lib().cdml_paged_copy(d[0].ptr, d[1].ptr, N.CACHE[kind], layers, stride, pages, P, dim, d[2].ptr,
                                    d[3].ptr, d[4].ptr, R, stream().handle))
    same([down(b, w.shape, w.dtype) for b, w in zip(d, want)], want)


# ---- together ------------------------------------------------------------------------------

class Engine:
    """One layer's serving loop on device buffers: plan, append, attention; beams reordered between steps."""

    def __init__(self, R, P, blocks, pages, H, HK, hd, kind, rows, max_new):
        self.R, self.P, self.blocks, self.pages, self.kind = R, P, blocks, pages, kind
        self.H, self.HK, self.hd, self.rows, self.max_new = H, HK, hd, rows, max_new
        D = HK * hd
        self.refs, self.table, self.kv = (M.ints(np.zeros(n)) for n in (pages, R * blocks, R))
        self.new, self.cu, self.slots, self.pos, self.status = (M.ints(np.zeros(n)) for n in (R, R + 1, rows, rows, 3))
        self.k, self.v = (up(np.full(pages * P * D, np.nan if kind == "f32" else -1), M.raw_dtype(kind)) for _ in range(2))
        self.q, self.nk, self.nv = up(np.zeros((rows, H * hd))), up(np.zeros((rows, D))), up(np.zeros((rows, D)))
        self.o = up(np.zeros((rows, H * hd)))
        self.size = (rows, R, max_new, blocks * P, H, HK, hd)
        self.ws, self.ws_n = M.ws("cdml_paged_attn_workspace_size", *self.size)

    def step(self, s):
        L, h = N.lib(), s.handle
        N.check(L.cdml_paged_plan(self.refs.ptr, self.pages, self.P, self.table.ptr, self.blocks, self.kv.ptr,
                                  self.new.ptr, self.R, self.rows, self.cu.ptr, self.slots.ptr, self.pos.ptr,
                                  self.status.ptr, h))
        D = self.HK * self.hd
        N.check(L.cdml_paged_append(self.nk.ptr, D, self.nv.ptr, D, self.k.ptr, self.v.ptr, N.CACHE[self.kind],
                                    self.slots.ptr, self.rows, self.pages, self.P, D, h))
        N.check(L.cdml_paged_attn(self.q.ptr, self.H * self.hd, self.k.ptr, self.v.ptr, N.CACHE[self.kind],
                                  self.pages, self.P, self.table.ptr, self.blocks, self.kv.ptr, self.cu.ptr,
                                  self.o.ptr, self.H * self.hd, *self.size, 0.125, None, self.ws.ptr, self.ws_n, h))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_serving_run_in_a_graph(kind):
    """Chunked prompts, then single tokens with beams reordered between them: the step is captured
    once and replayed; every replay matches dense attention over each row's own history."""
    r = rng(30)
    R, P, H, HK, hd = 6, 8, 4, 2, 64
    blocks, pages, rows, max_new = 12, 90, 40, 24
    e = Engine(R, P, blocks, pages, H, HK, hd, kind, rows, max_new)
    s = N.Stream()
    history = [np.zeros((0, 2, HK * hd)) for _ in range(R)]
    steps = [[13, 0, 24, 0, 1, 2], [24, 0, 11, 0, 0, 5], None, [1] * 6, [1] * 6, None, [1, 1, 0, 1, 1, 1], None, [1] * 6]
    graph = None
    src, dst, status = (M.ints(np.zeros(n)) for n in (R, R, 3))
    w, n = M.ws("cdml_paged_reorder_workspace_size", R, blocks)
    for turn, new in enumerate(steps):
        if new is None:
            parents = r.integers(0, R, R).astype(np.int32) if turn > 2 else np.array([0, 0, 2, 2, 4, 5], np.int32)
            d = M.ints(parents)
            N.check(N.lib().cdml_paged_reorder(e.refs.ptr, pages, P, e.table.ptr, blocks, e.kv.ptr, d.ptr, R, src.ptr,
                                               dst.ptr, status.ptr, w.ptr, n, s.handle))
            N.check(N.lib().cdml_paged_copy(e.k.ptr, e.v.ptr, N.CACHE[kind], 1, 0, pages, P, HK * hd, src.ptr, dst.ptr,
                                            e.kv.ptr, R, s.handle))
            s.synchronize()
            assert list(status.download((3,), np.int32, s))[::2] == [0, 0]
            history = [history[p] for p in parents]
            continue
        total = sum(new)
        q, k, v = (r.standard_normal((rows, D)).astype(np.float32) for D in (H * hd, HK * hd, HK * hd))
        for buf, a, t in ((e.q, q, np.float32), (e.nk, k, np.float32), (e.nv, v, np.float32),
                          (e.new, np.array(new), np.int32)):
            buf.upload(np.ascontiguousarray(a, t), s)
        if graph is None:
            e.step(s)  # the first step runs eagerly; a second run of it would append again
            s.synchronize()
            graph = C.c_void_p()
            N.check(N.lib().cdml_graph_capture_begin(s.handle))
            e.step(s)
            N.check(N.lib().cdml_graph_capture_end(s.handle, C.byref(graph)))
        else:
            N.check(N.lib().cdml_graph_launch(graph, s.handle))
        got = e.o.download((rows, H * hd), np.float32, s)
        assert list(e.status.download((3,), np.int32, s)) == [0, e.status.download((3,), np.int32, s)[1], total]
        first = 0
        for b, m in enumerate(new):
            rounded = np.stack([M.from_bits(M.to_bits(a[first:first + m], kind), kind) for a in (k, v)], 1)
            history[b] = np.concatenate([history[b], rounded])
            T = len(history[b])
            if m:
                dense = np.ascontiguousarray(history[b].transpose(1, 0, 2)).astype(np.float64)
                want, tol = M.attention(q[first:first + m], dense[0][:, None], dense[1][:, None],
                                        np.arange(T)[None], np.array([T]), np.array([0, m]), 1, H, HK, 0.125,
                                        np.zeros((m, H * hd)))
                assert (np.abs(got[first:first + m] - want) <= tol).all(), (turn, b)
            first += m
        np.testing.assert_array_equal(e.kv.download((R,), np.int32, s), [len(x) for x in history])
    N.check(N.lib().cdml_graph_destroy(graph))


def test_two_streams_at_once():
    r = rng(31)
    cases = []
    for i in range(2):
        q, bits, table, kv, cu, o = attention_case(r, "bf16", [900, 300, 50], [40, 1, 7], 16, 4, 2, 64)
        size = (len(q), 3, 40, 900, 4, 2, 64)
        w, n = M.ws("cdml_paged_attn_workspace_size", *size)
        d = [up(q), up(bits[0], np.int16), up(bits[1], np.int16), M.ints(table), M.ints(kv), M.ints(cu), up(o)]
        cases.append((N.Stream(), d, size, w, n, len(bits[0]), table.shape[1], o.shape,
                      M.attention(q, *(M.from_bits(b, "bf16").astype(np.float64) for b in bits), table, kv, cu, 16, 4, 2,
                                  0.125, o)))
    for _ in range(5):
        for s, d, size, w, n, pages, blocks, _, _ in cases:
            N.check(N.lib().cdml_paged_attn(d[0].ptr, 256, d[1].ptr, d[2].ptr, N.CACHE["bf16"], pages, 16, d[3].ptr,
                                            blocks, d[4].ptr, d[5].ptr, d[6].ptr, 256, *size, 0.125, None, w.ptr, n,
                                            s.handle))
    for s, d, _, _, _, _, _, shape, (want, tol) in cases:
        assert (np.abs(d[6].download(shape, np.float32, s) - want) <= tol).all()


def test_large_pools_in_spans():
    # more pages than one count covers, more new pages than are handed out at a time, little free in front
    r = rng(3)
    n, P = 200_003, 2
    refs = (r.random(n) < 0.9).astype(np.int32)
    refs[70_000:] = r.random(n - 70_000) < 0.3
    new = np.array([9000, 1, 0, 23_456, 40_000, 17], np.int32)
    kv = np.array([3, 1, 8, 0, 11, 2], np.int32)
    table = np.full((6, 21_000), -1, np.int32)
    taken = np.flatnonzero(refs)
    for b, m in enumerate(kv):
        table[b, :-(-m // P)] = taken[10 * b:10 * b - (-m // P)]
    same(M.call_plan(refs, table, kv, new, P, int(new.sum())), M.plan(refs, table, kv, new, P, int(new.sum())))
    # copies that find their pages past the first span
    refs[:66_000] = 1
    parents = np.array([0, 0, 0, 1, 1, 5], np.int32)
    want = M.reorder(refs, table, kv, parents, P)
    same(M.call_reorder(refs, table, kv, parents, P), want)


@pytest.mark.parametrize("B,K,V", [(3, 4, 300), (10, 5, 6000)])
def test_beam_steps_in_a_graph(B, K, V):
    """Plan, append, selection in place, reordering and copies, captured once: every replay equals the plain forms,
    with work and synchronisation of other kinds between the replays."""
    r = rng(32, B)
    R, P, blocks, dim, steps = B * K, 4, 7, 8, 6
    pages, L, s = R * blocks, N.lib(), N.Stream()
    refs, table, kv = np.zeros(pages, np.int32), np.full((R, blocks), -1, np.int32), np.zeros(R, np.int32)
    cache = [np.zeros((pages, P, dim), np.float32) for _ in range(2)]
    scores = -np.abs(r.standard_normal(R)).astype(np.float32)
    lengths, done = np.ones(R, np.int32), np.zeros(R, np.uint8)
    d_refs, d_table, d_kv, d_len, d_new = (M.ints(a) for a in (refs, table, kv, lengths, np.ones(R)))
    d_cu, d_slots, d_pos, d_par, d_tok, d_src, d_dst, st1, st2 = (M.ints(np.zeros(R + 3)) for _ in range(9))
    d_k, d_v, d_scores, d_x = up(cache[0]), up(cache[1]), up(scores), up(np.zeros((R, V)))
    d_done, d_nk, d_nv = up(done, np.uint8), up(np.zeros((R, dim))), up(np.zeros((R, dim)))
    w1, n1 = M.ws("cdml_beam_select_workspace_size", B, K, V)
    w2, n2 = M.ws("cdml_paged_reorder_workspace_size", R, blocks)
    h = s.handle

    def step():
        N.check(L.cdml_paged_plan(d_refs.ptr, pages, P, d_table.ptr, blocks, d_kv.ptr, d_new.ptr, R, R, d_cu.ptr,
                                  d_slots.ptr, d_pos.ptr, st1.ptr, h))
        N.check(L.cdml_paged_append(d_nk.ptr, dim, d_nv.ptr, dim, d_k.ptr, d_v.ptr, 0, d_slots.ptr, R, pages, P, dim, h))
        N.check(L.cdml_beam_select(d_x.ptr, V, d_scores.ptr, d_len.ptr, d_done.ptr, B, K, V, 2, 0.5, d_scores.ptr,
                                   d_len.ptr, d_done.ptr, d_par.ptr, d_tok.ptr, w1.ptr, n1, h))
        N.check(L.cdml_paged_reorder(d_refs.ptr, pages, P, d_table.ptr, blocks, d_kv.ptr, d_par.ptr, R, d_src.ptr,
                                     d_dst.ptr, st2.ptr, w2.ptr, n2, h))
        N.check(L.cdml_paged_copy(d_k.ptr, d_v.ptr, 0, 1, 0, pages, P, dim, d_src.ptr, d_dst.ptr, d_kv.ptr, R, h))

    graph = C.c_void_p()
    N.check(L.cdml_graph_capture_begin(h))
    step()
    N.check(L.cdml_graph_capture_end(h, C.byref(graph)))
    for _ in range(steps):
        x = (r.standard_normal((R, V)) * 2).astype(np.float32)
        nk, nv = r.standard_normal((2, R, dim)).astype(np.float32)
        for buf, a in ((d_x, x), (d_nk, nk), (d_nv, nv)):
            buf.upload(a, s)
        N.check(L.cdml_graph_launch(graph, h))
        refs, table, kv, _, slots, _, _ = M.plan(refs, table, kv, np.ones(R, np.int64), P, R)
        for c, a in zip(cache, (nk, nv)):
            c.reshape(-1, dim)[slots] = a
        want = M.beam(x, scores, lengths, done, K, 2, 0.5)
        refs, table, kv, src, dst, status = M.reorder(refs, table, kv, want[3], P)
        for c in cache:
            for b in np.flatnonzero(dst >= 0):
                c[dst[b], :kv[b] % P] = c[src[b], :kv[b] % P]
        lengths, done = want[1], want[2]
        scores = d_scores.download((R,), np.float32, s)
        assert np.allclose(scores, want[0], rtol=2.0 ** -23, atol=2.0 ** -23)
        same([d.download((R,), t, s) for d, t in ((d_len, np.int32), (d_done, np.uint8), (d_par, np.int32),
                                                  (d_tok, np.int32), (d_kv, np.int32), (d_src, np.int32))],
             (lengths, done, want[3], want[4], kv, src))
        same([d_refs.download((pages,), np.int32, s), st2.download((3,), np.int32, s)], (refs, status))
        got = d_table.download((R, blocks), np.int32, s)
        for b in range(R):
            used = -(-int(kv[b]) // P)
            np.testing.assert_array_equal(got[b, :used], table[b, :used])
        used = refs > 0
        for d, c in zip((d_k, d_v), cache):
            np.testing.assert_array_equal(d.download(c.shape, np.float32, s)[used], c[used])
    N.check(L.cdml_graph_destroy(graph))
