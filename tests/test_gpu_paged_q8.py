"""The 8-bit paged cache on the GPU: rows quantised as they are appended, copies, and cached rows of
every type read back, against plain restatements (paged_q8_model.py)."""
from __future__ import annotations

import numpy as np
import pytest

import paged_q8_model as Q
from abi_ops import down, stream, up
from cdml import native as N
from test_gpu_paged import pool, rng

pytestmark = pytest.mark.gpu

MAX, TINY = np.finfo(np.float32).max, np.float32(2.0 ** -149)


# ---- append ------------------------------------------------------------------------

def special_rows(hd):
    """Rows of values at the edges of the formats, [n, hd]."""
    at = np.arange(hd)
    rows = [np.zeros(hd), np.full(hd, TINY), np.full(hd, MAX), np.where(at % 2, -MAX, TINY),
            np.where(at == hd - 1, np.inf, 1), np.where(at == 0, np.nan, 3), np.where(at == hd // 2, -np.inf, 0),
            2.0 ** -126 * (at % 5 - 2), 2.0 ** -130 * at, np.where(at == 0, 448, (at % 29) / 2 + 0.25),
            np.where(at == 0, 1.75, 2.0 ** -(at % 20)), np.where(at == 0, 1.7500001, 2.0 ** -(at % 20)),
            np.where(at == 0, 127, at % 100 - 49.5),          # ties of I8, scale 1
            np.where(at == 0, -127 * 2.0 ** 90, (at % 100 - 50.5) * 2.0 ** 90),
            np.where(at == 0, 448, 16 + at % 14 + 0.5),       # ties of F8
            np.where(at == 0, 448, -(at % 9) * 2.0 ** -10),   # its smallest values, scale 1
            np.where(at % 2, -0.0, 0.0)]
    with np.errstate(over="ignore"):
        return np.array(rows).astype(np.float32)


@pytest.mark.parametrize("kind", ["i8", "f8"])
@pytest.mark.parametrize("heads,hd,more_k,more_v,P", [(1, 1, 0, 0, 16), (3, 5, 1, 2, 4), (4, 16, 0, 0, 16),
                                                      (2, 40, 4, 1, 8), (5, 64, 0, 64, 64), (8, 128, 0, 0, 1),
                                                      (1, 200, 8, 0, 16), (3, 256, 0, 4, 32), (2, 17, 0, 0, 2)])
def test_append(kind, heads, hd, more_k, more_v, P):
    r = rng(31, heads, hd)
    special = special_rows(hd)
    rows = 4 * len(special) + 7
    x = []
    for more in (more_k, more_v):
        t = np.full((rows, heads * hd + more), np.nan, np.float32)
        y = Q.random_rows(r, rows, heads, hd)
        for i, s in enumerate(special):
            y[4 * i, i % heads] = s
        t[:, :heads * hd] = y.reshape(rows, -1)
        x.append(t)
    pages = -(-rows * 2 // P)
    slots = r.permutation(pages * P)[:rows].astype(np.int32)
    slots[1::4] = r.choice([-1, -7, pages * P, 2 ** 31 - 1], len(slots[1::4]))
    codes = [r.integers(0, 256, (pages, heads, P, Q.width(hd))).astype(np.uint8) for _ in range(2)]
    scales = [r.standard_normal((pages, heads, P)).astype(np.float32) for _ in range(2)]
    want = [a.copy() for a in codes + scales]
    for side in range(2):
        c, s = Q.quantise(x[side][:, :heads * hd].reshape(rows, heads, hd), kind)
        for i, slot in enumerate(slots):
            if 0 <= slot < pages * P:
                want[side][slot // P, :, slot % P] = c[i]
                want[2 + side][slot // P, :, slot % P] = s[i]
    got = Q.call_append(x[0], x[0].shape[1], x[1], x[1].shape[1], codes, scales, kind, slots, P, heads, hd)
    for g, w in zip(got[0] + got[1], want):
        np.testing.assert_array_equal(g, w)


@pytest.mark.parametrize("kind,half_step", [("i8", 0.5), ("f8", None)])
def test_what_is_read_back_lies_within_half_a_step(kind, half_step):
    """I8: half a scale, and the roundings of the scale and of the product, both relative to the value; F8: 2^-4 of the
    value, or half of the smallest step 2^-9 of a scale (products by a power of two are exact)."""
    r, heads, hd, P, n = rng(32), 4, 64, 16, 320
    x = Q.random_rows(r, n, heads, hd)
    pages = n // P
    empty = [np.zeros((pages, heads, P, hd), np.uint8)] * 2, [np.zeros((pages, heads, P), np.float32)] * 2
    rows = x.reshape(n, -1)
    (kc, vc), (ks, vs) = Q.call_append(rows, heads * hd, -rows, heads * hd, *empty, kind, np.arange(n, dtype=np.int32), P,
                                       heads, hd)
    c = {"kind": kind, "P": P, "heads": heads, "hd": hd, "k": kc, "v": vc, "ks": ks, "vs": vs}
    k, v, bad = Q.call_read(c, np.arange(pages, dtype=np.int32)[None], np.array([n]), np.array([0, n]), n, heads * hd,
                            heads * hd)
    np.testing.assert_array_equal(k, -v)
    s = np.moveaxis(ks, 1, 2).reshape(n, heads, 1).astype(np.float64)
    x = x.astype(np.float64)
    step = s / 2 + np.abs(x) * 2.0 ** -23 if kind == "i8" else np.maximum(np.abs(x) * 2.0 ** -4, s * 2.0 ** -10)
    assert bad == 0 and (np.abs(k.reshape(x.shape) - x) <= step).all()


# ---- read --------------------------------------------------------------------------

def read_plain(c, table, kv, cu, rows, ld, side, fill=7.0, n_pages=None):
    out, bad = np.full((rows, ld), fill, np.float32), 0
    P, dim = c["P"], c["heads"] * c["hd"]
    for b in range(len(kv)):
        first, end = max(int(cu[b]), 0), min(int(cu[b + 1]), rows)
        for row in range(first, end):
            t = min(max(int(kv[b]), 0), table.shape[1] * P) - (int(cu[b + 1]) - row)
            out[row, :dim] = 0
            if t < 0:
                continue
            page = int(table[b, t // P])
            if not 0 <= page < (n_pages or len(c["k"])):
                bad = 1
                continue
            with np.errstate(invalid="ignore"):
                out[row, :dim] = c[side + "x"][page, t % P].astype(np.float32)
    return out, bad


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16", "i8", "f8"])
@pytest.mark.parametrize("lens,parts,P,heads,hd,more", [
    ([60] * 4, None, 16, 4, 16, 0), ([1, 0, 33, 7, 250], None, 8, 2, 40, 4), ([5], None, 1, 1, 1, 0),
    ([300, 2, 0, 64], [40, 2, 0, 64], 32, 8, 128, 0), ([9, 70], [12, 70], 16, 3, 5, 1), ([100, 31], None, 64, 1, 256, 0),
    ([3] * 150, [1, 3, 0] * 50, 2, 2, 17, 3), ([4000], None, 16, 2, 64, 0)])
def test_read(kind, lens, parts, P, heads, hd, more):
    r = rng(33, hd, P)
    B, blocks = len(lens), -(-max(lens) // P) + 1
    _, table = pool(r, B, blocks, P, lens, held=0)
    c = Q.random_cache(r, kind, B * blocks, P, heads, hd)
    cu = np.concatenate([[0], np.cumsum(lens if parts is None else parts)]).astype(np.int32)
    rows, ldk, ldv = int(cu[-1]) + 2, heads * hd + more, heads * hd + 2 * more
    kv = np.array(lens, np.int32)
    k, v, bad = Q.call_read(c, table, kv, cu, rows, ldk, ldv)
    np.testing.assert_array_equal(k, read_plain(c, table, kv, cu, rows, ldk, "k")[0])
    np.testing.assert_array_equal(v, read_plain(c, table, kv, cu, rows, ldv, "v")[0])
    assert bad == 0


@pytest.mark.parametrize("kind", ["bf16", "i8", "f8"])
def test_read_of_pages_that_are_none_and_tables_that_end(kind):
    r, P, heads, hd = rng(34), 8, 2, 24
    c = Q.random_cache(r, kind, 20, P, heads, hd)
    table = r.permutation(20).astype(np.int32).reshape(4, 5)
    table[0, 1], table[1, 0], table[3, 4] = -1, 2 ** 31 - 1, 17
    kv = np.array([30, 12, -4, 1000], np.int32)  # the last ends at 40, the table's tokens
    cu = np.array([0, 30, 42, 45, 55], np.int32)
    want = [read_plain(c, table, kv, cu, 60, heads * hd, s, n_pages=17) for s in "kv"]
    k, v, bad = Q.call_read(c, table, kv, cu, 60, heads * hd, heads * hd, n_pages=17)
    np.testing.assert_array_equal(k, want[0][0])
    np.testing.assert_array_equal(v, want[1][0])
    assert bad == 1 == want[0][1]


@pytest.mark.parametrize("kind", ["i8", "f8"])
def test_rows_with_infinities_read_as_nan(kind):
    r, P, heads, hd = rng(35), 16, 2, 32
    c = Q.random_cache(r, kind, 2, P, heads, hd)
    x = Q.random_rows(r, 2 * P, heads, hd).reshape(2, P, heads, hd)
    x[0, 3, 1, 7], x[1, 0, 0, 0] = np.inf, np.nan
    Q.put(c, "k", x)
    k, v, _ = Q.call_read(c, np.array([[0, 1]], np.int32), np.array([32]), np.array([0, 32]), 32, heads * hd, heads * hd)
    k = k.reshape(32, heads, hd)
    want = np.zeros((32, heads), bool)
    want[3, 1] = want[16, 0] = True
    np.testing.assert_array_equal(np.isnan(k).all(-1), want)
    np.testing.assert_array_equal(np.isnan(k).any(-1), want)
    assert np.isfinite(v).all()


# ---- copy --------------------------------------------------------------------------

@pytest.mark.parametrize("layers,P,heads,hd,more", [(1, 16, 4, 16, 0), (3, 8, 2, 40, 5), (2, 64, 8, 128, 0), (1, 1, 1, 5, 0),
                                                    (2, 4096, 2, 16, 3)])
def test_copy(layers, P, heads, hd, more):
    r, pages, B = rng(36, P, hd), 9, 5
    stride = pages * P + more
    n = layers * stride * heads
    data = [r.integers(0, 256, n * Q.width(hd)).astype(np.uint8) for _ in range(2)] + [
        r.standard_normal(n).astype(np.float32) for _ in range(2)]
    src, dst = np.array([0, 1, -1, 0, 3], np.int32), np.array([5, 6, 7, 8, pages], np.int32)
    kv = np.array([P * 2 + 1, 3 * P - 1, 1, P * 3, 2], np.int32)
    want = [a.copy() for a in data]
    for a, w in zip(want, (Q.width(hd), Q.width(hd), 1, 1)):
        for l in range(layers):
            x = a[l * stride * heads * w:][:pages * heads * P * w].reshape(pages, heads, P, w)
            for s, d, m in zip(src, dst, kv % P):
                if 0 <= s < pages and 0 <= d < pages:
                    x[d, :, :m] = x[s, :, :m]
    d = [up(a, a.dtype) for a in data + [src, dst, kv]]
    N.check(N.lib().cdml_paged_copy_q8(*(b.ptr for b in d[:4]), layers, stride, pages, P, heads, hd,
                                       *(b.ptr for b in d[4:]), B, stream().handle))
    for b, w in zip(d, want):
        np.testing.assert_array_equal(down(b, w.shape, w.dtype), w)
