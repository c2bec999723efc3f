"""Attention over the paged cache where keys, values and probabilities differ by large powers of
two: no row may depend on the size of a token that it does not see, no column on another's."""
from __future__ import annotations

import numpy as np
import pytest

import paged_model as M
from test_gpu_paged import attention_case, check_attention, rng

pytestmark = pytest.mark.gpu


def ratios(kind, exponents=(20, 28, 40)):
    return (20, 26) if kind == "f16" else exponents


CASES = [(kind, e) for kind in ("f32", "f16", "bf16") for e in ratios(kind)]


def rebuilt(bits, kind, table, lens, change):
    """The caches with change(tokens of request b [len, dim], b) in the place of every request's tokens."""
    x = M.from_bits(bits, kind).copy()
    for b, m in enumerate(lens):
        at = np.arange(m)
        x[table[b, at // x.shape[1]], at % x.shape[1]] = change(x[table[b, at // x.shape[1]], at % x.shape[1]], b)
    return M.to_bits(x, kind)


def small(kind):
    """What puts N(0, 1) values low in the type's range, so that 2^26 times them still lies within it."""
    return np.float32(2.0 ** -13 if kind == "f16" else 1)


@pytest.mark.parametrize("kind,e", CASES)
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("which", [0, 1])
def test_tokens_of_other_sizes_within_a_tile(kind, e, hd, which):
    # tokens 16 to 31 are larger by 2^e, which rows 0 to 15 do not see; every other token; the first ones
    r = rng(40, hd, e, which)
    large = [np.arange(32) >= 16, np.arange(48) % 2 == 0, np.arange(100) < 16]
    lens = [len(x) for x in large]
    q, bits, table, kv, cu, o = attention_case(r, kind, lens, [32, 48, 90], 16, 1, 1, hd)
    bits[which] = rebuilt(bits[which], kind, table, lens,
                          lambda x, b: x * small(kind) * np.where(large[b], np.float32(2.0 ** e), 1)[:, None])
    check_attention(kind, q, bits, table, kv, cu, o, 16, 1, 1)


@pytest.mark.parametrize("kind,e", CASES)
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_dims_of_other_sizes(kind, e, hd):
    # every fourth dim of V is larger by 2^e; then K's, where Q is zero
    r = rng(41, hd, e)
    lens, news = [40, 130], [40, 70]
    for which in (1, 0):
        q, bits, table, kv, cu, o = attention_case(r, kind, lens, news, 16, 2, 1, hd)
        larger = np.where(np.arange(hd) % 4 == which, np.float32(2.0 ** e), 1)
        bits[which] = rebuilt(bits[which], kind, table, lens, lambda x, b: x * small(kind) * larger)
        if which == 0:
            q.reshape(len(q), 2, hd)[:, :, larger > 1] = 0
        check_attention(kind, q, bits, table, kv, cu, o, 16, 2, 1)


@pytest.mark.parametrize("kind,e", [("f32", 24), ("f32", 30), ("f32", 40), ("bf16", 24), ("bf16", 40), ("f16", 20),
                                    ("f16", 26)])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("order", ["up", "down", "mixed"])
def test_values_that_grow_as_scores_fall(kind, e, hd, order):
    # 32 keys and more whose V is larger by 2^e and whose probability is smaller by as much: their part in
    # the sums is as large as the others'
    r = rng(42, hd, e)
    lens, news = [96, 70], [24, 30]
    q, bits, table, kv, cu, o = attention_case(r, kind, lens, news, 16, 1, 1, hd)
    scale = float(np.float32(1) / np.sqrt(np.float32(hd)))
    q *= np.float32(0.1)
    q[:, 0] = 1 / scale

    def far(m):
        at = np.arange(m)
        return {"up": at >= 32, "down": at < 32, "mixed": at * 7 % 3 == 0}[order]

    def keys(x, b):
        x[:, 0] = np.where(far(len(x)), -e * np.log(2.0), 0)
        return x

    bits[0] = rebuilt(bits[0], kind, table, lens, keys)
    bits[1] = rebuilt(bits[1], kind, table, lens,
                      lambda x, b: x * small(kind) * np.where(far(len(x)), np.float32(2.0 ** e), 1)[:, None])
    check_attention(kind, q, bits, table, kv, cu, o, 16, 1, 1)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("e", [-20, -40])
def test_dims_that_are_nearly_dead(kind, e):
    # four neighbouring dims of K, V and Q far below the others (in fp16, subnormal ones or zeros)
    r = rng(43, -e)
    lens, news = [300, 33], [70, 33]
    q, bits, table, kv, cu, o = attention_case(r, kind, lens, news, 16, 2, 1, 64)
    for i in range(2):
        x = M.from_bits(bits[i], kind).copy()
        x[..., 20:24] *= np.float32(2.0 ** e)
        bits[i] = M.to_bits(x, kind)
    q.reshape(len(q), 2, 64)[:, :, 40:44] *= np.float32(2.0 ** e)
    check_attention(kind, q, bits, table, kv, cu, o, 16, 2, 1)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("which", [0, 1])
def test_rows_of_any_number_agree(kind, which):
    # the same request as single tokens, a few and many rows, its last tokens larger
    r = rng(44, which)
    q, bits, table, kv, cu, o = attention_case(r, kind, [64], [40], 16, 1, 1, 64)
    e = 20 if kind == "f16" else 30
    bits[which] = rebuilt(bits[which], kind, table, [64],
                          lambda x, b: x * small(kind) * np.where(np.arange(64) >= 50, np.float32(2.0 ** e), 1)[:, None])
    for n in (1, 8, 40):
        for m in (64, 60, 49):
            check_attention(kind, q[:n], bits, table, np.array([m], np.int32), np.array([0, n], np.int32), o[:n], 16, 1, 1)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("T,n", [(60, 1), (3000, 1), (60, 8), (3000, 8), (60, 40), (3000, 40)])
def test_the_lowest_finite_scores(kind, T, n):
    """Scores of -3.17e38 and -3.25e38 in log2 units, next to -FLT_MAX: the latter's keys, every one from the
    middle on, have no weight, and the former's are equal, so that o is the mean of their V, all 3."""
    r = rng(45)
    q, bits, table, kv, cu, o = attention_case(r, kind, [T], [n], 16, 1, 1, 8)
    k, v = (np.zeros_like(M.from_bits(b, kind)) for b in bits)
    at = np.arange(T)
    low = np.where(at < T // 2, np.float32(-1e19), np.float32(-1.025e19))
    k[table[0, at // 16], at % 16, 0] = low
    v[table[0, at // 16], at % 16] = np.where(at < T // 2, 3, 7)[:, None]
    bits = [M.to_bits(x, kind) for x in (k, v)]
    q[:] = 0
    q[:, 0] = np.float32(2.2e19)
    got, _ = M.call_attention(q, *bits, kind, table, kv, cu, 16, 1, 1, 1.0, o)
    np.testing.assert_allclose(got, 3, rtol=(2 * T + 32) * 2.0 ** -24)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,n", [(60, 1), (3000, 1), (60, 8), (3000, 8), (60, 40), (3000, 40)])
def test_scores_of_minus_infinity(kind, T, n):
    # a row that sees such scores alone is 0, as one that sees no token; beside others they have no weight
    r = rng(46)
    q, bits, table, kv, cu, o = attention_case(r, kind, [T], [n], 16, 1, 1, 64)
    k, v = (M.from_bits(b, kind).copy() for b in bits)
    at = np.arange(T)
    q[:, 0] = 1
    for some in (0, 3, T):  # finite ones: the last of them
        k[table[0, at // 16], at % 16, 0] = np.where(at >= T - some, 0, -np.inf)
        v[table[0, at // 16], at % 16] = 3
        got, _ = M.call_attention(q, M.to_bits(k, kind), M.to_bits(v, kind), kind, table, kv, cu, 16, 1, 1, 0.125, o)
        seen = np.minimum(T, T - n + 1 + np.arange(n))
        none = seen <= T - some
        assert not got[none].any()
        np.testing.assert_allclose(got[~none], 3, rtol=(2 * T + 32) * 2.0 ** -24)
