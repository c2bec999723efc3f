"""cdml_beam_select on the GPU against its plain restatement in float64."""
from __future__ import annotations

import numpy as np
import pytest

import paged_model as M

pytestmark = pytest.mark.gpu


def check(x, scores, lengths, done, K, eos=2, alpha=0.0, **more):
    x, scores = np.asarray(x, np.float32), np.asarray(scores, np.float32)
    lengths, done = np.asarray(lengths, np.int32), np.asarray(done, np.uint8)
    want = M.beam(x, scores, lengths, done, K, eos, alpha)
    got = M.call_beam(x, scores, lengths, done, K, eos, alpha, **more)
    for g, w, name in zip(got[1:], want[1:], ("lengths", "finished", "parents", "tokens")):
        np.testing.assert_array_equal(g, w, err_msg=name)
    # a total is a sum in 64 bits of fp32 exponentials (1 step of 2^-23 each at most), rounded once
    fine = np.isfinite(want[0])
    np.testing.assert_array_equal(np.isfinite(got[0]), fine)
    assert (np.abs(got[0][fine] - want[0][fine]) <= 2.0 ** -23 + 2.0 ** -24 * np.abs(want[0][fine])).all()
    return got


def inputs(r, B, K, V, std=2.0):
    R = B * K
    return (r.standard_normal((R, V)) * std, -np.abs(r.standard_normal(R)) * 3 - 5, r.integers(0, 20, R),
            (r.random(R) < 0.15))


@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 1, 2), (2, 3, 5), (4, 4, 200), (3, 5, 2048), (2, 7, 2049), (1, 12, 8191),
                                   (5, 8, 9000), (1, 64, 4100), (2, 33, 70), (2, 4, 50021), (1, 3, 140_000),
                                   (300, 2, 33)])
@pytest.mark.parametrize("alpha", [0.0, 0.6])
def test_selection(B, K, V, alpha):
    check(*inputs(np.random.default_rng([1, B, K, V]), B, K, V), K, eos=min(2, V - 1), alpha=alpha)


@pytest.mark.parametrize("V", [6, 300, 5000])
def test_equal_logits_take_the_lowest_token(V):
    r = np.random.default_rng([2, V])
    B, K = 3, 4
    x, scores, lengths, done = inputs(r, B, K, V)
    x = np.round(x)  # many ties inside a beam
    check(x, scores, lengths, done, K)
    # equal beams: the lowest beam first, then its lowest tokens
    x[:] = 0.5
    scores[:] = -1.0
    got = check(x, scores, np.full(B * K, 3), np.zeros(B * K), K)
    assert list(got[3][:K]) == [0] * K and list(got[4][:K]) == list(range(K))


def test_signed_zeros_are_equal():
    x = np.zeros((2, 70), np.float32)
    x[:, ::2] = -0.0
    got = check(x, [-1.0, -2.0], [1, 1], [0, 0], 2)
    assert list(got[4]) == [0, 1] and list(got[3]) == [0, 0]


def test_first_step_has_one_beam():
    r = np.random.default_rng(3)
    B, K, V = 3, 4, 77
    x = r.standard_normal((B * K, V))
    scores = np.where(np.arange(B * K) % K == 0, 0.0, -np.inf)
    got = check(x, scores, np.zeros(B * K), np.zeros(B * K), K)
    np.testing.assert_array_equal(got[3], np.arange(B).repeat(K) * K)


def test_places_without_a_candidate():
    # one live beam and two tokens for four places; a request without any
    x = np.zeros((8, 2), np.float32)
    x[:, 1] = 1
    scores = np.array([-np.inf, -3, np.nan, -np.inf] + [-np.inf] * 4, np.float32)
    got = check(x, scores, np.arange(8), np.zeros(8), 4, eos=1)
    assert list(got[3]) == [1, 1, 2, 3, 4, 5, 6, 7] and list(got[4][:4]) == [1, 0, 1, 1]


def test_finished_beams_keep_their_place():
    r = np.random.default_rng(4)
    x, scores, lengths, _ = inputs(r, 4, 4, 50)
    for alpha in (0.0, 1.0):
        check(x, scores, lengths, np.ones(16), 4, alpha=alpha)
        check(x, scores, lengths, np.arange(16) % 2, 4, alpha=alpha)
    check(x, scores, lengths, np.zeros(16), 4, eos=-1)
    check(x, scores, lengths, np.arange(16) % 2, 4, eos=-1)


@pytest.mark.parametrize("V", [40, 6000])
def test_masked_and_broken_logits(V):
    r = np.random.default_rng([5, V])
    B, K = 4, 3
    x, scores, lengths, done = inputs(r, B, K, V)
    x[0, 3:] = -np.inf            # fewer tokens than places
    x[1] = -np.inf                # none
    x[2, 7] = np.nan
    x[4, 5] = np.inf              # no distribution
    x[5] = np.nan
    x[6, ::2] = -np.inf
    x[7] = -3.4e38                # the type's lowest value is a logit like any other
    x[8] *= 1e20
    x[9] *= 1e-30
    done[:] = 0
    check(x, scores, lengths, done, K)


def test_large_logits_and_lengths():
    r = np.random.default_rng(6)
    x, scores, lengths, done = inputs(r, 4, 4, 3000)
    for shift in (1e4, -1e4, 6.5e4, 7e4, 1e6):
        check((x + shift).astype(np.float32), scores, lengths * 1000, done, 4, alpha=0.6)


def test_in_place_and_strided():
    r = np.random.default_rng(7)
    x, scores, lengths, done = inputs(r, 6, 5, 333)
    check(x, scores, lengths, done, 5, in_place=True)
    check(x, scores, lengths, done, 5, ldl=340)
    check(x, scores, lengths, done, 5, ldl=335, in_place=True, alpha=-0.5)


def test_sums_decide_between_beams_that_lie_close():
    # two beams whose best totals differ by 1e-7: the sums' rounding must not swap them
    r = np.random.default_rng(8)
    V = 20_000
    for trial in range(8):
        x = (r.standard_normal((2, V)) * 2).astype(np.float32)
        w = x.astype(np.float64)
        norm = w.max(1) + np.log(np.exp(w - w.max(1, keepdims=True)).sum(1))
        best = w.max(1) - norm
        scores = np.array([-20.0, 0.0], np.float32)
        scores[1] = np.float32(-20.0 + best[0] - best[1])
        check(x, scores, [5, 5], [0, 0], 2)
