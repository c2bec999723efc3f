"""DeviceLanguageModel.GenerateBeam: beam search over the paged cache against a search that
scores every beam with the oracle's whole forward pass."""
from __future__ import annotations

import numpy as np
import pytest

from cdml import host, synth
from oracle import oracle as O

pytestmark = pytest.mark.gpu


def search(ref, prompt, K, n, eos, alpha):
    """(beams best first, scores, the smallest gap that decided anything)."""
    beams, gap = [([], 0.0, False)], np.inf
    alpha = float(np.float32(alpha))
    for _ in range(n):
        found = []
        for i, (toks, score, done) in enumerate(beams):
            if done:
                found.append((score / len(toks) ** alpha, -i, 0, toks, score, True))
                continue
            x = ref.forward(np.array(list(prompt) + toks, np.int32))[-1].astype(np.float64)
            logp = x - x.max() - np.log(np.exp(x - x.max()).sum())
            for t in np.argsort(-logp, kind="stable")[:K + 1]:
                total = score + logp[t]
                found.append((total / (len(toks) + 1) ** alpha, -i, -t, toks + [int(t)], total, t == eos))
        found.sort(key=lambda f: f[:3], reverse=True)
        keys = np.array([f[0] for f in found[:K + 1]])
        gap = min(gap, np.min(-np.diff(keys), initial=np.inf))
        beams = [f[3:] for f in found[:K]]
    return [b[0] for b in beams], [b[1] for b in beams], gap


def model(cfg, seed, capacity, biased=True):
    w = synth.lm_weights(cfg, seed, biased=biased)
    # logits spread as a trained model's, so that a search has something to find
    w["out_proj"] = w["out_proj"] * np.float32(4)
    lm, _ = host.language_model(cfg, w)
    return host.module().DeviceLanguageModel(lm, capacity), O.LanguageModel(cfg, w)


@pytest.mark.parametrize("heads,K,n,alpha,eos", [(4, 1, 12, 0.0, -1), (4, 4, 20, 0.0, -1), (2, 3, 18, 0.7, 5),
                                                 (4, 4, 20, 0.0, 17), (1, 5, 9, 1.0, -1)])
def test_beams_match_the_whole_search(heads, K, n, alpha, eos):
    cfg = {"vocab": 200, "dim": 64, "heads": heads, "layers": 2, "ff": 128, "max_seq": 64}
    dev, ref = model(cfg, 21, 4 * K)
    ids = synth.token_ids(31, 100, 200)
    prompts = [ids[:7], ids[7:8], ids[8:40], ids[40:57]]  # ragged, one of a single token
    tokens, scores = dev.GenerateBeam(prompts, K, n, eos, alpha)
    assert scores.shape == (4, K)
    for p, got, s in zip(prompts, tokens, scores):
        want, total, gap = search(ref, p, K, n, eos, alpha)
        assert gap > 1e-4  # far above the logits' rounding: the choices are decided
        assert len(got) == K
        for g, w in zip(got, want):
            if eos in w:
                w = w[:w.index(eos) + 1]
            np.testing.assert_array_equal(g, list(p) + w)
        np.testing.assert_allclose(s, total, rtol=1e-3, atol=1e-3)


def test_one_beam_is_greedy():
    cfg = {"vocab": 200, "dim": 64, "heads": 4, "layers": 2, "ff": 128, "max_seq": 64}
    dev, _ = model(cfg, 22, 6)
    ids = synth.token_ids(32, 6 * 20, 200).reshape(6, 20)
    greedy = dev.GenerateGreedy(ids, 30)
    for _ in range(2):  # a second search starts from an empty pool again
        tokens, _ = dev.GenerateBeam(list(ids), 1, 30)
        np.testing.assert_array_equal([t[0] for t in tokens], greedy)
    np.testing.assert_array_equal(dev.GenerateGreedy(ids, 30), greedy)


def test_length_limits_and_refusals():
    cfg = {"vocab": 50, "dim": 32, "heads": 2, "layers": 1, "ff": 64, "max_seq": 24}
    dev, ref = model(cfg, 23, 6)
    ids = synth.token_ids(33, 24, 50)
    tokens, scores = dev.GenerateBeam([ids[:20], ids[:3]], 3, 40)
    assert [len(t) for beams in tokens for t in beams] == [24] * 3 + [7] * 3
    tokens, scores = dev.GenerateBeam([ids], 2, 5)
    assert all(np.array_equal(t, ids) for t in tokens[0]) and not scores.any()
    m = host.module()
    for bad in (([], 2, 5), ([ids[:3]], 0, 5), ([ids[:3]], 7, 5), ([ids[:3]] * 4, 2, 5), ([ids[:3]], 2, -1),
                ([ids[:3]], 2, 5, 50), ([np.array([50])], 2, 5), ([np.array([-1])], 2, 5)):
        with pytest.raises(m.ArgumentOutOfRangeException):
            dev.GenerateBeam(*bad)
    for bad in ([ids[:0]], [np.arange(25) % 50]):
        with pytest.raises(m.ArgumentException):
            dev.GenerateBeam(bad, 2, 5)


def test_fewer_tokens_than_beams():
    cfg = {"vocab": 3, "dim": 16, "heads": 2, "layers": 1, "ff": 32, "max_seq": 40}
    dev, ref = model(cfg, 24, 5)
    tokens, scores = dev.GenerateBeam([np.array([1, 2])], 5, 1)
    x = ref.forward(np.array([1, 2], np.int32))[-1].astype(np.float64)
    logp = np.sort(x - x.max() - np.log(np.exp(x - x.max()).sum()))[::-1]
    np.testing.assert_allclose(scores[0][:3], logp, atol=1e-4)
    assert np.isneginf(scores[0][3:]).all()
    tokens, scores = dev.GenerateBeam([np.array([1, 2])], 5, 30)
    assert np.isfinite(scores).all() and len({tuple(t) for t in tokens[0]}) == 5
