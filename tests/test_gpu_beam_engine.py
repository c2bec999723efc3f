"""DeviceLanguageModel.GenerateBeam: what the engine holds and refuses."""
from __future__ import annotations

import numpy as np
import pytest

from cdml import host, synth

pytestmark = pytest.mark.gpu


def engine(cfg, capacity, seed=25):
    lm, _ = host.language_model(cfg, synth.lm_weights(cfg, seed))
    return host.module().DeviceLanguageModel(lm, capacity)


def test_memory_does_not_grow_with_the_steps():
    # keys that cross many chunks, then longer searches: one workspace, allocated before the first step
    cfg = {"vocab": 40, "dim": 32, "heads": 4, "layers": 1, "ff": 32, "max_seq": 1600}
    dev = engine(cfg, 8)
    ids = synth.token_ids(41, 1600, 40)
    first = dev.GenerateBeam([ids[:5], ids[5:8]], 4, 3)
    held = dev.allocations
    long = dev.GenerateBeam([ids[:5], ids[5:8]], 4, 1500)
    assert dev.allocations == held
    dev.GenerateBeam([ids[:1200], ids[:40]], 2, 300)
    dev.GenerateBeam([ids[:1590]], 8, 10)
    assert dev.allocations == held
    again = dev.GenerateBeam([ids[:5], ids[5:8]], 4, 3)
    for a, b in zip(first[0], again[0]):
        for x, y in zip(a, b):
            np.testing.assert_array_equal(x, y)
    np.testing.assert_array_equal(first[1], again[1])
    assert all(len(t) == 1505 for t in long[0][0])


def test_models_that_cannot_be_searched():
    m = host.module()
    dev = engine({"vocab": 20, "dim": 288, "heads": 1, "layers": 1, "ff": 16, "max_seq": 16}, 4)
    held = dev.allocations
    with pytest.raises(m.InvalidOperationException, match="256"):
        dev.GenerateBeam([np.array([1, 2])], 2, 3)
    assert dev.allocations == held  # refused before its pool is allocated
    wide = engine({"vocab": 20, "dim": 256, "heads": 1, "layers": 1, "ff": 16, "max_seq": 16}, 4)
    tokens, scores = wide.GenerateBeam([np.array([1, 2]), np.array([3])], 2, 3)
    assert np.isfinite(scores).all()
    np.testing.assert_array_equal([t[0] for t in wide.GenerateBeam([np.array([1, 2])], 1, 3)[0]],
                                  wide.GenerateGreedy(np.array([[1, 2]]), 3))
