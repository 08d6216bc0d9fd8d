"""GPU: every entry of the tables that nmx_pages_update leaves: a sequence's pages, -1 behind them where it had some
before, and what was there where it never had any."""
from __future__ import annotations

import numpy as np
import pytest

from tests.test_gpu_pages import KV_F16, Box, Model


def entries(m):
    """The tables in full, from the most pages that each sequence has had (now among them)."""
    out = np.full((m.seqs, m.wide), -9, np.int32)
    for s, t in enumerate(m.table):
        out[s, :max(m.had[s], len(t))] = -1
        out[s, :len(t)] = t
    return out


def test_the_model_tells_them_apart():
    m = Model(np.random.default_rng(0), 2, 16, 9, 4, caches=0)
    assert m.step([-1, -1], [0, 0], [40, 5]) == [0, 4, 0, 0]
    assert entries(m).tolist() == [[0, 1, 2, -9], [3, -9, -9, -9]]
    assert m.step([0, 0], [16, 99], [0, 0])[0] == 0
    assert entries(m).tolist() == [[0, -1, -1, -9], [0, 1, 2, -9]]
    assert m.step([0, -1], [99, 0], [0, 0])[0] == 0
    assert entries(m).tolist() == [[0, -1, -1, -9], [-1, -1, -1, -9]]


@pytest.mark.gpu
@pytest.mark.parametrize("seed,S,npages", [(0, 1, 9), (1, 5, 30), (2, 17, 60), (3, 64, 300), (4, 7, 17000)])
def test_entries(dev, seed, S, npages):
    """Steps of all kinds, some without room; the last batch counts its pages in memory."""
    rng = np.random.default_rng(seed)
    m = Model(rng, S, 16, npages, 9, caches=0, kv=KV_F16)
    box = Box(dev, m)
    for i in range(25):
        stay = rng.random(S) < 0.7
        src = np.where(stay, np.arange(S), rng.integers(-1, S, S)).tolist()
        keep = np.where(rng.random(S) < 0.7, 10 ** 6, rng.integers(-2, 150, S)).tolist()
        add = np.where(rng.random(S) < 0.2, rng.integers(0, 100, S), rng.integers(0, 3, S)).tolist()
        pack = int(rng.random() < 0.3)
        assert box.step(src, keep, add, pack) == m.step(src, keep, add, pack), i
        assert (box.b["table"].numpy() == entries(m)).all(), i
    box.free()
