"""Batches whose starts go back, or past the call's rows (GPU): a start below one
before it counts as that one and one past the rows as their number, so the call gives
what the batch put in order gives, bit for bit."""
from __future__ import annotations

import numpy as np
import pytest

from tests._layer import Cache
from tests.test_gpu_attention import KINDS, call

pytestmark = pytest.mark.gpu

CASES = [  # starts, the call's rows
    ([0, 50, 0, 100], 100), ([0, 50, 10, 30, 100], 100), ([0, 100, 0, 100, 0, 100], 100), ([100, 0, 60, 100], 100),
    ([40, -5, 90, 20, 1 << 30], 100), ([0, 30, 20, 70], 60), ([-(1 << 31), 12, (1 << 31) - 1, 3], 20),
    ([0, 7, 3, 8, 2, 9, 1, 10], 10), ([0, *([3, 1] * 40), 60], 60),
]


def in_order(starts, rows):
    return np.maximum.accumulate(np.clip(starts, 0, rows)).astype(np.int32)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("heads", [1, 8])
def test_attention(hip, kind, case, heads):
    starts, rows = CASES[case]
    seqs = len(starts) - 1
    q = np.random.default_rng(case).standard_normal((rows, heads, 64)).astype(np.float32)
    print(f"attention {kind} starts={starts[:8]} rows={rows} heads={heads}", flush=True)
    got = []
    for s in (in_order(starts, rows), np.array(starts, np.int32)):
        # long enough for splits, which the second launch joins
        cache = Cache(hip, kind, [900 + 7 * i for i in range(seqs)], [0] * seqs, 16, 1, 64, seed=case)
        cache.starts = s
        cache.upload()
        got.append(call(hip, cache, q, 0.125))
    assert np.isfinite(got[0]).all()
    assert np.array_equal(*got)
