"""Sizes that the cache's kernels do not count (no GPU): refused before anything is
launched, by every operator over a cache."""
from __future__ import annotations

import pytest

from weft_amd import ggml as G
from tests.test_layer_refusals import A, INVALID, batch, refused


@pytest.mark.parametrize("d,heads", [(32, 1 << 26), (1 << 15, 1 << 16), (1 << 16, 1 << 16), (1 << 30, 2),
                                     ((1 << 31) - 32, (1 << 31) - 1)])
def test_values_of_a_token(d, heads):
    # rows that share memory, as any strides are taken
    pool = G.tensor(G.Q8_0, (d, 1, heads, 1), A[8], [34, 0, 0, 0])
    x = G.tensor(G.F32, (d, heads, 1, 2), A[0], [4, 0, 0, 0])
    one = G.tensor(G.F32, (d, heads, 1, 1), A[0], [4, 0, 0, 0])
    assert refused(G.kv_write, one, one, batch(), pool, pool) == INVALID
    assert refused(G.kv_read, pool, pool, batch(), x, x) == INVALID
    assert refused(G.attention, one, pool, pool, batch(), one, 0.1, 0, 0, A[10], 1 << 30) == INVALID
