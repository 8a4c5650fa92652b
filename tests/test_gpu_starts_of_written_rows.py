"""kv_write of batches whose starts go back or past the call's rows (GPU): as the
batch put in order, which is also how the attention places its queries."""
from __future__ import annotations

import numpy as np
import pytest

from tests._layer import Cache
from tests.test_gpu_kv_cache import KINDS, expected_pool
from tests.test_gpu_starts_out_of_order import CASES, in_order
from weft_amd import ggml as G

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_rows_are_written_where_the_queries_are(hip, kind, case):
    starts, rows = CASES[case]
    seqs, heads, d = len(starts) - 1, 2, 64
    cache = Cache(hip, kind, [120 + i for i in range(seqs)], [0] * seqs, 16, heads, d, seed=case)
    cache.starts = np.array(starts, np.int32)
    cache.upload()
    x = np.random.default_rng(case).standard_normal((rows, heads, d)).astype(np.float32)
    xd = hip.to_dev(x)
    t = G.tensor(G.F32, (d, heads, rows), xd.ptr)
    print(f"kv_write {kind} starts={starts[:8]} rows={rows}", flush=True)
    G.kv_write(t, t, cache.batch, cache.pools["k"], cache.pools["v"])
    hip.torch.cuda.synchronize()
    assert hip.last_error() == 0
    cache.starts = in_order(starts, rows)
    cache.news = list(np.diff(cache.starts))
    for name in ("k", "v"):
        assert np.array_equal(cache.pool(name), expected_pool(cache, name, x))
