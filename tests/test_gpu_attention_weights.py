"""Softmax weights far below a row's largest (GPU).

One key takes nearly all of the weight and its value is zero, so the output is the
sum over keys whose weights are e^-12 to e^-18 of it.  Scores are exact: the key's
values and the queries have 16 bits.  What is left are roundings of at most 2^-11
each of a value, a weight and (in two places) a score, on keys whose values are
independent, so the error's norm is at most four of them: 2e-3 of the result's."""
from __future__ import annotations

import numpy as np
import pytest

from tests._layer import Cache, attend, encode
from tests.test_gpu_attention import KINDS, call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("length,news", [(1000, 1), (1000, 7), (4099, 1), (4099, 70)])
def test_a_key_that_takes_nearly_all_the_weight(hip, kind, d, length, news):
    # 127 / 64 and 2 are a record's largest value with a step of 2^-6 and 2^-2: exact
    big = 127 / 64 if kind == "q8_0" else 2.0
    for gap in (12, 15, 18):
        for at in (0, 133):
            cache = Cache(hip, kind, [length], [news], 16, 1, d, seed=41, spread=0.5)
            page, slot = cache.table[0, at // 16], at % 16
            for name, x in (("k", np.full((1, d), big, np.float32)), ("v", np.zeros((1, d), np.float32))):
                cache.host[name][page, 0, slot] = cache.rows[name][0][at, 0] = encode(kind, x)[0]
            cache.upload()
            scale = 1 / np.sqrt(d)
            rng = np.random.default_rng(42)
            q = gap / (scale * big * d) + rng.standard_normal((news, 4, d)) * 0.1
            q = q.astype(np.float16).astype(np.float32)
            print(f"attention {kind} d={d} length={length} news={news} gap={gap} at={at}", flush=True)
            want, _, _ = attend(cache, q, scale)
            for src in ("f32", "f16"):
                got = call(hip, cache, q, scale, src=src)
                assert np.isfinite(got).all()
                for row in range(news):
                    error, size = np.linalg.norm(got[row] - want[row]), np.linalg.norm(want[row])
                    assert error <= 2e-3 * size, (gap, at, src, row, error / size)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [300, 1000, 3000, 1e4])
def test_scores_of_any_size(hip, kind, size):
    """Scores of 1e5 to 1e9, whose 32 bits no longer hold their fractions.  A row whose
    largest leads by more than roundings of 2^-11 of its products can move it (twice, of
    each score) is its key's value."""
    for news in (1, 5, 70):
        cache = Cache(hip, kind, [150], [news], 16, 2, 64, seed=61, spread=size)
        q = np.random.default_rng(62).standard_normal((news, 8, 64)) * size
        q = q.astype(np.float16).astype(np.float32)
        print(f"attention {kind} scores of {size}^2 news={news}", flush=True)
        k = [cache.values("k", 0)[:, h // 4] for h in range(8)]
        v = [cache.values("v", 0)[:, h // 4] for h in range(8)]
        for src in ("f32", "f16"):
            got = call(hip, cache, q, 0.125, src=src)
            assert np.isfinite(got).all()
            checked = 0
            for t in range(news):
                for h in range(8):
                    seen = k[h][:150 - news + t + 1]
                    s = seen @ q[t, h] * 0.125
                    first, second = np.argsort(s)[:-3:-1]
                    if s[first] - s[second] > 50 + 4 * 2.1 * 2.0 ** -11 * 0.125 * (np.abs(seen) @ np.abs(q[t, h])).max():
                        checked += 1
                        want = v[h][first]
                        assert (np.abs(got[t, h] - want) <= np.abs(want) * 2.0 ** -10).all()
            assert checked > 2 * news
