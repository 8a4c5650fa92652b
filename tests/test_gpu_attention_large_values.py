"""Quantized values of V past what 16 bits hold (GPU): kv_write makes such records of
finite values, a step of 16 bits times a code.  They are finite values like others: to
the rows that see their key, in steps that all rows see whole and in steps they do
not, and nothing to the rows before."""
from __future__ import annotations

import numpy as np
import pytest

from tests._layer import Cache, attend, attention_bound, encode
from tests.test_gpu_attention import call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["q8_0", "q4_0"])
@pytest.mark.parametrize("d", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("page", [16, 24, 64])
def test_large_values(hip, kind, d, page):
    for length, news in ((150, 1), (150, 3), (150, 70), (400, 1), (400, 3), (400, 70), (1500, 130)):
        for window, sinks in ((0, 0), (60, 2)):
            cache = Cache(hip, kind, [length], [news], page, 2, d, seed=51)
            rng = np.random.default_rng(52)
            first = length - news
            for p in {1, 5, 70, first - 30, first, min(first + 1, length - 1), length - 2, length - 1}:
                x = (rng.standard_normal((1, d)) * rng.choice([3e4, 1e5, 1e6])).astype(np.float32)
                if kind == "q8_0":
                    x = np.clip(x, -8e6, 8e6)  # its steps stay in 16 bits
                else:
                    x = np.clip(x, -5e5, 5e5)
                cache.rows["v"][0][p, 1] = encode(kind, x)[0]
                cache.host["v"][cache.table[0, p // page], 1, p % page] = cache.rows["v"][0][p, 1]
            cache.upload()
            q = rng.standard_normal((news, 8, d)).astype(np.float32)
            print(f"large values {kind} d={d} page={page} length={length} news={news} window={window}", flush=True)
            got = call(hip, cache, q, 1 / np.sqrt(d), window, sinks)
            want, mass, reach = attend(cache, q, 1 / np.sqrt(d), window, sinks)
            assert np.abs(cache.values("v", 0)).max() > 65504 and np.isfinite(want).all()
            assert np.isfinite(got).all()
            bad = np.abs(got - want) > attention_bound(mass, reach, want, False)
            assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3], got[bad][:3], want[bad][:3])
