"""Values of the cache that are not finite, or past what 16 bits hold (GPU).

Only V is spoiled, so every score is finite: a channel whose visible values are all
finite has a finite output, within attention_bound of the definition in 64 bits, in
the rows that see the spoiled key and in those that do not.  A row that sees an
infinite or NaN value has no finite output in that channel."""
from __future__ import annotations

import numpy as np
import pytest

from tests._layer import Cache, attend, attention_bound
from tests.test_gpu_attention import KINDS, call

pytestmark = pytest.mark.gpu


def compare(hip, cache, q, scale, window=0, sinks=0):
    got = call(hip, cache, q, scale, window, sinks)
    with np.errstate(invalid="ignore"):
        want, mass, reach = attend(cache, q, scale, window, sinks)
        bound = attention_bound(mass, reach, want, False)
    clean = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), clean)
    bad = np.abs(got[clean] - want[clean]) > bound[clean]
    assert not bad.any(), (int(bad.sum()), got[clean][bad][:3], want[clean][bad][:3])
    return clean


# one value or record of a key: first, in the middle, last; sizes with one lane a
# row's part and with several
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("page", [16, 24, 64])
def test_a_key_with_one_spoiled_part(hip, kind, d, page):
    for news in (1, 3, 70):
        for byte in (0x7c, 0x7e):  # infinity, NaN
            cache = Cache(hip, kind, [150], [news], page, 2, d, seed=31)
            keys = {20, 140} if news == 1 else {20, 147, 148} if news == 3 else {20, 90, 131, 147}
            e = 2 if kind == "f16" else {"q8_0": 34, "q4_0": 18}[kind]
            parts = d if kind == "f16" else d // 32
            for i, p in enumerate(sorted(keys)):
                at = e * (i * 7 % parts if i else parts - 1)
                for rows in (cache.host["v"][cache.table[0, p // page], 1, p % page], cache.rows["v"][0][p, 1]):
                    rows[at:at + 2] = 0, byte
            cache.upload()
            q = np.random.default_rng(32).standard_normal((news, 8, d)).astype(np.float32)
            print(f"spoiled part {kind} d={d} page={page} news={news} {byte:#x}", flush=True)
            clean = compare(hip, cache, q, 1 / np.sqrt(d))
            assert clean[:, :4].all() and not clean[:, 4:].all() and clean[:, 4:].any()
