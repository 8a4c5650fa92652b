"""Every output of the attention is finite and within attention_bound (GPU), over
scales of any size and pages far apart: a NaN, as a read of a slot that holds no row
gives, is an error, and so is an output that is not written."""
from __future__ import annotations

import numpy as np
import pytest

from tests._layer import Cache, attend, attention_bound
from tests.test_gpu_attention import KINDS, call
from tests.test_gpu_far_pages import FAR, NEAR, spread_pages
from weft_amd import ggml as G

pytestmark = pytest.mark.gpu


def within(got, want, mass, reach):
    assert np.isfinite(got).all()
    error = np.abs(got - want)
    assert (error <= attention_bound(mass, np.abs(reach), want, False)).all(), error.max()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale,spread", [(0.0, 1.0), (-0.125, 1.0), (1e-6, 1.0), (0.69, 0.2), (0.7, 0.2), (3.0, 0.05),
                                          (-3.0, 0.05), (1000.0, 1e-4)])
def test_scales(hip, kind, scale, spread):
    for news in (1, 70):
        for src in ("f32", "f16"):
            cache = Cache(hip, kind, [150], [news], 16, 2, 64, seed=21)
            q = np.random.default_rng(22).standard_normal((news, 8, 64)) * spread
            q = q.astype(np.float16 if src == "f16" else np.float32).astype(np.float32)
            print(f"attention {kind} scale={scale} news={news} {src}", flush=True)
            within(call(hip, cache, q, scale, src=src), *attend(cache, q, scale))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("stride,length", [(NEAR, 640), (FAR, 40)])
def test_pages_far_apart(hip, kind, stride, length):
    for news in (1, min(length, 70)):
        print(f"attention over far pages {kind} stride={stride} length={length} news={news}", flush=True)
        cache = Cache(hip, kind, [length], [news], 16, 2, 64, seed=length)
        spread_pages(hip, cache, stride)
        q = np.random.default_rng(3).standard_normal((news, 8, 64)).astype(np.float32)
        qd, od = hip.to_dev(q), hip.empty(4 * q.size, fill=0xFF)  # NaN
        qt, ot = (G.tensor(G.F32, (64, 8, news), x.ptr) for x in (qd, od))
        size = G.attention_work_size(qt, cache.pools["k"], cache.pools["v"], cache.batch)
        work = hip.empty(max(16, size), fill=0xFF)
        G.attention(qt, cache.pools["k"], cache.pools["v"], cache.batch, ot, 0.125, 0, 0, work.ptr, size)
        hip.torch.cuda.synchronize()
        assert hip.last_error() == 0
        within(od.numpy(np.float32, q.shape).astype(np.float64), *attend(cache, q, 0.125))
