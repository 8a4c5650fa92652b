"""Caches whose pages lie far apart (GPU): offsets past 2^32 bytes, and pages of
2^31 bytes and more.  Tolerances are those of the attention's and the cache's own
tests: attention_bound for outputs, equality for records and their values."""
from __future__ import annotations

import numpy as np
import pytest

from tests._layer import RECORD, Cache, attend, attention_bound, decode, encode
from weft_amd import ggml as G

pytestmark = pytest.mark.gpu
NEAR, FAR = (1 << 27) + 64, (1 << 31) + 2  # bytes between pages


def spread_pages(hip, cache, stride):
    """The cache's pools again with their pages ``stride`` bytes apart."""
    torch = hip.torch
    for name in ("k", "v"):
        pool = torch.from_numpy(cache.host[name])
        n, size = pool.shape[0], pool[0].numel()
        far = torch.empty((n - 1) * stride + size, dtype=torch.uint8, device="cuda")
        far.as_strided((n, size), (stride, 1)).copy_(pool.reshape(n, size))
        t = cache.pools[name]
        nb = [{"f16": 2}.get(cache.kind, RECORD[cache.kind]), t.nb[1], t.nb[2], stride]
        cache.dev[name] = far
        cache.pools[name] = G.tensor(t.type, list(t.ne), far.data_ptr(), nb)


def pages_of(cache, name, stride):
    shape = cache.host[name].shape
    size = cache.host[name][0].size
    return cache.dev[name].as_strided((shape[0], size), (stride, 1)).cpu().numpy().reshape(shape)


@pytest.mark.parametrize("kind", ["f16", "q8_0", "q4_0"])
@pytest.mark.parametrize("stride,length", [(NEAR, 640), (FAR, 40)])
def test_attention(hip, kind, stride, length):
    for news in (1, min(length, 70)):
        print(f"attention over far pages {kind} stride={stride} length={length} news={news}", flush=True)
        cache = Cache(hip, kind, [length], [news], 16, 2, 64, seed=length)
        spread_pages(hip, cache, stride)
        q = np.random.default_rng(3).standard_normal((news, 8, 64)).astype(np.float32)
        qd, od = hip.to_dev(q), hip.empty(4 * q.size)
        qt, ot = (G.tensor(G.F32, (64, 8, news), x.ptr) for x in (qd, od))
        size = G.attention_work_size(qt, cache.pools["k"], cache.pools["v"], cache.batch)
        work = hip.empty(max(16, size))
        G.attention(qt, cache.pools["k"], cache.pools["v"], cache.batch, ot, 0.125, 0, 0, work.ptr, size)
        hip.torch.cuda.synchronize()
        assert hip.last_error() == 0
        got = od.numpy(np.float32, q.shape).astype(np.float64)
        want, mass, reach = attend(cache, q, 0.125)
        assert not (np.abs(got - want) > attention_bound(mass, reach, want, False)).any()


@pytest.mark.parametrize("kind", ["f16", "q8_0", "q4_0"])
@pytest.mark.parametrize("stride,length", [(NEAR, 640), (FAR, 40)])
def test_cache(hip, kind, stride, length):
    print(f"cache of far pages {kind} stride={stride} length={length}", flush=True)
    news, heads, d = length - 5, 2, 64
    cache = Cache(hip, kind, [length], [news], 16, heads, d, seed=length)
    spread_pages(hip, cache, stride)
    rng = np.random.default_rng(4)
    x = {name: rng.standard_normal((news, heads, d)).astype(np.float32) for name in ("k", "v")}
    dev = {name: hip.to_dev(x[name]) for name in x}
    G.kv_write(*(G.tensor(G.F32, (d, heads, news), dev[n].ptr) for n in ("k", "v")), cache.batch,
               cache.pools["k"], cache.pools["v"])
    out = {name: hip.empty(4 * length * heads * d) for name in x}
    G.kv_read(cache.pools["k"], cache.pools["v"], cache.batch,
              *(G.tensor(G.F32, (d, heads, length), out[n].ptr) for n in ("k", "v")))
    hip.torch.cuda.synchronize()
    assert hip.last_error() == 0
    for name in ("k", "v"):
        pool = cache.host[name].copy()
        for t in range(news):
            p = 5 + t
            pool[cache.table[0, p // 16], :, p % 16] = encode(kind, x[name][t])
        assert np.array_equal(pages_of(cache, name, stride), pool)
        rows = np.concatenate([cache.rows[name][0][:5], encode(kind, x[name])])
        got = out[name].numpy(np.float32, (length, heads, d))
        assert np.array_equal(got, decode(kind, rows).astype(np.float32))
