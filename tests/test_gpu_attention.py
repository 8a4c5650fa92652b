"""Attention over the paged cache against 64 bits on the cache's own values (GPU).

Every output lies within attention_bound (what rounding queries, keys, values and
weights once to 16 bits can do); over a call the error's norm is at most 2e-3 of
the result's (four roundings of at most 2^-11 each).  Slots that hold no row of a
sequence are NaN, so a read of one shows."""
from __future__ import annotations

import numpy as np
import pytest

from tests._layer import Cache, attend, attention_bound
from weft_amd import ggml as G

pytestmark = pytest.mark.gpu
KINDS = ["f16", "q8_0", "q4_0"]


def call(hip, cache, q, scale, window=0, sinks=0, src="f32", dst="f32", pad=0, short=0):
    tokens, heads, d = q.shape
    es, ts, fs = (4, G.F32, np.float32) if src == "f32" else (2, G.F16, np.float16)
    ed, td, fd = (4, G.F32, np.float32) if dst == "f32" else (2, G.F16, np.float16)
    host = np.zeros((tokens, heads, d + pad), fs)
    host[..., :d] = q
    qd = hip.to_dev(host)
    od = hip.empty(ed * tokens * heads * (d + pad), fill=0x3C)
    qt = G.tensor(ts, (d, heads, tokens), qd.ptr, [es, es * (d + pad), es * (d + pad) * heads, 0])
    ot = G.tensor(td, (d, heads, tokens), od.ptr, [ed, ed * (d + pad), ed * (d + pad) * heads, 0])
    size = G.attention_work_size(qt, cache.pools["k"], cache.pools["v"], cache.batch)
    work = hip.empty(max(16, size), fill=0x7F)
    G.attention(qt, cache.pools["k"], cache.pools["v"], cache.batch, ot, scale, window, sinks, work.ptr, size)
    hip.torch.cuda.synchronize()
    assert hip.last_error() == 0
    got = od.numpy(fd, (tokens, heads, d + pad))
    if pad:
        assert (np.ascontiguousarray(got[..., d:]).view(np.uint8) == 0x3C).all()
    return got[..., :d].astype(np.float64)


def check(hip, kind, lengths, news, page, kv_heads, heads, d, window=0, sinks=0, src="f32", dst="f32", pad=0,
          slots_first=False, seed=0, spread=1.0, edit=None):
    cache = Cache(hip, kind, lengths, news, page, kv_heads, d, seed, slots_first, spread)
    if edit is not None:
        edit(cache)
        cache.upload()
    tokens = int(cache.starts[-1])
    q = np.random.default_rng(seed + 1).standard_normal((tokens, heads, d)).astype(np.float32)
    if src == "f16":
        q = q.astype(np.float16).astype(np.float32)
    scale = 1 / np.sqrt(d)
    print(f"attention {kind} lengths={lengths[:4]} news={news[:4]} page={page} kv={kv_heads} heads={heads} d={d} "
          f"window={window} sinks={sinks} {src}->{dst} pad={pad} slots_first={slots_first}", flush=True)
    got = call(hip, cache, q, scale, window, sinks, src, dst, pad)
    want, mass, reach = attend(cache, q, scale, window, sinks)
    assert np.isfinite(got).all()
    bad = np.abs(got - want) > attention_bound(mass, reach, want, dst == "f16")
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3], got[bad][:3], want[bad][:3])
    assert (got[mass.sum(-1) == 0] == 0).all()
    norm = np.linalg.norm(want)
    assert np.linalg.norm(got - want) <= 2e-3 * norm + 1e-12
    return cache, q, got


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 257, 1000])
def test_one_token_of_every_length(hip, kind, length):
    check(hip, kind, [length], [1], 16, 2, 8, 128, seed=length)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("share", [1, 3, 8])
def test_head_sizes_and_shared_heads(hip, kind, d, share):
    for lengths, news in (([70, 1, 150], [1, 1, 1]), ([70, 33, 150], [70, 1, 20])):
        check(hip, kind, lengths, news, 24, 2, 2 * share, d, src="f16", dst="f16", seed=d + share)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("page", [16, 32, 128])
def test_chunks_over_pages_of_whole_lines(hip, kind, d, page):
    """Pages of a power of two slots that follow each other, every head size, and
    the same with heads between the slots."""
    for slots_first in (False, True):
        check(hip, kind, [301, 77], [140, 77], page, 2, 4, d, slots_first=slots_first, seed=d + page)
        check(hip, kind, [301, 77], [140, 77], page, 2, 4, d, 50, 3, slots_first=slots_first, seed=d + page)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("news", [2, 4, 5, 16, 17, 31, 32, 33, 63, 64, 65, 130])
def test_chunks_of_every_size(hip, kind, news):
    for before in (0, 1, 97):
        check(hip, kind, [before + news], [news], 32, 1, 4, 64, seed=news + before, dst="f16")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (17, 4), (33, 4), (64, 64), (100, 40), (129, 1),
                                          (1000, 4), (50, 2000)])
def test_windows_and_sinks(hip, kind, window, sinks):
    for lengths, news in (([400, 30, 3], [1, 1, 1]), ([300, 250, 40], [90, 250, 7])):
        check(hip, kind, lengths, news, 16, 2, 8, 64, window, sinks, seed=window + sinks)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [1, 7, 16, 48, 64, 256])
def test_page_sizes_and_layouts(hip, kind, page):
    for slots_first in (False, True):
        for news in ([1, 1], [200, 19]):
            check(hip, kind, [270, 83], news, page, 3, 6, 96, slots_first=slots_first, seed=page)


def test_strides_and_types(hip):
    for src in ("f32", "f16"):
        for dst in ("f32", "f16"):
            for pad in (0, 1, 3, 8):
                for news in ([1, 1], [60, 3]):
                    check(hip, "q8_0", [130, 40], news, 16, 2, 8, 64, src=src, dst=dst, pad=pad, seed=pad)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale,spread", [(0.0, 1.0), (-0.125, 1.0), (1e-6, 1.0), (0.69, 0.2), (0.7, 0.2), (3.0, 0.05),
                                          (-3.0, 0.05), (1000.0, 1e-4)])
def test_scales(hip, kind, scale, spread):
    """Zero, negative, tiny and large ones (past what queries of 16 bits could take)."""
    for news in (1, 70):
        for src in ("f32", "f16"):
            cache = Cache(hip, kind, [150], [news], 16, 2, 64, seed=21)
            q = np.random.default_rng(22).standard_normal((news, 8, 64)) * spread
            q = q.astype(np.float16 if src == "f16" else np.float32).astype(np.float32)
            print(f"attention {kind} scale={scale} news={news} {src}", flush=True)
            got = call(hip, cache, q, scale, src=src)
            want, mass, reach = attend(cache, q, scale)
            assert not (np.abs(got - want) > attention_bound(mass, np.abs(reach), want, False)).any()


@pytest.mark.parametrize("kind", KINDS)
def test_rows_that_see_nothing(hip, kind):
    """Lengths of zero and shorter than the new tokens, sequences without new
    tokens, and queries whose every visible page was given back."""
    check(hip, kind, [0, 3, 20, 50], [2, 7, 0, 1], 16, 2, 4, 64, seed=1)

    def no_pages(cache):
        cache.table[0, :] = -1
        cache.table[1, 1] = -1
    check(hip, kind, [40, 90], [40, 60], 16, 2, 4, 64, seed=2, edit=no_pages)
    check(hip, kind, [40, 90], [1, 1], 16, 2, 4, 64, seed=2, edit=no_pages)


@pytest.mark.parametrize("kind", KINDS)
def test_pages_behind_the_window_may_be_gone(hip, kind):
    def evict(cache):
        for p in range(1, 30):
            cache.table[0, p] = -1 if p % 2 else cache.n_pages + 5
    for n in (1, 40):
        check(hip, kind, [600], [n], 16, 2, 8, 64, window=64, sinks=4, seed=n, edit=evict)


def test_a_length_past_the_table_sees_what_is_there(hip):
    def longer(cache):
        cache.lengths[0] = 1 << 30

    for n in (1, 5):
        cache = Cache(hip, "q8_0", [48], [n], 16, 1, 64, seed=3)
        q = np.random.default_rng(4).standard_normal((n, 4, 64)).astype(np.float32)
        rows = cache.lengths[0]
        longer(cache)
        cache.upload()
        got = call(hip, cache, q, 0.125)
        cache.lengths[0], cache.news[0] = rows, n
        # every query's position is past all 48 keys
        full = Cache(hip, "q8_0", [48], [n], 16, 1, 64, seed=3)
        want = np.zeros_like(got)
        k, v = full.values("k", 0), full.values("v", 0)
        for t in range(n):
            for h in range(4):
                s = k[:, 0] @ q[t, h].astype(np.float64) * 0.125
                p = np.exp(s - s.max())
                want[t, h] = p @ v[:, 0] / p.sum()
        assert np.linalg.norm(got - want) <= 2e-3 * np.linalg.norm(want)


def test_rows_of_no_sequence_stay(hip):
    def later(cache):
        cache.starts[:] = [2, 4]
        cache.news = [2]
    cache = Cache(hip, "f16", [30], [6], 16, 1, 64, seed=5)
    later(cache)
    cache.upload()
    q = np.random.default_rng(4).standard_normal((6, 4, 64)).astype(np.float32)
    got = call(hip, cache, q, 0.125)
    untouched = np.frombuffer(b"\x3c" * 4, np.float32)[0]
    assert (got[[0, 1, 4, 5]] == untouched).all()
    want, _, _ = attend(cache, q, 0.125)
    assert np.linalg.norm(got[2:4] - want[2:4]) <= 2e-3 * np.linalg.norm(want[2:4])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("news", [1, 50])
def test_one_key_rules(hip, kind, news):
    """Keys far apart in score: one weight is one and the rest are nearly zero,
    so a row is one key's value."""
    check(hip, kind, [200], [news], 16, 1, 4, 64, seed=6, spread=6.0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("news", [1, 3, 70])
def test_infinity_and_nan_in_keys_nobody_sees(hip, kind, news):
    """An infinite or NaN key or value reaches only the queries that see it: of
    a chunk, those before the window has passed it."""
    length, window, sinks = 150, 60, 2
    cache = Cache(hip, kind, [length], [news], 16, 1, 64, seed=7)
    q = np.random.default_rng(8).standard_normal((news, 4, 64)).astype(np.float32)
    lowest = length - news - window + 1  # the first key of the first query's window
    spoiled = {5, lowest - 1} | ({lowest, lowest + 5} if news > 1 else set())
    for name, byte in (("k", 0x7c), ("v", 0x7e)):
        for p in spoiled:
            row = cache.host[name][cache.table[0, p // 16], 0, p % 16]
            row[:2] = 0, byte  # an infinite or NaN value, or a record's step
            cache.rows[name][0][p, 0, :2] = 0, byte
    cache.upload()
    got = call(hip, cache, q, 0.125, window, sinks)
    with np.errstate(invalid="ignore"):
        want, mass, reach = attend(cache, q, 0.125, window, sinks)
    clean = np.isfinite(want).all((1, 2))
    assert clean.sum() == (news if news == 1 else max(0, news - 6)) and clean.any() == (news != 3)
    assert (np.isfinite(got).all((1, 2)) == clean).all()
    bound = attention_bound(mass, reach, want, False)
    assert (np.abs(got[clean] - want[clean]) <= bound[clean]).all()


def test_long_context_and_batches(hip):
    """Splits of the key axis: one long sequence, and many uneven ones."""
    check(hip, "q4_0", [20011], [1], 64, 2, 8, 128, seed=9)
    check(hip, "f16", [9001], [9], 256, 1, 8, 128, seed=9)
    check(hip, "q8_0", [5000, 12, 1700, 1, 333] * 15, [1] * 75, 64, 1, 4, 64, seed=10)
    check(hip, "q8_0", [5000, 12, 1700, 1, 333], [30, 12, 1, 1, 200], 64, 1, 4, 64, seed=10, dst="f16")


def test_two_calls_agree_bit_for_bit(hip):
    for news in ([1, 1], [150, 40]):
        a = check(hip, "q8_0", [3000, 700], news, 64, 2, 8, 128, seed=11)[2]
        b = check(hip, "q8_0", [3000, 700], news, 64, 2, 8, 128, seed=11)[2]
        assert np.array_equal(a, b)


def test_graph_replays_follow_the_lengths(hip):
    """A captured decode step replayed as the lengths grow."""
    torch = hip.torch
    cache = Cache(hip, "q8_0", [120, 45], [1, 1], 16, 2, 64, seed=12)
    q = np.random.default_rng(13).standard_normal((2, 8, 64)).astype(np.float32)
    qd, od = hip.to_dev(q), hip.empty(4 * q.size)
    qt, ot = G.tensor(G.F32, (64, 8, 2), qd.ptr), G.tensor(G.F32, (64, 8, 2), od.ptr)
    size = G.attention_work_size(qt, cache.pools["k"], cache.pools["v"], cache.batch)
    work = hip.empty(max(16, size), fill=0x7F)

    def step():
        G.attention(qt, cache.pools["k"], cache.pools["v"], cache.batch, ot, 0.125, 0, 0, work.ptr, size)

    step()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            hip._lib.set_stream(side.cuda_stream)
            step()
    hip._lib.set_stream(torch.cuda.current_stream().cuda_stream)
    for lengths in ([120, 45], [60, 3], [119, 44], [1, 45], [120, 45]):
        cache.dev["lengths"].t[:8].view(torch.int32).copy_(torch.tensor(lengths, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = od.numpy(np.float32).copy()
        step()
        torch.cuda.synchronize()
        assert np.array_equal(replayed, od.numpy(np.float32))
