"""kv_write and kv_read on the paged cache (GPU): records bit for bit as the
oracle's quantizers write them, values exactly the records', and no byte of the
pool touched beside the new tokens' rows."""
from __future__ import annotations

import numpy as np
import pytest

from tests._layer import Cache, RECORD, decode, encode, row_bytes
from weft_amd import ggml as G

pytestmark = pytest.mark.gpu
KINDS = ["f16", "q8_0", "q4_0"]


def write(hip, cache, src="f32", seed=1, pad=0, data=None):
    """Writes every sequence's new tokens; the rows written, as float32."""
    rng = np.random.default_rng(seed)
    tokens, h, d = int(cache.starts[-1]), cache.kv_heads, cache.d
    e, t = (4, G.F32) if src == "f32" else (2, G.F16)
    out, args, keep = {}, [], []
    for name in ("k", "v"):
        x = rng.standard_normal((tokens, h, d)).astype(np.float32) if data is None else data.astype(np.float32)
        if src == "f16":
            x = x.astype(np.float16).astype(np.float32)
        host = np.zeros((tokens, h, d + pad), np.float32 if src == "f32" else np.float16)
        host[..., :d] = x
        dev = hip.to_dev(host)
        keep.append(dev)
        args.append(G.tensor(t, (d, h, tokens), dev.ptr, [e, e * (d + pad), e * (d + pad) * h, 0]))
        out[name] = x
    print(f"kv_write {cache.kind} lengths={cache.lengths[:4]} news={cache.news[:4]} page={cache.page} heads={h} d={d} "
          f"src={src} slots_first={cache.slots_first}", flush=True)
    G.kv_write(*args, cache.batch, cache.pools["k"], cache.pools["v"])
    hip.torch.cuda.synchronize()
    assert hip.last_error() == 0
    return out


def expected_pool(cache, name, x):
    want = cache.host[name].copy()
    for i, (length, n) in enumerate(zip(cache.lengths, cache.news)):
        for t in range(n):
            p = length - n + t
            if 0 <= p < cache.table.shape[1] * cache.page and 0 <= cache.table[i, p // cache.page] < cache.n_pages:
                want[cache.table[i, p // cache.page], :, p % cache.page] = encode(cache.kind, x[cache.starts[i] + t])
    return want


SHAPES = [  # lengths, news, page, heads, d
    ([1], [1], 16, 8, 128), ([131], [1], 16, 8, 128), ([40, 7, 100], [40, 7, 100], 16, 2, 64),
    ([33, 65, 5, 64], [1, 65, 0, 32], 32, 3, 96), ([130, 70], [3, 70], 24, 1, 256), ([9, 3], [9, 1], 1, 5, 32),
    ([300], [300], 256, 2, 192), ([20] * 70, [2] * 70, 7, 1, 160),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_rows_are_the_quantizers_records(hip, kind, case):
    lengths, news, page, heads, d = SHAPES[case]
    for slots_first, src, pad in ((False, "f32", 0), (True, "f16", 0), (False, "f32", 1), (True, "f16", 3)):
        cache = Cache(hip, kind, lengths, news, page, heads, d, seed=case, slots_first=slots_first)
        x = write(hip, cache, src, seed=case, pad=pad)
        for name in ("k", "v"):
            assert np.array_equal(cache.pool(name), expected_pool(cache, name, x[name]))


def test_absent_pages_short_lengths_and_rows_of_no_sequence_are_left(hip):
    """A page given back, an entry past the pool, a length shorter than the new
    tokens, a length past the table, starts that leave rows over."""
    for kind in KINDS:
        cache = Cache(hip, kind, [40, 3, 64, 10], [40, 5, 2, 2], 16, 2, 64, seed=2)
        cache.table[0, 1], cache.table[2, 3] = -1, cache.n_pages
        cache.lengths[1], cache.lengths[3] = 2, 16 * cache.table.shape[1] + 1
        cache.upload()
        x = write(hip, cache)
        for name in ("k", "v"):
            assert np.array_equal(cache.pool(name), expected_pool(cache, name, x[name]))
        cache = Cache(hip, kind, [8, 8], [3, 3], 16, 2, 64, seed=3)
        cache.starts[:] = [2, 3, 5]  # rows 0 and 1 belong to none
        cache.news = [1, 2]
        cache.upload()
        cache.starts[-1] = 5
        x = write(hip, cache)
        for name in ("k", "v"):
            assert np.array_equal(cache.pool(name), expected_pool(cache, name, x[name]))


def test_records_of_extremes(hip):
    """Zeros, one value, both signs of the largest magnitude (the first counts),
    ties between codes, subnormal steps, the largest 16-bit values."""
    d = 64
    x = np.zeros((6, 1, d), np.float32)
    x[1, 0, 5] = -2.5
    x[2, 0, 3], x[2, 0, 40], x[2, 0, 4], x[2, 0, 41] = 4.0, -4.0, -4.0, 4.0
    x[3, 0] = (np.arange(d) - 32) / 2
    x[4, 0] = np.arange(d) * 1e-6
    x[5, 0] = np.linspace(-65000, 65000, d)
    for kind in KINDS:
        cache = Cache(hip, kind, [6], [6], 4, 1, d, seed=1)
        got = write(hip, cache, data=x)
        for name in ("k", "v"):
            assert np.array_equal(cache.pool(name), expected_pool(cache, name, got[name]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_reads_are_the_records_values(hip, kind, case):
    lengths, news, page, heads, d = SHAPES[case]
    for slots_first, dst, pad, extra in ((False, "f16", 0, 0), (True, "f32", 0, 5), (False, "f32", 1, 0), (True, "f16", 1, 3)):
        cache = Cache(hip, kind, lengths, news, page, heads, d, seed=case + 50, slots_first=slots_first)
        cache.table[0, -1] = -1 if len(lengths) > 1 else cache.table[0, -1]
        cache.upload()
        n, seqs = max(lengths) + extra, len(lengths)
        e, t, ft = (4, G.F32, np.float32) if dst == "f32" else (2, G.F16, np.float16)
        w = d + pad
        outs = [hip.empty(e * seqs * n * heads * w, fill=0x3C) for _ in range(2)]
        desc = [G.tensor(t, (d, heads, n, seqs), x.ptr, [e, e * w, e * w * heads, e * w * heads * n]) for x in outs]
        print(f"kv_read {kind} case={case} slots_first={slots_first} {dst} pad={pad}", flush=True)
        G.kv_read(cache.pools["k"], cache.pools["v"], cache.batch, *desc)
        hip.torch.cuda.synchronize()
        for name, dev in zip(("k", "v"), outs):
            got = dev.numpy(ft, (seqs, n, heads, w))
            want = np.zeros((seqs, n, heads, d), ft)
            for i, length in enumerate(lengths):
                there = np.repeat(cache.table[i], page)[:length] >= 0
                v = cache.values(name, i).astype(np.float32).astype(ft)
                want[i, :length] = np.where(there[:, None, None], v, 0)
            assert np.array_equal(got[..., :d], want)
            assert (got[..., d:].view(np.uint8) == 0x3C).all()


def test_offsets_past_32_bits(hip):
    """A pool of more than 4 GiB: its last pages are written and read back."""
    torch = hip.torch
    kind, page, heads, d = "q8_0", 64, 8, 256
    rb = row_bytes(kind, d)
    n_pages = (1 << 32) // (rb * heads * page) + 5
    k = torch.zeros(n_pages * page * heads * rb, dtype=torch.uint8, device="cuda")
    v = torch.zeros(n_pages * page * heads * rb, dtype=torch.uint8, device="cuda")
    table = hip.to_dev(np.array([[n_pages - 1, n_pages - 3]], np.int32))
    starts, lengths = hip.to_dev(np.array([0, 100], np.int32)), hip.to_dev(np.array([100], np.int32))
    pools = [G.tensor(G.Q8_0, (d, page, heads, n_pages), x.data_ptr()) for x in (k, v)]
    batch = G.kv_batch(G.tensor(G.I32, (2, 1), table.ptr), G.tensor(G.I32, (2,), starts.ptr),
                       G.tensor(G.I32, (1,), lengths.ptr))
    x = np.random.default_rng(0).standard_normal((100, heads, d)).astype(np.float32)
    xd = hip.to_dev(x)
    t = G.tensor(G.F32, (d, heads, 100), xd.ptr)
    G.kv_write(t, t, batch, *pools)
    outs = [hip.empty(4 * 100 * heads * d) for _ in range(2)]
    G.kv_read(*pools, batch, *[G.tensor(G.F32, (d, heads, 100, 1), y.ptr) for y in outs])
    torch.cuda.synchronize()
    want = decode(kind, encode(kind, x)).astype(np.float32)
    for y in outs:
        assert np.array_equal(y.numpy(np.float32, (100, heads, d)), want)
    del k, v
    torch.cuda.empty_cache()


def test_write_and_read_on_another_stream(hip):
    torch = hip.torch
    cache = Cache(hip, "q8_0", [300], [300], 16, 4, 128, seed=4, fill=False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    hip._lib.set_stream(side.cuda_stream)
    try:
        x = write(hip, cache)
    finally:
        hip._lib.set_stream(torch.cuda.current_stream().cuda_stream)
    for name in ("k", "v"):
        assert np.array_equal(cache.pool(name), expected_pool(cache, name, x[name]))
    assert RECORD["q8_0"] == 34
