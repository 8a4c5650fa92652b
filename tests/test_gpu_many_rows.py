"""Calls of so many rows that a launch of one thread a value, or of a workgroup a row,
would pass 2^32 threads (GPU).  Rows share memory where they may, so that the calls
stay small."""
from __future__ import annotations

import numpy as np
import pytest

from tests._layer import decode, encode
from weft_amd import ggml as G

pytestmark = pytest.mark.gpu


def test_norm(hip):
    torch = hip.torch
    rows, k = (1 << 26) + 3 + 4, 4
    x = torch.arange(rows, device="cuda", dtype=torch.int32).remainder_(1009).float().add_(1)
    y = torch.full((rows, k), float("nan"), device="cuda", dtype=torch.float16)
    # row i is x[i], x[i + 1], ..: rows lie one value apart
    n = rows - k
    print(f"add_rms_norm rows={n} k={k}", flush=True)
    G.add_rms_norm(G.tensor(G.F32, (k, n), x.data_ptr(), [4, 4, 0, 0]), None, None, None,
                   G.tensor(G.F16, (k, n), y.data_ptr(), [2, 8, 0, 0]), 1e-5)
    torch.cuda.synchronize()
    assert hip.last_error() == 0
    y = y[:n]
    assert torch.isfinite(y).all()
    for at in (0, 12345, n - 1000):
        s = x[:n + k - 1].unfold(0, k, 1)[at:at + 1000].double()
        want = s / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-5)
        # 16 bits' rounding and a few of 32
        assert ((y[at:at + 1000].double() - want).abs() <= want.abs() * (2.0 ** -11 + 2.0 ** -20)).all()


def test_write(hip):
    """All but the last tokens belong to no sequence, and all read one row but they."""
    torch = hip.torch
    tokens, d, page = (1 << 26) + 5, 32, 8
    x = np.random.default_rng(1).standard_normal((1, d)).astype(np.float32)
    xd = hip.to_dev(x)
    pools = [hip.empty(page * 34, fill=0x11) for _ in range(2)]
    desc = [G.tensor(G.Q8_0, (d, page, 1, 1), p.ptr) for p in pools]
    table, starts = hip.to_dev(np.zeros((1, 1), np.int32)), hip.to_dev(np.array([tokens - 3, tokens], np.int32))
    lengths = hip.to_dev(np.array([5], np.int32))
    batch = G.kv_batch(G.tensor(G.I32, (1, 1), table.ptr), G.tensor(G.I32, (2,), starts.ptr),
                       G.tensor(G.I32, (1,), lengths.ptr))
    rows = G.tensor(G.F32, (d, 1, tokens), xd.ptr, [4, 0, 0, 0])
    print(f"kv_write tokens={tokens}", flush=True)
    G.kv_write(rows, rows, batch, *desc)
    torch.cuda.synchronize()
    assert hip.last_error() == 0
    want = np.full((page, 34), 0x11, np.uint8)
    want[2:5] = encode("q8_0", x)
    for p in pools:
        assert np.array_equal(p.numpy(np.uint8, (page, 34)), want)


def test_read(hip):
    """Only the last page is there."""
    torch = hip.torch
    n, d, page = (1 << 27) + 9, 32, 1 << 20
    width = -(-n // page)
    x = np.random.default_rng(2).standard_normal((9, d)).astype(np.float32)
    records = encode("q8_0", x)
    pool = torch.zeros(page * 34, dtype=torch.uint8, device="cuda")
    pool[:9 * 34] = torch.from_numpy(records.reshape(-1)).cuda()
    desc = G.tensor(G.Q8_0, (d, page, 1, 1), pool.data_ptr())
    table = np.full((1, width), -1, np.int32)
    table[0, -1] = 0
    table, starts = hip.to_dev(table), hip.to_dev(np.array([0, 0], np.int32))
    lengths = hip.to_dev(np.array([n], np.int32))
    batch = G.kv_batch(G.tensor(G.I32, (width, 1), table.ptr), G.tensor(G.I32, (2,), starts.ptr),
                       G.tensor(G.I32, (1,), lengths.ptr))
    outs = [torch.full((n, d), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2)]
    print(f"kv_read positions={n}", flush=True)
    G.kv_read(desc, desc, batch, *(G.tensor(G.F16, (d, 1, n, 1), y.data_ptr()) for y in outs))
    torch.cuda.synchronize()
    assert hip.last_error() == 0
    want = torch.from_numpy(decode("q8_0", records).astype(np.float16)).cuda()
    for y in outs:
        assert torch.equal(y[-9:], want)
        assert not y[:-9].any()
    del outs, y
    torch.cuda.empty_cache()


def test_attention(hip):
    """257 sequences of one token, 65535 heads on the same queries and the same rows
    of the cache: every output row is the first."""
    torch = hip.torch
    seqs, heads, d, page, length = 257, 65535, 64, 16, 5
    k, v = np.random.default_rng(3).standard_normal((2, length, d)).astype(np.float32)
    pools = []
    for x in (k, v):
        pool = np.zeros((page, 68), np.uint8)
        pool[:length] = encode("q8_0", x)
        pools.append(hip.to_dev(pool))
    desc = [G.tensor(G.Q8_0, (d, page, heads, 1), p.ptr, [34, 68, 0, 0]) for p in pools]
    table, starts = hip.to_dev(np.zeros((seqs, 1), np.int32)), hip.to_dev(np.arange(seqs + 1, dtype=np.int32))
    lengths = hip.to_dev(np.full(seqs, length, np.int32))
    batch = G.kv_batch(G.tensor(G.I32, (1, seqs), table.ptr), G.tensor(G.I32, (seqs + 1,), starts.ptr),
                       G.tensor(G.I32, (seqs,), lengths.ptr))
    q = np.random.default_rng(4).standard_normal(d).astype(np.float32)
    qd = hip.to_dev(q)
    qt = G.tensor(G.F32, (d, heads, seqs), qd.ptr, [4, 0, 0, 0])
    out = torch.full((seqs, heads, d), float("nan"), dtype=torch.float16, device="cuda")
    assert G.attention_work_size(qt, *desc, batch) == 0
    print(f"attention heads={heads} sequences={seqs}", flush=True)
    G.attention(qt, *desc, batch, G.tensor(G.F16, (d, heads, seqs), out.data_ptr()), 0.125)
    torch.cuda.synchronize()
    assert hip.last_error() == 0
    k, v = (decode("q8_0", encode("q8_0", x)) for x in (k, v))
    p = np.exp(k @ q * 0.125)
    want = p @ v / p.sum()
    # roundings of values and the output, 2^-11 each of at most the largest value's
    assert np.abs(out[0, 0].double().cpu().numpy() - want).max() <= 2.0 ** -10 * np.abs(v).max()
    assert (out == out[0, 0]).all()
