"""log_probs against 64 bits (GPU).

With u = 2^-24, d = (x - max) scale, p = e^d / S, E|d| and E d^2 the means under p.  d is off by
2 u |d|, its exponential by 2 u |d| + 1.5 u |d| (the product with log2 e and its constant) and 4 u
(the instruction); S passes at most N = 32 values a chunk, the chunks of a lane and 16 more
additions.  So S is off by (3.5 E|d| + 4 + N) u of itself, its logarithm by that and 2 u of its
size, a log probability by that and 2 u |d|; sum e d by (3.5 E d^2 + (N + 8) E|d|) u of S.
Ids are compared for equality: the order is by (value, lowest id) and nothing is computed."""
from __future__ import annotations

import numpy as np
import pytest

from weft_amd import ggml as G

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
NP = {G.F32: np.float32, G.F16: np.float16}


def best(row, n):
    """The ids of the n largest numbers, of equal ones the lowest first; -1 where none is left."""
    ids = np.flatnonzero(~np.isnan(row))
    v = row[ids].astype(np.float64) + 0.0
    ids = ids[np.lexsort((ids, -v))][:n]
    return np.concatenate([ids, np.full(n - len(ids), -1, ids.dtype)])


def run(hip, x, given=None, top=0, entropy=True, scale=1.0, pad=0, offset=0):
    rows, v = x.shape
    t = G.F16 if x.dtype == np.float16 else G.F32
    buf = np.full((rows, v + pad), np.nan, x.dtype)
    buf[:, :v] = x
    e = x.itemsize
    xd = hip.to_dev(buf, offset * e)
    lt = G.tensor(t, (v, rows), xd.ptr, [e, e * (v + pad), 0, 0])
    tensors, dev = {}, {}

    def matrix(name, a, kind):
        wide = np.full((rows, a.shape[1] + (2 if pad else 0)), 77, a.dtype)
        wide[:, :a.shape[1]] = a
        dev[name] = (hip.to_dev(wide), a.shape, wide.shape)
        tensors[name] = G.tensor(kind, (a.shape[1], rows), dev[name][0].ptr, [4, 4 * wide.shape[1], 0, 0])

    if given is not None:
        matrix("tokens", given.astype(np.int32), G.I32)
        matrix("token_lp", np.full(given.shape, 5.0, np.float32), G.F32)
    if top:
        matrix("top_ids", np.full((rows, top), -7, np.int32), G.I32)
        matrix("top_lp", np.full((rows, top), 5.0, np.float32), G.F32)
    ed = hip.to_dev(np.full(rows, 5.0, np.float32))
    size = G.log_probs_work_size(lt, top)
    work = hip.empty(size, fill=0xff)
    print(f"log_probs rows={rows} v={v} type={t} given={None if given is None else given.shape[1]} top={top} scale={scale} "
          f"pad={pad} work={size}", flush=True)
    G.log_probs(lt, tensors.get("tokens"), tensors.get("token_lp"), G.tensor(G.F32, (rows,), ed.ptr) if entropy else None,
                tensors.get("top_ids"), tensors.get("top_lp"), scale, work.ptr, size)
    hip.torch.cuda.synchronize()
    assert hip.last_error() == 0
    out = {"entropy": ed.numpy(np.float32)}
    for name, (b, shape, wide) in dev.items():
        a = b.numpy(np.int32 if name in ("tokens", "top_ids") else np.float32, wide)
        assert (a[:, shape[1]:] == 77).all()
        out[name] = a[:, :shape[1]]
    return out


def check(hip, x, given=None, top=0, scale=1.0, **kw):
    out = run(hip, x, given, top, scale=scale, **kw)
    rows, v = x.shape
    n_add = 32 * 33 + 16  # no test's row has more chunks a lane
    with np.errstate(invalid="ignore", divide="ignore"):
        for r in range(rows):
            z = x[r].astype(np.float64)
            spoiled = np.isnan(z).any() or (z == np.inf).any()
            empty = not spoiled and (z == -np.inf).all()
            d = (z - z.max()) * np.float64(np.float32(scale))
            e = np.exp(d)
            s = e.sum()
            seen = e > 0
            d1, d2 = (e[seen] * -d[seen]).sum() / s, (e[seen] * d[seen] ** 2).sum() / s
            log_s = np.log(s)
            off_s = (3.5 * d1 + 4 + n_add) * U
            off_log = off_s + 2 * U * abs(log_s) + U

            def same(got, ids):
                lp = np.full(len(ids), np.nan) if spoiled else np.full(len(ids), -np.inf) if empty else d[ids] - log_s
                fine = np.isfinite(lp)
                assert np.array_equal(np.isnan(got), np.isnan(lp)) and np.array_equal(got == -np.inf, lp == -np.inf)
                assert (np.abs(got[fine] - lp[fine]) <= off_log + 3 * U * np.abs(d[ids][fine]) + U * np.abs(lp[fine])).all()

            if given is not None:
                there = (given[r] >= 0) & (given[r] < v)
                assert (out["token_lp"][r][~there] == 5.0).all()
                same(out["token_lp"][r][there].astype(np.float64), given[r][there])
            if kw.get("entropy", True):
                h = out["entropy"][r]
                if spoiled:
                    assert np.isnan(h)
                elif empty:
                    assert h == 0
                else:
                    want = log_s + d1
                    assert abs(h - want) <= off_log + (3.5 * d2 + (n_add + 8) * d1) * U + d1 * off_s + U * abs(want)
            if top:
                ids = best(x[r], top)
                assert np.array_equal(out["top_ids"][r], ids)
                lp = out["top_lp"][r].astype(np.float64)
                if spoiled:
                    assert np.isnan(lp).all()
                else:
                    same(lp, ids)
    return out


def logits(rows, v, t=G.F32, seed=0, spread=2.5):
    return (np.random.default_rng(seed + rows * 7 + v).standard_normal((rows, v)) * spread).astype(NP[t])


def asked(rows, v, n, seed=0):
    return np.random.default_rng(seed).integers(0, v, (rows, n)).astype(np.int32)


@pytest.mark.parametrize("t", [G.F32, G.F16])
@pytest.mark.parametrize("rows,v", [(1, 1), (3, 2), (2, 63), (5, 64), (2, 65), (4, 257), (300, 130), (2, 2047), (2, 2048),
                                    (3, 2049), (2, 8191), (2, 8193), (1, 50021), (3, 100003), (1030, 5000), (1100, 9001)])
def test_sizes(hip, rows, v, t):
    x = logits(rows, v, t)
    for top in sorted({0, 1, min(v, 20), min(v, 64)}):
        check(hip, x, asked(rows, v, 3), top)


@pytest.mark.parametrize("t", [G.F32, G.F16])
@pytest.mark.parametrize("v,offset", [(98770, 0), (8192 + 37, 1), (16384 + 300, 0), (466, 0), (1090, 3), (70, 1)])
def test_ends_of_few_values(hip, v, offset, t):
    """A last range, or last waves, of fewer values than alternatives, and of a few more; many equal."""
    x = logits(3, v, t)
    x[1] = np.round(x[1])
    x[2, -50:] += np.float32(20)  # the answer is there
    for top in (5, 33, 64):
        check(hip, x, asked(3, v, 1), top, offset=offset)


@pytest.mark.parametrize("top", [0, 5])
def test_parts_left_out(hip, top):
    x = logits(4, 3000)
    check(hip, x, None, top)
    check(hip, x, asked(4, 3000, 1), top, entropy=False)
    check(hip, x, asked(4, 3000, 130), top)


@pytest.mark.parametrize("t", [G.F32, G.F16])
@pytest.mark.parametrize("scale", [0.5, 1.25, 1e-3, 40.0])
def test_temperatures(hip, scale, t):
    check(hip, logits(3, 20011, t), asked(3, 20011, 2), 10, scale)


@pytest.mark.parametrize("scale", [1e-42, 1e-37, 3e37, 3.3e38])
@pytest.mark.parametrize("v", [5, 700, 40000])
def test_the_smallest_and_largest_scales(hip, v, scale):
    """Flat, and split among the largest alone; a difference times the scale stays finite."""
    x = (np.random.default_rng(v).integers(0, 5, (3, v)) / 4).astype(np.float32)
    check(hip, x, asked(3, v, 2), min(v, 9), scale)


@pytest.mark.parametrize("t", [G.F32, G.F16])
def test_strides_and_alignment(hip, t):
    for v, pad, offset in ((1000, 8, 0), (1001, 3, 1), (33000, 5, 3), (33001, 0, 1)):
        check(hip, logits(5, v, t), asked(5, v, 2), 7, pad=pad, offset=offset)


@pytest.mark.parametrize("v", [40, 3000, 40000])
@pytest.mark.parametrize("t", [G.F32, G.F16])
def test_orders_and_ties(hip, v, t):
    """Rows that are hard on the choice of the largest: sorted, equal, of two values, the largest all in one lane's
    places, zeros of both signs, few distinct values."""
    rng = np.random.default_rng(v)
    up = np.sort(logits(1, v, G.F32)[0])
    lane = np.full(v, -1.0)
    lane[np.arange(v) % 1024 < 4] = 5 + rng.random((np.arange(v) % 1024 < 4).sum())
    x = np.stack([up, up[::-1], np.zeros(v), np.where(rng.random(v) < 0.5, 0.0, -0.0), np.where(np.arange(v) % 7 == 3, 1, -1),
                  lane, np.round(logits(1, v)[0]), np.arange(v) % 64, np.full(v, -3.0e4), -np.arange(v) / 128]).astype(NP[t])
    for top in (1, 5, 40 if v == 40 else 64):
        check(hip, x, asked(len(x), v, 2), top)


@pytest.mark.parametrize("v", [40, 3000, 40000])
@pytest.mark.parametrize("t", [G.F32, G.F16])
def test_barred_and_spoiled(hip, v, t):
    low = np.finfo(NP[t]).min
    x = logits(12, v, t)
    x[0] = -np.inf
    x[1, : v - 3] = -np.inf
    x[2] = low
    x[3, 1:] = low
    x[4, v // 2] = np.nan
    x[5, v // 3] = np.inf
    x[6, ::2] = -np.inf
    x[7] = np.nan
    x[8, 2:] = np.nan
    x[9, : v // 2], x[9, v // 2:] = -np.inf, low
    x[10] = np.finfo(NP[t]).max
    x[11, :5], x[11, 5] = np.inf, np.nan
    given = asked(12, v, 3)
    given[:, 0], given[:, 2] = -1, v
    given[1, 1] = v - 1
    for top in (1, 20, 40):
        check(hip, x, given, top)


def test_a_row_of_one_peak_keeps_its_entropy(hip):
    """Logits far from zero whose differences are small, and a peak over a flat rest."""
    x = np.stack([logits(1, 9000)[0] + np.float32(30000), np.where(np.arange(9000) == 77, 40, 0)]).astype(np.float32)
    check(hip, x, asked(2, 9000, 1), 3)


def test_a_long_row(hip):
    check(hip, logits(1, 3000001), asked(1, 3000001, 5), 64)


def test_calls_agree_another_stream_and_a_graph(hip):
    torch = hip.torch
    rows, v, top = 3, 40000, 12
    xd, ids = hip.to_dev(logits(rows, v)), asked(rows, v, 2)
    td, ld, ed = hip.to_dev(ids), hip.empty(4 * ids.size), hip.empty(4 * rows)
    tid, tlp = hip.empty(4 * rows * top), hip.empty(4 * rows * top)
    lt = G.tensor(G.F32, (v, rows), xd.ptr)
    size = G.log_probs_work_size(lt, top)
    work = hip.empty(size, fill=0xff)
    assert size > 0
    args = [lt, G.tensor(G.I32, (2, rows), td.ptr), G.tensor(G.F32, (2, rows), ld.ptr), G.tensor(G.F32, (rows,), ed.ptr),
            G.tensor(G.I32, (top, rows), tid.ptr), G.tensor(G.F32, (top, rows), tlp.ptr), 1.0, work.ptr, size]
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=side):
            hip._lib.set_stream(side.cuda_stream)
            G.log_probs(*args)
    finally:
        hip._lib.set_stream(torch.cuda.current_stream().cuda_stream)
    for seed in range(3):
        x = logits(rows, v, seed=seed + 50)
        xd.t[:x.nbytes].copy_(torch.from_numpy(x.view(np.uint8).reshape(-1)))
        graph.replay()
        torch.cuda.synchronize()
        once = [b.numpy(np.uint32).copy() for b in (ld, ed, tid, tlp)]
        want = check(hip, x, ids, top)
        for a, name, dt in zip(once, ("token_lp", "entropy", "top_ids", "top_lp"), (np.float32, np.float32, np.int32, np.float32)):
            assert np.array_equal(a.view(dt).reshape(-1), want[name].reshape(-1))
