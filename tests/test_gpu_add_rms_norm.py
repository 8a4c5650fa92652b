"""add_rms_norm against 64 bits (GPU).

The 32-bit error of y: the square sum's terms pass at most 32 + K / 2048 additions
(a lane's own, then the trees over lanes and waves), each off by 2^-24, half of
which reaches the root; sum, product and division add under 8 more.  A record's
value is off by that and half a step (and a 16-bit step's own rounding, 2^-11);
its step is that of its largest value to the same relative error."""
from __future__ import annotations

import numpy as np
import pytest

from weft_amd import ggml as G

pytestmark = pytest.mark.gpu

OUT = {"f32": (G.F32, 1, 4), "f16": (G.F16, 1, 2), "q8_0": (G.Q8_0, 32, 34), "q8_1": (G.Q8_1, 32, 36),
       "q8_k": (G.Q8_K, 256, 292)}
EPS = 1e-5


def reference(x, r, w):
    s32 = x if r is None else x + r  # one rounding, as the operator's
    s = s32.astype(np.float64)
    y = s / np.sqrt((s * s).mean(-1, keepdims=True) + EPS)
    return s32, y if w is None else y * w.astype(np.float64)


def run(hip, rows, k, dst, residual=True, weight=True, total="own", pad=0, seed=0, data=None, offset=0):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((rows, k)) * 2).astype(np.float32) if data is None else data
    r = rng.standard_normal((rows, k)).astype(np.float32) if residual else None
    w = (1 + 0.2 * rng.standard_normal(k)).astype(np.float32) if weight else None
    t, block, size = OUT[dst]
    row = k // block * size

    def padded(a):
        b = np.full((rows, k + pad), 7.5, np.float32)
        b[:, :k] = a
        return hip.to_dev(b, offset)

    nb = [4, 4 * (k + pad), 0, 0]
    xd = padded(x)
    rd = padded(r) if residual else None
    wd = hip.to_dev(w, offset) if weight else None
    y_row = row + (4 if pad else 0)
    yd = hip.empty(rows * y_row, fill=0xA5)
    td = xd if total == "x" else hip.empty(4 * rows * (k + pad), fill=0x5A) if total == "own" else None
    print(f"add_rms_norm rows={rows} k={k} {dst} r={residual} w={weight} total={total} pad={pad} off={offset}", flush=True)
    G.add_rms_norm(G.tensor(G.F32, (k, rows), xd.ptr, nb), G.tensor(G.F32, (k, rows), rd.ptr, nb) if residual else None,
                   G.tensor(G.F32, (k,), wd.ptr) if weight else None,
                   G.tensor(G.F32, (k, rows), td.ptr, nb) if td is not None else None,
                   G.tensor(t, (k, rows), yd.ptr, [size, y_row, 0, 0]), EPS)
    hip.torch.cuda.synchronize()
    s, y = reference(x, r, w)
    if td is not None:
        got = td.numpy(np.float32, (rows, k + pad))
        assert np.array_equal(got[:, :k], s, equal_nan=True)
        if pad:
            assert (got[:, k:] == (7.5 if total == "x" else np.frombuffer(b"\x5a" * 4, np.float32)[0])).all()
    raw = yd.numpy(np.uint8, (rows, y_row))
    assert (raw[:, row:] == 0xA5).all()
    return np.ascontiguousarray(raw[:, :row]), y


def check(raw, y, dst, k):
    rows = y.shape[0]
    u = 2.0 ** -24 * (16 + k / 4096 + 8)
    if dst in ("f32", "f16"):
        got = raw.view(np.float32 if dst == "f32" else np.float16).astype(np.float64)
        assert (np.abs(got - y) <= np.abs(y) * (u + (2.0 ** -11 if dst == "f16" else 0)) + (2.0 ** -25 if dst == "f16" else 0)).all()
        return
    _, block, size = OUT[dst]
    rec = raw.reshape(rows, -1, size)
    b = y.reshape(rows, -1, block)
    top = np.abs(b).max(-1, keepdims=True)
    if dst == "q8_k":
        step = np.ascontiguousarray(rec[..., :4]).view(np.float32).astype(np.float64)
        q = np.ascontiguousarray(rec[..., 4:260]).view(np.int8).astype(np.float64)
        sums = np.ascontiguousarray(rec[..., 260:]).view(np.int16)
        assert np.array_equal(sums, q.reshape(rows, -1, 16, 16).sum(-1).astype(np.int16))
        ds = 2 * u
    else:
        step = np.ascontiguousarray(rec[..., :2]).view(np.float16).astype(np.float64)
        q = np.ascontiguousarray(rec[..., size - 32:]).view(np.int8).astype(np.float64)
        ds = 2 * u + 2.0 ** -11
        if dst == "q8_1":
            s = np.ascontiguousarray(rec[..., 2:4]).view(np.float16).astype(np.float64)
            want = q.sum(-1, keepdims=True) * top / 127
            assert (np.abs(s - want) <= np.abs(want) * (2.0 ** -11 + 2 * u) + 2.0 ** -25).all()
    assert (np.abs(np.abs(step) - top / 127) <= top / 127 * ds + 2.0 ** -25).all()
    assert (np.abs(q).max(-1) == np.where(top[..., 0] > 0, 127, 0)).all()
    assert (np.abs(step * q - b) <= top / 127 * (0.5 + 127 * (ds + u) + 1e-3) + 2.0 ** -24 * 127).all()


@pytest.mark.parametrize("dst,k", [(d, k) for d in OUT for k in (256, 512, 4096, 5120, 11008, 16384, 16640, 65536)])
def test_rows_of_every_length(hip, dst, k):
    for rows in (1, 3):
        raw, y = run(hip, rows, k, dst, seed=k + rows)
        check(raw, y, dst, k)


@pytest.mark.parametrize("dst,k", [("f32", k) for k in (1, 2, 3, 5, 63, 64, 65, 255, 1023, 4097, 16387)] +
                         [("f16", k) for k in (1, 3, 66, 257, 4099)] +
                         [("q8_0", k) for k in (32, 96, 224, 1056, 4128)] + [("q8_1", k) for k in (32, 160, 4064)])
def test_odd_lengths(hip, dst, k):
    raw, y = run(hip, 5, k, dst, seed=k)
    check(raw, y, dst, k)


@pytest.mark.parametrize("dst", list(OUT))
def test_many_rows_strides_and_alignment(hip, dst):
    for rows, k, pad, offset in ((1000, 768, 0, 0), (37, 1280, 4, 0), (37, 1280, 3, 4), (37, 1280, 0, 8)):
        raw, y = run(hip, rows, k, dst, pad=pad, offset=offset, seed=pad + rows)
        check(raw, y, dst, k)


@pytest.mark.parametrize("k", [512, 20480])
@pytest.mark.parametrize("residual,weight,total", [(False, True, "own"), (True, False, None), (False, False, None),
                                                   (True, True, "x"), (False, True, "x")])
def test_what_may_be_left_out_and_the_sum_over_x(hip, residual, weight, total, k):
    for dst in ("f32", "q8_0"):
        raw, y = run(hip, 4, k, dst, residual, weight, total, seed=3)
        check(raw, y, dst, k)


@pytest.mark.parametrize("dst", list(OUT))
def test_a_row_of_zeros_and_one_of_extremes(hip, dst):
    x = np.zeros((3, 512), np.float32)
    x[1, 7] = -3.0
    x[2] = np.float32(1e-30)
    raw, y = run(hip, 3, 512, dst, residual=False, weight=False, data=x)
    check(raw, y, dst, 512)


def test_infinity_and_nan_stay_in_their_row(hip):
    x = np.ones((3, 512), np.float32)
    x[0, 5], x[1, 6] = np.nan, np.inf
    raw, y = run(hip, 3, 512, "f32", residual=False, weight=False, data=x)
    got = raw.view(np.float32)
    assert np.isnan(got[0]).all() and np.isnan(got[1, 6]) and (np.delete(got[1], 6) == 0).all()
    check(raw[2:], y[2:], "f32", 512)


def test_two_calls_agree_and_another_stream(hip):
    torch = hip.torch
    a, _ = run(hip, 9, 4096, "q8_k", seed=5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    hip._lib.set_stream(side.cuda_stream)
    try:
        b, _ = run(hip, 9, 4096, "q8_k", seed=5)
    finally:
        hip._lib.set_stream(torch.cuda.current_stream().cuda_stream)
    assert np.array_equal(a, b)


def test_the_records_feed_mul_mat(hip):
    """MUL_MAT on the norm's Q8_K records equals MUL_MAT on its F32 row."""
    import oracle as o
    k, n, m = 1024, 96, 5
    raw, _ = run(hip, m, k, "q8_k", seed=8)
    f32, _ = run(hip, m, k, "f32", seed=8)
    w = hip.to_dev(o.quantize("q4_k", o.seeded_normal(1, (n, k), 0.02)))
    s0 = G.tensor(G.Q4_K, (k, n), w.ptr)
    outs = []
    for t, a in ((G.Q8_K, raw), (G.F32, f32.view(np.float32))):
        xd, yd = hip.to_dev(a), hip.empty(4 * n * m)
        s1, d = G.tensor(t, (k, m), xd.ptr), G.tensor(G.F32, (n, m), yd.ptr)
        size = G.mul_mat_work_size(s0, s1)
        work = hip.empty(max(size, 4))
        G.mul_mat(s0, s1, d, work.ptr, size)
        hip.torch.cuda.synchronize()
        outs.append(yd.numpy(np.float32))
    assert np.abs(outs[0] - outs[1]).max() <= 1e-4 * np.abs(outs[1]).max()
