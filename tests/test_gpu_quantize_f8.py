"""quantize_f8 against its formula (GPU).  Every step of it is a correctly rounded 32-bit
operation, so codes and scales are equal, bit for bit (NaN: any NaN code)."""
from __future__ import annotations

import numpy as np
import pytest

from tests._f8 import BLOCK, F8, F16, F32, VALUE, Rows, Scales, codes_of, quantize, up
from weft_amd import ggml as G

pytestmark = pytest.mark.gpu


def check(hip, x, blocks, t=F32, pad=0, y_pad=0, offset=0, y_offset=0, block_major=False):
    rows, k = x.shape
    print(f"quantize_f8 {rows}x{k} type={t} blocks={blocks} pad={pad},{y_pad} offset={offset},{y_offset}", flush=True)
    xd = Rows(hip, t, x, pad=pad, offset=offset)
    yd = Rows(hip, F8, shape=x.shape, pad=y_pad, offset=y_offset)
    sd = Scales(hip, shape=(up(rows) if blocks else rows, up(k)), block_major=block_major, pad=1)
    G.quantize_f8(xd.tensor, yd.tensor, sd.tensor)
    hip.torch.cuda.synchronize()
    assert hip.last_error() == 0
    codes, scales = quantize(x.astype(np.float32), BLOCK if blocks else 1)
    got = yd.numpy()
    nan = np.isnan(VALUE[codes])
    assert np.array_equal(sd.numpy(), scales)
    assert np.array_equal(got[~nan], codes[~nan]) and np.isnan(VALUE[got[nan]]).all()
    return got


def rows_of(rows, k, t=F32, seed=0):
    rng = np.random.default_rng(seed + 1000 * rows + k)
    x = rng.standard_normal((rows, k)) * np.exp(2 * rng.standard_normal(k))
    return np.clip(x, -6e4, 6e4).astype(np.float16 if t == F16 else np.float32)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("blocks", [False, True])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 128), (2, 7), (3, 127), (5, 129), (16, 256), (17, 1000), (127, 640),
                                    (128, 384), (129, 385), (300, 4101), (1, 70001)])
def test_sizes(hip, rows, k, blocks, t):
    check(hip, rows_of(rows, k, t), blocks, t)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("blocks", [False, True])
def test_strides_and_alignment(hip, blocks, t):
    x = rows_of(131, 523, t)
    e = 2 if t == F16 else 4
    for pad, y_pad, offset, y_offset, major in ((5, 0, 0, 0, True), (5, 3, e, 1, False), (0, 8, 3 * e, 7, True)):
        check(hip, x, blocks, t, pad, y_pad, offset, y_offset, major)


@pytest.mark.parametrize("rows,k,pad", [(1500, 1537, 0), (1300, 1664, 1), (2049, 2049, 0), (129, 17000, 8)])
def test_many_blocks_that_share_lines(hip, rows, k, pad):
    """More blocks than one turn of the launch's order, whole turns and a rest."""
    check(hip, rows_of(rows, k, F32), True, F32, y_pad=pad)


def test_every_code_and_every_tie(hip):
    """Factor 1: the codes' values, the points halfway between them and their neighbours."""
    v = VALUE[:127]
    mid = (v[1:] + v[:-1]) / 2
    near = np.concatenate([v, mid, np.nextafter(mid.astype(np.float32), np.float32(0)),
                           np.nextafter(mid.astype(np.float32), np.float32(500))]).astype(np.float32)
    near = np.concatenate([near, -near])
    x = np.zeros((up(len(near)) + 7, BLOCK), np.float32)
    x[:, 0] = 448
    flat = np.resize(near, (x.shape[0], BLOCK - 1))
    x[:, 1:] = flat
    assert len(np.unique(codes_of(x))) == 254  # every number
    check(hip, x, False)


@pytest.mark.parametrize("blocks", [False, True])
def test_extremes(hip, blocks):
    x = np.zeros((5, 300), np.float32)
    x[1] = np.float32(1e-38) * np.arange(300)
    x[2] = np.float32(3.4e38)
    x[2, 5:200:3] = -1
    x[3, ::2] = np.float32(2.0 ** -100)
    x[3, 1::2] = np.float32(-2.0 ** -149)
    x[4] = -0.0
    check(hip, x, blocks)
    # what is not finite becomes NaN in its place and leaves the others' scale alone
    y = rows_of(5, 300)
    y[0, 7], y[1, 130], y[3, 299], y[4, :] = np.nan, np.inf, -np.inf, np.inf
    check(hip, y, blocks)


def test_another_stream_and_a_graph(hip):
    torch = hip.torch
    x = rows_of(40, 1030)
    xd, yd, sd = Rows(hip, F32, x), Rows(hip, F8, shape=x.shape), Scales(hip, shape=(40, up(1030)))
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=side):
            hip._lib.set_stream(side.cuda_stream)
            G.quantize_f8(xd.tensor, yd.tensor, sd.tensor)
    finally:
        hip._lib.set_stream(torch.cuda.current_stream().cuda_stream)
    for seed in range(3):
        x = rows_of(40, 1030, seed=seed)
        xd.dev.t[:x.nbytes].copy_(torch.from_numpy(x.view(np.uint8).reshape(-1)))
        graph.replay()
        torch.cuda.synchronize()
        codes, scales = quantize(x, 1)
        assert np.array_equal(yd.numpy(), codes) and np.array_equal(sd.numpy(), scales)
