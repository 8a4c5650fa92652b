"""8-bit floats with block scales as numpy has them, and the buffers the tests of their
quantizer and products share: rows apart by any bytes, with NaN codes and NaN scales in
every byte that holds no value."""
from __future__ import annotations

import numpy as np

from weft_amd import ggml as G

BLOCK = 128
F32, F16, F8 = G.F32, G.F16, G.F8_E4M3
NP = {F32: np.float32, F16: np.float16, F8: np.uint8}
SIZE = {F32: 4, F16: 2, F8: 1}


def up(n):
    return -(-n // BLOCK)


def _table():
    """The value of every code, from its fields."""
    c = np.arange(256)
    e, f = c >> 3 & 15, c & 7
    v = np.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e - 10.0))
    v = np.where(c & 0x80, -v, v)
    v[[0x7f, 0xff]] = np.nan
    return v


VALUE = _table()


def codes_of(v):
    """Codes of the e4m3 numbers nearest v (float32, at most 448 in magnitude after rounding), ties to even."""
    v = v.astype(np.float64)
    bad = ~np.isfinite(v)
    a = np.abs(np.where(bad, 0, v))
    step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(a, 2.0 ** -20))), -6) - 3)
    q = np.round(a / step) * step  # half to even
    code = np.searchsorted(VALUE[:127], q).astype(np.uint8)
    assert (VALUE[code] == q).all()
    return np.where(bad, 0x7f, code | np.where(np.signbit(v), 0x80, 0)).astype(np.uint8)


def quantize(x, rows):
    """(codes, scales (bands of rows, blocks)) of float32 x (r, k) by the formula in 32 bits."""
    r, k = x.shape
    wide = np.zeros((-(-r // rows) * rows, up(k) * BLOCK), np.float32)
    wide[:r, :k] = x
    b = wide.reshape(-1, rows, up(k), BLOCK)
    a = np.abs(np.where(np.isfinite(b), b, 0)).max((1, 3))
    a = np.maximum(a, np.float32(2.0 ** -100))
    with np.errstate(invalid="ignore"):
        y = b * (np.float32(448) / a)[:, None, :, None]
    codes = codes_of(np.where(np.isfinite(b), y, np.nan)).reshape(wide.shape)[:r, :k]
    return codes, a / np.float32(448)


def values(codes, scales, rows):
    """Their values in float64."""
    r, k = codes.shape
    s = np.repeat(np.repeat(scales.astype(np.float64), rows, 0)[:r], BLOCK, 1)[:, :k]
    return VALUE[codes] * s


class Rows:
    """A matrix on the device with `pad` elements of poison behind each row, its base `offset` bytes past an aligned one."""

    def __init__(self, hip, t, a=None, shape=None, pad=0, offset=0):
        rows, k = a.shape if a is not None else shape
        self.t, self.rows, self.k, self.pad = t, rows, k, pad
        host = np.full((rows, k + pad), 0x7f if t == F8 else 7.0, NP[t])
        if t != F8:
            host[:] = np.nan
        if a is not None:
            host[:, :k] = a
        self.dev = hip.to_dev(host, offset)
        self.tensor = G.tensor(t, (k, rows), self.dev.ptr, [SIZE[t], SIZE[t] * (k + pad), 0, 0])

    def numpy(self):
        """The matrix as it is now; the bytes behind its rows are the poison they were."""
        a = self.dev.numpy(NP[self.t], (self.rows, self.k + self.pad))
        rest = a[:, self.k:]
        assert (rest == 0x7f).all() if self.t == F8 else np.isnan(rest).all()
        return a[:, :self.k]


class Scales:
    """Scales (rows, blocks) on the device, block-major or row-major."""

    def __init__(self, hip, a=None, shape=None, block_major=False, pad=0):
        rows, blocks = a.shape if a is not None else shape
        self.rows, self.blocks, self.block_major, self.pad = rows, blocks, block_major, pad
        host = np.full((blocks, rows + pad) if block_major else (rows, blocks + pad), np.nan, np.float32)
        if a is not None:
            host[:, :a.T.shape[1] if block_major else blocks] = a.T if block_major else a
        self.shape = host.shape
        self.dev = hip.to_dev(host)
        nb = [4 * (rows + pad), 4] if block_major else [4, 4 * (blocks + pad)]
        self.tensor = G.tensor(F32, (blocks, rows), self.dev.ptr, [*nb, 0, 0])

    def numpy(self):
        a = self.dev.numpy(np.float32, self.shape)
        if self.block_major:
            assert np.isnan(a[:, self.rows:]).all()
            return np.ascontiguousarray(a[:, :self.rows].T)
        assert np.isnan(a[:, self.blocks:]).all()
        return a[:, :self.blocks]
