"""Plain 64-bit forms of the operators between a decoder layer's products, and
the device buffers their tests share: a paged cache built from rows of values
(the oracle's records), in either page layout, with every byte that holds no row
poisoned (NaN in 16 bits, NaN scales and random codes in the quantized types)."""
from __future__ import annotations

import numpy as np

import oracle as o
from weft_amd import ggml as G

KV_TYPE = {"f16": G.F16, "q8_0": G.Q8_0, "q4_0": G.Q4_0}
RECORD = {"f16": 64, "q8_0": 34, "q4_0": 18}
EPS16 = 2.0 ** -11  # unit roundoff of 16-bit values


def row_bytes(kind, d):
    return RECORD[kind] * (d // 32)


def encode(kind, x):
    """Rows (..., d) of float32 as cache bytes (..., row_bytes)."""
    d = x.shape[-1]
    if kind == "f16":
        return x.astype(np.float16).view(np.uint8)
    return o.quantize(kind, np.ascontiguousarray(x.reshape(-1, d))).reshape(*x.shape[:-1], row_bytes(kind, d))


def decode(kind, b):
    """Their values in float64."""
    if kind == "f16":
        return np.ascontiguousarray(b).view(np.float16).astype(np.float64)
    r = b.reshape(*b.shape[:-1], b.shape[-1] // RECORD[kind], RECORD[kind])
    step = np.ascontiguousarray(r[..., :2]).view(np.float16).astype(np.float64)
    if kind == "q8_0":
        q = np.ascontiguousarray(r[..., 2:]).view(np.int8).astype(np.float64)
    else:
        q = np.concatenate([r[..., 2:] & 15, r[..., 2:] >> 4], -1).astype(np.float64) - 8
    return (step * q).reshape(*b.shape[:-1], b.shape[-1] // RECORD[kind] * 32)


class Cache:
    """Sequences of ``lengths`` tokens in pages taken in random order."""

    def __init__(self, hip, kind, lengths, news, page, kv_heads, d, seed, slots_first=False, spread=1.0, fill=True):
        rng = np.random.default_rng(seed)
        self.hip, self.kind, self.page, self.kv_heads, self.d = hip, kind, page, kv_heads, d
        self.lengths, self.news, self.slots_first = list(lengths), list(news), slots_first
        n = len(self.lengths)
        used = [-(-max(0, x) // page) for x in self.lengths]
        self.n_pages = sum(used) + 2
        order = rng.permutation(self.n_pages)
        self.table = np.full((n, max([1, *used])), -1, np.int32)
        at = 0
        for i, u in enumerate(used):
            self.table[i, :u] = order[at:at + u]
            at += u
        self.starts = np.concatenate([[0], np.cumsum(self.news)]).astype(np.int32)
        self.rows = {}   # name -> per sequence (length, kv_heads, bytes)
        self.host = {}
        for name in ("k", "v"):
            pool = rng.integers(0, 256, (self.n_pages, kv_heads, page, row_bytes(kind, d)), dtype=np.uint8)
            if kind == "f16":
                pool[..., 1::2] = 0x7e
            else:
                rec = pool.reshape(self.n_pages, kv_heads, page, -1, RECORD[kind])
                rec[..., 0], rec[..., 1] = 0x01, 0x7e
            self.rows[name] = []
            for i, length in enumerate(self.lengths):
                length = max(0, length)
                x = rng.standard_normal((length, kv_heads, d)).astype(np.float32)
                if name == "k":
                    x *= np.float32(spread)
                rows = encode(kind, x) if length else np.zeros((0, kv_heads, row_bytes(kind, d)), np.uint8)
                self.rows[name].append(rows)
                if fill:
                    for p in range(length):
                        pool[self.table[i, p // page], :, p % page] = rows[p]
            self.host[name] = pool
        self.upload()

    def upload(self):
        hip, e = self.hip, {"f16": 2}.get(self.kind, RECORD[self.kind])
        self.dev, self.pools = {}, {}
        rb = row_bytes(self.kind, self.d)
        for name in ("k", "v"):
            pool = self.host[name]
            if self.slots_first:  # (pages, slots, heads, row)
                pool = np.ascontiguousarray(pool.swapaxes(1, 2))
                nb = [e, rb * self.kv_heads, rb, rb * self.kv_heads * self.page]
            else:
                nb = [e, rb, rb * self.page, rb * self.kv_heads * self.page]
            self.dev[name] = hip.to_dev(pool)
            self.pools[name] = G.tensor(KV_TYPE[self.kind], (self.d, self.page, self.kv_heads, self.n_pages),
                                        self.dev[name].ptr, nb)
        self.dev["table"] = hip.to_dev(self.table)
        self.dev["starts"] = hip.to_dev(self.starts)
        self.dev["lengths"] = hip.to_dev(np.array(self.lengths, np.int32))
        n = len(self.lengths)
        self.batch = G.kv_batch(G.tensor(G.I32, (self.table.shape[1], n), self.dev["table"].ptr),
                                G.tensor(G.I32, (n + 1,), self.dev["starts"].ptr),
                                G.tensor(G.I32, (n,), self.dev["lengths"].ptr))

    def pool(self, name):
        """The device pool as it is now, (pages, heads, slots, row)."""
        shape = self.host[name].shape
        if self.slots_first:
            shape = (shape[0], shape[2], shape[1], shape[3])
            return self.dev[name].numpy(np.uint8, shape).swapaxes(1, 2)
        return self.dev[name].numpy(np.uint8, shape)

    def values(self, name, i):
        return decode(self.kind, self.rows[name][i])


def attend(cache, q, scale, window=0, sinks=0):
    """float64 attention of q (tokens, heads, d); also, per output, the sum of
    p |v| and the largest scale sum |q k| that its error bound needs."""
    tokens, heads, d = q.shape
    share = heads // cache.kv_heads
    out, mass, reach = np.zeros((3, tokens, heads, d))
    for i, (length, n) in enumerate(zip(cache.lengths, cache.news)):
        k, v = cache.values("k", i), cache.values("v", i)
        there = np.repeat(cache.table[i], cache.page)[:max(0, length)] >= 0
        for t in range(n):
            pos = length - n + t
            j = np.arange(len(k))
            seen = there & (j <= pos)
            if window:
                seen &= (j > pos - window) | (j < sinks)
            if not seen.any():
                continue
            row = cache.starts[i] + t
            for h in range(heads):
                kk, vv, x = k[seen, h // share], v[seen, h // share], q[row, h].astype(np.float64)
                s = kk @ x * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                out[row, h] = p @ vv
                mass[row, h] = p @ np.abs(vv)
                reach[row, h] = scale * (np.abs(kk) @ np.abs(x)).max()
    return out, mass, reach


def attention_bound(mass, reach, out, half_out):
    """What rounding q, k, v and p once each to 16 bits (unit roundoff u = 2^-11)
    can do, with everything else in 32 bits: a score moves by at most
    delta = 2.1 u reach, a weight by exp(2 delta) - 1 and its own u, a value by u."""
    u = EPS16
    delta = 2.1 * u * reach
    return mass * (np.exp(2 * delta) - 1 + 2.1 * u) + (u * np.abs(out) if half_out else 0) + 1e-6
