"""head_norm_rope against 64 bits and longer (GPU).

With u = 2^-24.  The norm: at most 8 + 6 additions of the squares (half of it reaches the
root) and five more operations: 12 u.  An angle's remainder of a turn is rounded to 32 bits
(pi u at most), its turns are computed in 64 bits of which eight operations and an exponent of
up to 2^5 leave 2^-46 of the whole angle; sine and cosine are within 4 u, their product with
the magnitude and the two products and the sum within 4 u more.  So a turned value is off by
(|a| + |b|) g (24 u + 2^-46 t), others by 12 u of their size; 16-bit outputs add 2^-11 of theirs."""
from __future__ import annotations

import numpy as np
import pytest

from weft_amd import ggml as G

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-6
NP = {G.F32: np.float32, G.F16: np.float16}


def reference(x, w, p, n, neighbours, base, scale, g, factors, normed):
    """(y, bound) in long doubles; x (tokens, heads, d)."""
    x = x.astype(np.longdouble)
    if normed:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)
        if w is not None:
            x = x * w
    y, off = x.copy(), np.abs(x) * 12 * U
    i = np.arange(n // 2)
    t = p.astype(np.longdouble)[:, None] * scale * np.longdouble(base) ** (-2 * i / np.longdouble(max(n, 1)))
    if factors is not None:
        t = t / factors
    two_pi = 2 * np.longdouble("3.14159265358979323846264338327950288")
    turns = t / two_pi
    r = (turns - np.round(turns)) * two_pi
    c, s, t = np.cos(r)[:, None], np.sin(r)[:, None], np.abs(t)[:, None]
    a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + n // 2)
    u, v = x[..., a], x[..., b]
    y[..., a], y[..., b] = g * (u * c - v * s), g * (u * s + v * c)
    off[..., a] = off[..., b] = (np.abs(u) + np.abs(v)) * g * (24 * U + 2.0 ** -46 * t)
    return y, off


def run(hip, tokens=3, heads=4, kv_heads=2, d=128, n=None, neighbours=False, src=G.F32, dst=G.F32, base=10000.0, scale=1.0,
        g=1.0, factors=False, normed=True, weights=True, pos=None, strided=False, in_place=False, seed=0, offset=0,
        x=None):
    n = d if n is None else n
    rng = np.random.default_rng(seed + 17 * tokens + d + n)
    pos = np.arange(tokens) + 5 if pos is None else pos
    pos = np.resize(np.array(pos, np.int32), tokens)
    f = (1 + 7 * rng.random(n // 2)).astype(np.float32) if factors else None
    host, dev, out, t_in, t_out, w, wd = [{} for _ in range(7)]
    names = [("q", heads)] + ([("k", kv_heads)] if kv_heads else [])
    for name, h in names:
        a = (3 * rng.standard_normal((tokens, h, d))).astype(NP[src]) if x is None else np.resize(x, (tokens, h, d)).astype(NP[src])
        host[name] = a
        # strided: a token's heads lie in a wider row (as a joined product of q, k and v has them), values behind are poison
        gap = 3 if strided else 0
        buf = np.full((tokens, h + gap, d + gap), np.nan, NP[src])
        buf[:, :h, :d] = a
        e, eo = buf.itemsize, np.dtype(NP[dst]).itemsize
        dev[name] = hip.to_dev(buf, offset * e)
        t_in[name] = G.tensor(src, (d, h, tokens), dev[name].ptr, [e, e * (d + gap), e * (d + gap) * (h + gap), 0])
        if in_place:
            out[name], t_out[name] = dev[name], t_in[name]
        else:
            out[name] = hip.to_dev(np.full((tokens, h + gap, d + gap), np.nan, NP[dst]), offset * eo)
            t_out[name] = G.tensor(dst, (d, h, tokens), out[name].ptr, [eo, eo * (d + gap), eo * (d + gap) * (h + gap), 0])
        w[name] = (1 + 0.2 * rng.standard_normal(d)).astype(np.float32) if weights and normed else None
        wd[name] = hip.to_dev(w[name]) if w[name] is not None else None
    pd, fd = hip.to_dev(pos), hip.to_dev(f) if f is not None else None
    print(f"head_norm_rope tokens={tokens} heads={heads},{kv_heads} d={d} n={n} neighbours={neighbours} {src}->{dst} "
          f"strided={strided} in_place={in_place} normed={normed}", flush=True)

    def vec(v, m):
        return None if v is None else G.tensor(G.F32, (m,), v.ptr)

    G.head_norm_rope(t_in["q"], t_in.get("k"), t_out["q"], t_out.get("k"),
                     G.tensor(G.I32, (tokens,), pd.ptr) if n else None, G.head_rope(n, neighbours, base, scale, g),
                     EPS if normed else None, vec(wd["q"], d), vec(wd.get("k"), d), vec(fd, n // 2))
    hip.torch.cuda.synchronize()
    assert hip.last_error() == 0
    got = {}
    for name, h in names:
        gap = 3 if strided else 0
        buf = out[name].numpy(NP[dst], (tokens, h + gap, d + gap))
        assert np.isnan(buf[:, h:]).all() and np.isnan(buf[:, :, d:]).all()
        got[name] = buf[:, :h, :d]
        y, off = reference(host[name], w[name], pos, n, neighbours, base, scale, g, f, normed)
        if dst == G.F16:
            off = off + np.abs(y) * 2.0 ** -11 + 2.0 ** -25
        bad = ~np.isfinite(y)
        assert np.array_equal(np.isnan(got[name]), np.isnan(y.astype(np.float64)))
        assert (np.abs(got[name].astype(np.longdouble) - y)[~bad] <= off[~bad] + 1e-37).all(), name
    return got


TYPES = [(s, o) for s in (G.F32, G.F16) for o in (G.F32, G.F16)]


@pytest.mark.parametrize("src,dst", TYPES)
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("d,n", [(128, 128), (64, 64), (96, 96), (80, 80), (256, 256), (192, 128), (128, 32), (96, 64), (64, 0),
                                 (1, 0), (2, 2), (3, 2), (7, 6), (63, 34), (130, 126), (255, 250), (256, 2), (36, 36)])
def test_head_sizes(hip, d, n, neighbours, src, dst):
    run(hip, 3, 5, 2, d, n, neighbours, src, dst)


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 32, 8), (1, 1, 0), (2, 1, 1), (48, 16, 16), (700, 7, 1), (5000, 3, 2),
                                                   (3, 200, 40)])
def test_tokens_and_heads(hip, tokens, heads, kv_heads, neighbours):
    run(hip, tokens, heads, kv_heads, 64, 64, neighbours)


@pytest.mark.parametrize("src,dst", TYPES)
def test_strides_and_alignment(hip, src, dst):
    for d, n, neighbours in ((128, 128, False), (96, 64, True), (80, 48, False)):
        run(hip, 9, 6, 3, d, n, neighbours, src, dst, strided=True)
        run(hip, 9, 6, 3, d, n, neighbours, src, dst, strided=True, offset=1)


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("t", [G.F32, G.F16])
def test_in_place(hip, t, neighbours):
    run(hip, 40, 9, 3, 128, 128, neighbours, t, t, in_place=True)
    run(hip, 7, 9, 3, 96, 64, neighbours, t, t, in_place=True, strided=True)


def test_far_positions(hip):
    for base, scale in ((10000.0, 1.0), (500000.0, 0.25), (1e6, 1.0), (0.5, 1.0)):
        run(hip, 8, 4, 2, 128, 128, base=base, scale=scale, factors=True,
            pos=[0, 1, 131071, 1000003, (1 << 24) + 1, (1 << 31) - 1, -1, -(1 << 31)] if base >= 1 else [0, 1, 50])


def test_magnitude_scale_and_factors(hip):
    for neighbours in (False, True):
        run(hip, 6, 4, 2, 128, 96, neighbours, scale=0.125, g=1.25, factors=True, pos=[4000, 70000, 3])


@pytest.mark.parametrize("kw", [{"normed": False}, {"weights": False}, {"normed": False, "n": 0}, {"n": 0}])
def test_parts_left_out(hip, kw):
    run(hip, 5, 4, 2, 128, **{"n": 64, **kw})


def test_zero_rows_and_extremes(hip):
    x = np.zeros((2, 4, 128), np.float32)
    x[1, 0] = 1e-30
    x[1, 1, 5] = 1e18
    run(hip, 2, 4, 4, 128, x=x)


def test_nan_stays_in_its_head(hip):
    x = np.random.default_rng(0).standard_normal((2, 4, 128)).astype(np.float32)
    x[0, 1, 100] = np.nan
    got = run(hip, 2, 4, 0, 128, x=x)["q"]
    assert np.isnan(got[0, 1]).all() and np.isnan(got).sum() == 128


def test_a_graph_follows_its_positions(hip):
    torch = hip.torch
    d, tokens = 64, 4
    x = np.random.default_rng(1).standard_normal((tokens, 3, d)).astype(np.float32)
    xd, yd, pd = hip.to_dev(x), hip.empty(x.nbytes), hip.to_dev(np.zeros(tokens, np.int32))
    q, y = (G.tensor(G.F32, (d, 3, tokens), b.ptr) for b in (xd, yd))
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=side):
            hip._lib.set_stream(side.cuda_stream)
            G.head_norm_rope(q, None, y, None, G.tensor(G.I32, (tokens,), pd.ptr), G.head_rope(d), EPS)
    finally:
        hip._lib.set_stream(torch.cuda.current_stream().cuda_stream)
    for first in (0, 7, 100000):
        pos = np.arange(first, first + tokens, dtype=np.int32)
        pd.t[:16].copy_(torch.from_numpy(pos.view(np.uint8)))
        graph.replay()
        torch.cuda.synchronize()
        want, off = reference(x, None, pos, d, False, 10000.0, 1.0, 1.0, None, True)
        assert (np.abs(yd.numpy(np.float32, x.shape) - want) <= off).all()
