"""What the norm, cache and attention entry points refuse, before anything is
launched (no GPU): the code raised, and that nothing stays recorded."""
from __future__ import annotations

import pytest

from weft_amd import _lib, ggml as G

INVALID, NOT_SUPPORTED = 1, 801
A = [(i + 1) << 20 for i in range(12)]  # stand-ins for device addresses


def refused(fn, *args):
    with pytest.raises(_lib.HipError) as e:
        fn(*args)
    assert _lib.load().weft_hip_get_last_error() == 0
    return e.value.code


# ------------------------------------------------------------------- the norm
def norm_args(k=512, rows=4, t=G.Q8_0):
    x, r, s = (G.tensor(G.F32, (k, rows), A[i]) for i in range(3))
    return [x, r, G.tensor(G.F32, (k,), A[3]), s, G.tensor(t, (k, rows), A[4]), 1e-5]


def norm_with(i, tensor, **kw):
    a = norm_args(**kw)
    a[i] = tensor
    return a


def test_norm_shapes_strides_and_addresses():
    for i in (0, 1, 3):
        assert refused(G.add_rms_norm, *norm_with(i, G.tensor(G.F32, (480, 4), A[0]))) == INVALID
        assert refused(G.add_rms_norm, *norm_with(i, G.tensor(G.F32, (512, 5), A[0]))) == INVALID
        assert refused(G.add_rms_norm, *norm_with(i, G.tensor(G.F32, (512, 4, 2), A[0]))) == INVALID
        assert refused(G.add_rms_norm, *norm_with(i, G.tensor(G.F32, (512, 4), A[0] + 2))) == INVALID
        assert refused(G.add_rms_norm, *norm_with(i, G.tensor(G.F32, (512, 4), 0))) == INVALID
        assert refused(G.add_rms_norm, *norm_with(i, G.tensor(G.F32, (512, 4), A[0], [8, 4096, 0, 0]))) == INVALID
        assert refused(G.add_rms_norm, *norm_with(i, G.tensor(G.F32, (512, 4), A[0], [4, 2050, 0, 0]))) == INVALID
    assert refused(G.add_rms_norm, *norm_with(2, G.tensor(G.F32, (511,), A[3]))) == INVALID
    for t in (G.Q8_0, G.Q8_K, G.F32, G.F16):
        assert refused(G.add_rms_norm, *norm_with(4, G.tensor(t, (512, 4), 0), t=t)) == INVALID
        assert refused(G.add_rms_norm, *norm_with(4, G.tensor(t, (512, 3), A[4]), t=t)) == INVALID
        assert refused(G.add_rms_norm, *norm_with(4, G.tensor(t, (512, 4), A[4] + 1), t=t)) == INVALID
    assert refused(G.add_rms_norm, None, *norm_args()[1:]) == INVALID
    assert refused(G.add_rms_norm, *norm_with(4, None)) == INVALID


def test_norm_types_rows_and_eps():
    for i in (0, 1, 2, 3):
        assert refused(G.add_rms_norm, *norm_with(i, G.tensor(G.F16, (512, 4), A[0]))) == NOT_SUPPORTED
    assert refused(G.add_rms_norm, *norm_with(4, G.tensor(G.Q4_0, (512, 4), A[4]))) == NOT_SUPPORTED
    assert refused(G.add_rms_norm, *norm_args(k=288, t=G.Q8_K)) == INVALID  # no whole records
    assert refused(G.add_rms_norm, *norm_args(k=48, t=G.Q8_0)) == INVALID
    for eps in (-1e-6, float("nan")):
        assert refused(G.add_rms_norm, *norm_args()[:5], eps) == INVALID


def test_empty_norm_launches_nothing():
    G.add_rms_norm(*norm_args(rows=0))
    assert _lib.load().weft_hip_get_last_error() == 0


# ------------------------------------------------------ the cache, the attention
def batch(n=2, width=3, **kw):
    t = {"pages": G.tensor(G.I32, (width, n), A[5]), "starts": G.tensor(G.I32, (n + 1,), A[6]),
         "lengths": G.tensor(G.I32, (n,), A[7]), **kw}
    return G.kv_batch(t["pages"], t["starts"], t["lengths"])


def pool(t=G.Q8_0, d=64, page=16, heads=2, pages=8, at=8, nb=None):
    return G.tensor(t, (d, page, heads, pages), A[at], nb)


def rows(t=G.F32, d=64, heads=2, tokens=5, at=0, outer=1):
    return G.tensor(t, (d, heads, tokens, outer), A[at])


def every_call():
    """(call with a batch and a pair of pools) of the three operators over a cache."""
    def write(b, k, v):
        G.kv_write(rows(), rows(at=1), b, k, v)

    def read(b, k, v):
        G.kv_read(k, v, b, rows(outer=2), rows(at=1, outer=2))

    def attend(b, k, v):
        G.attention(rows(heads=4), k, v, b, rows(heads=4, at=1), 0.1, 0, 0, A[10], 1 << 30)

    return [write, read, attend]


@pytest.mark.parametrize("which", range(3))
def test_pools(which):
    call = every_call()[which]
    ok = pool()
    assert refused(call, batch(), None, ok) == INVALID
    assert refused(call, batch(), ok, None) == INVALID
    assert refused(call, batch(), ok, pool(t=G.Q4_0)) == NOT_SUPPORTED
    for t in (G.F32, G.Q8_1, G.Q4_K):
        bad = G.tensor(t, (256, 16, 2, 8), A[8])
        assert refused(call, batch(), bad, bad) == NOT_SUPPORTED
    for kw in ({"d": 96}, {"page": 32}, {"heads": 4}, {"pages": 9}):
        assert refused(call, batch(), ok, pool(**kw)) == INVALID
    for bad in (pool(at=0, nb=[34, 69, 2176, 4352]), pool(nb=[36, 72, 2176, 4352]), pool(nb=[34, 68, 2177, 4352]),
                G.tensor(G.Q8_0, (64, 16, 2, 8), A[8] + 1), G.tensor(G.Q8_0, (64, 16, 2, 8), 0),
                G.tensor(G.F16, (48, 16, 2, 8), A[8]), G.tensor(G.Q8_0, (64, 0, 2, 8), A[8])):
        assert refused(call, batch(), bad, bad) == INVALID


@pytest.mark.parametrize("which", range(3))
def test_batches(which):
    call = every_call()[which]
    k = pool()
    assert refused(call, None, k, k) == INVALID
    for kw in ({"starts": G.tensor(G.I32, (2,), A[6])}, {"pages": G.tensor(G.I32, (3, 3), A[5])},
               {"lengths": G.tensor(G.I32, (3,), A[7])}, {"pages": G.tensor(G.F32, (3, 2), A[5])},
               {"lengths": G.tensor(G.F32, (2,), A[7])}, {"starts": G.tensor(G.I32, (3,), A[6] + 2)},
               {"pages": G.tensor(G.I32, (3, 2), A[5], [4, 14, 28, 28])},
               {"pages": G.tensor(G.I32, (3, 2), A[5], [8, 24, 48, 48])}, {"starts": G.tensor(G.I32, (3,), 0)}):
        assert refused(call, batch(**kw), k, k) == INVALID


def test_rows_of_the_cache():
    k = pool()
    for bad in (rows(d=96), rows(heads=3), rows(outer=2), G.tensor(G.F32, (64, 2, 5), A[0] + 1),
                G.tensor(G.F32, (64, 2, 5), A[0], [4, 258, 512, 0]), G.tensor(G.F32, (64, 2, 5), 0)):
        assert refused(G.kv_write, bad, bad, batch(), k, k) == INVALID
    assert refused(G.kv_write, rows(tokens=4), rows(tokens=5), batch(), k, k) == INVALID
    assert refused(G.kv_write, rows(), rows(t=G.F16), batch(), k, k) == NOT_SUPPORTED
    assert refused(G.kv_write, rows(t=G.Q8_0), rows(t=G.Q8_0), batch(), k, k) == NOT_SUPPORTED
    assert refused(G.kv_read, k, k, batch(), rows(outer=1), rows(outer=1)) == INVALID  # a batch of two
    assert refused(G.kv_read, k, k, batch(), rows(outer=2), rows(outer=2, tokens=6)) == INVALID
    assert refused(G.kv_read, k, k, batch(), rows(outer=2), rows(outer=2, t=G.F16)) == NOT_SUPPORTED


def test_queries_and_outputs():
    k = pool()

    def call(q, o, scale=0.1, window=0, sinks=0, work=A[10], size=1 << 40, k=k):
        return refused(G.attention, q, k, k, batch(), o, scale, window, sinks, work, size)

    q, o = rows(heads=4), rows(heads=4, at=1)
    for bad in (rows(heads=3), rows(heads=0), rows(heads=4, d=96), rows(heads=4, outer=2),
                G.tensor(G.F32, (64, 4, 5), A[0] + 2), G.tensor(G.F32, (64, 4, 5), 0)):
        assert call(bad, o) == INVALID
    for bad in (rows(heads=2), rows(heads=4, tokens=4), G.tensor(G.F32, (64, 4, 5), A[1], [4, 256, 1026, 0]),
                G.tensor(G.F32, (64, 4, 5), 0)):
        assert call(q, bad) == INVALID
    assert call(rows(heads=4, t=G.Q8_0), o) == NOT_SUPPORTED
    assert call(q, rows(heads=4, t=G.Q8_0)) == NOT_SUPPORTED
    assert call(q, o, window=-1) == INVALID
    assert call(q, o, sinks=-1) == INVALID
    for s in (float("inf"), float("nan")):
        assert call(q, o, scale=s) == INVALID
    odd = pool(d=32)
    assert call(rows(heads=4, d=32), rows(heads=4, d=32, at=1), k=odd) == NOT_SUPPORTED


def test_empty_calls_launch_nothing():
    k, none = pool(), batch(n=0)
    G.kv_write(rows(tokens=0), rows(tokens=0), batch(), k, k)
    G.kv_write(rows(), rows(), none, k, k)
    G.kv_read(k, k, batch(), rows(tokens=0, outer=2), rows(tokens=0, outer=2))
    G.attention(rows(heads=4, tokens=0), k, k, batch(), rows(heads=4, tokens=0, at=1), 0.1)
    G.attention(rows(heads=4), k, k, none, rows(heads=4, at=1), 0.1)
    assert _lib.load().weft_hip_get_last_error() == 0
