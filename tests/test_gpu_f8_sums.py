"""Products of 8-bit floats to 16 bits, whose sums have 32 bits whatever the number of tokens (GPU).

An output's sum is off by b as 32-bit outputs are (tests/test_gpu_mul_mat_f8.py), then rounded: 2^-11 of its
size, 2^-25 below 2^-14.  The bound of a product that may cut its sums is none here.

Of a whole result of independent terms: with r the error of the rounded 64-bit result, an
error e before the rounding adds its norm at most, and the roundings of the n shifted numbers
have the norm of r within 1 / (2 sqrt(n)) of it in the mean square (three of these: 1 % from 22500 outputs on).  A
block's partial sums are no larger than the row's in the mean, so e is at most (127 2^-23 + (2 + blocks) 2^-24) of
the result's norm."""
from __future__ import annotations

import numpy as np
import pytest

from tests._f8 import F8, F16, F32, VALUE, Rows, Scales, up
from tests.test_gpu_mul_mat_f8 import Case, Case2, bound
from weft_amd import ggml as G

pytestmark = pytest.mark.gpu

# by tiles of 32, 64 and 128 tokens, with K in ranges, rows through registers, tiles of 256 and theirs with a rest
SHAPES = [(17, 300, 640), (40, 2048, 1024), (70, 2000, 384), (200, 515, 1111), (509, 700, 2048), (1024, 1500, 640),
          (4096, 3841, 1024), (2040, 9001, 1024)]


def sharp(c):
    """The case's outputs, each within its own bound and all of them within theirs."""
    c.call()
    c.hip.torch.cuda.synchronize()
    assert c.hip.last_error() == 0
    got = c.yd.numpy().astype(np.float64)
    want, mass = c.want()
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound(mass, want, c.k, F16)).all()
    r = np.linalg.norm(want.astype(np.float16).astype(np.float64) - want)
    e = (127 * 2.0 ** -23 + (2 + up(c.k)) * 2.0 ** -24) * np.linalg.norm(want)
    off = np.linalg.norm(got - want)
    print(f"off {off / np.linalg.norm(want):.3e}, the rounding alone {r / np.linalg.norm(want):.3e}", flush=True)
    if want.size >= 22500:
        assert off <= 1.01 * r + e
    return got


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("src", [F8, F16])
def test_whole_results(hip, m, n, k, src):
    sharp(Case(hip, m, n, k, src, F16))


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_sums_that_cancel(hip, m, n, k):
    """Each eight values have two products of the largest size and opposite signs beside six of 15 to 18: of the
    eight, 90 to 108 are left.  The bound is 128 x 2^-23 of a mass of 2 x 448^2 an eight, 6.2."""
    c = Case(hip, m, n, k, F8, F16)
    rng = np.random.default_rng(k)
    sixteen, one = 0x58, 0x38
    assert VALUE[sixteen] == 16 and VALUE[one] == 1 and VALUE[0x7e] == 448
    i = np.arange(k) % 8
    c.w_codes = np.where(i == 0, 0x7e, np.where(i == 1, 0xfe, sixteen - 1 + rng.integers(0, 3, (n, k)))).astype(np.uint8)
    c.x_codes = np.broadcast_to(np.where(i < 2, 0x7e, one).astype(np.uint8), (m, k)).copy()
    c.x_codes[:, k // 8 * 8:] = 0  # an eight that the row's end cuts has no pair
    c.w_scales[:], c.x_scales[:] = 1 / 128, 1 / 16
    sharp_pairs = Case2(hip, c)
    got = sharp_pairs.check()
    want, mass = c.want()
    assert (want >= k // 8 * 85 / 2048).all()
    assert (np.abs(got - want) <= bound(mass, want, k, F16)).all()


@pytest.mark.parametrize("m", [30, 70, 300])
def test_every_code(hip, m):
    """One code a row: each product alone, in places of a block, is the exact one's rounding."""
    rng = np.random.default_rng(m)
    c = Case(hip, m, 256, 256, F8, F16)
    finite = np.array([i for i in range(256) if np.isfinite(VALUE[i])], np.uint8)
    c.w_codes = rng.permuted(np.resize(finite, (256, 256)), axis=1)
    c.w_scales[:], c.x_scales[:] = 1 / 64, 1
    c.x_codes = rng.choice(finite, (m, 256))
    sharp(Case2(hip, c))
    for k0 in range(0, 256, 37):
        c.x_codes = np.zeros((m, 256), np.uint8)
        c.x_codes[:, k0] = rng.choice(finite, m)
        got = Case2(hip, c).check()
        assert np.array_equal(got, (np.outer(VALUE[c.x_codes[:, k0]], VALUE[c.w_codes[:, k0]]) / 64).astype(np.float16))


@pytest.mark.parametrize("m,n,k", [(20, 140, 700), (300, 140, 700), (4096, 3841, 640)])
def test_zeros_and_scales(hip, m, n, k):
    """Blocks of zeros, scales of zero and large ones beside small ones."""
    c = Case(hip, m, n, k, F8, F16)
    c.w_scales[0, 2] = 0
    c.w_scales[1, 3] *= 512
    c.x_scales[0, 1] = 1e-20
    c.x_codes[m - 1] = 0x80  # minus zero
    c.w_codes[n - 1] = 0
    got = sharp(Case2(hip, c))
    assert (got[m - 1] == 0).all() and (got[:, n - 1] == 0).all()


@pytest.mark.parametrize("m,n,k", [(37, 270, 515), (700, 270, 515), (3850, 4096, 640)])
def test_nan_and_infinity_stay_in_their_rows(hip, m, n, k):
    rng = np.random.default_rng(m)
    w, x = rng.standard_normal((n, k)).astype(np.float32), rng.standard_normal((m, k)).astype(np.float32)
    w[3, k - 1], w[200, 0], x[m - 1, 130] = np.nan, np.inf, -np.inf
    got = Case(hip, m, n, k, F8, F16, w=w, x=x).check()
    nan = np.isnan(got)
    assert nan[:, [3, 200]].all() and nan[m - 1].all() and nan.sum() == 2 * m + n - 2


@pytest.mark.parametrize("m,n,k", [(50, 390, 1300), (400, 390, 1300), (3841, 4096, 1024)])
def test_calls_agree_and_overlap(hip, m, n, k):
    """The same call again, on two streams with a work buffer each, gives the same bits."""
    torch = hip.torch
    cases = [Case(hip, m, n, k, F32, F16, seed=s) for s in (1, 2)]
    first = [sharp(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    try:
        for _ in range(3):
            for c, s in zip(cases, streams):
                hip._lib.set_stream(s.cuda_stream)
                c.call()
    finally:
        hip._lib.set_stream(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for c, f in zip(cases, first):
        assert np.array_equal(c.yd.numpy().astype(np.float64), f)


@pytest.mark.parametrize("m,n,k", [(24, 140, 500), (300, 140, 500), (4096, 3841, 640)])
def test_a_graph_replayed_with_other_inputs(hip, m, n, k):
    torch = hip.torch
    c = Case(hip, m, n, k, F8, F16)
    size = G.mul_mat_f8_work_size(c.wd.tensor, c.xd.tensor)
    work = hip.empty(size, fill=0x7f)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=side):
            hip._lib.set_stream(side.cuda_stream)
            G.mul_mat_f8(c.wd.tensor, c.wsd.tensor, c.xd.tensor, c.xsd.tensor, c.yd.tensor, work.ptr, size)
    finally:
        hip._lib.set_stream(torch.cuda.current_stream().cuda_stream)
    for seed in range(3):
        c.x_codes = np.random.default_rng(seed).permuted(c.x_codes, axis=1)
        c.xd.dev.t[:c.x_codes.size].copy_(torch.from_numpy(c.x_codes.reshape(-1)))
        graph.replay()
        torch.cuda.synchronize()
        got = c.yd.numpy().copy()
        assert np.array_equal(sharp(c).astype(np.float16), got)


@pytest.mark.parametrize("n", [300, 2000])
def test_a_token_is_the_same_whatever_the_number_of_tokens(hip, n):
    """What a token's outputs may differ by between calls of different kernels: their sums' rounding in 32 bits."""
    rng = np.random.default_rng(n)
    w = rng.standard_normal((n, 640)).astype(np.float32)
    x = rng.standard_normal((2100, 640)).astype(np.float32)
    few, wide = (Case(hip, m, n, 640, F32, F16, w=w, x=x[:m]) for m in (16, 2100))
    a, b = sharp(few), sharp(wide)[:16]
    want, mass = few.want()
    assert (np.abs(a - b) <= 2 * bound(mass, want, 640, F16)).all()
    # in the mean far fewer: two roundings of numbers that differ by e differ by a step with the chance e / step, and e is
    # 128 x 2^-24 of a value at most where steps are 2^-11 of it and more: 1.6 %
    assert (a != b).mean() <= 0.016


@pytest.mark.parametrize("m,n,k", [(441, 33613, 256), (1874, 8710, 384), (4090, 3900, 512), (4096, 3841, 640), (3850, 4096, 1152)])
def test_large_tiles_of_few_blocks(hip, m, n, k):
    """Tiles of 256 load two blocks ahead: from two blocks on, odd and even numbers of them."""
    hip._lib.launch_log()
    sharp(Case(hip, m, n, k, F8, F16))
    assert "f8_large_kernel" in hip._lib.launch_log()
