"""The most rows a call may have (GPU): 2^31 - 1 rows that share memory, as their outputs do.  Past
2^32 threads a launch would be cut short, so the calls are launched in parts."""
from __future__ import annotations

import numpy as np
import pytest

from tests._f8 import quantize
from weft_amd import ggml as G

pytestmark = pytest.mark.gpu
MOST = (1 << 31) - 1


def done(hip):
    hip.torch.cuda.synchronize()
    assert hip.last_error() == 0


@pytest.mark.parametrize("rows", [MOST, MOST - 63])
def test_quantize_f8(hip, rows):
    x = np.float32([3.0, -0.5, 0.1])
    xd, codes, scales = hip.to_dev(x), hip.empty(3), hip.empty(4)
    print(f"quantize_f8 rows={rows}", flush=True)
    G.quantize_f8(G.tensor(G.F32, (3, rows), xd.ptr, [4, 0, 0, 0]), G.tensor(G.F8_E4M3, (3, rows), codes.ptr, [1, 0, 0, 0]),
                  G.tensor(G.F32, (1, rows), scales.ptr, [4, 0, 0, 0]))
    done(hip)
    want, s = quantize(x[None], 1)
    assert np.array_equal(codes.numpy(), want[0]) and scales.numpy(np.float32)[0] == s[0, 0]


@pytest.mark.parametrize("m,n", [(MOST, 1), (1, MOST), (40, MOST // 16)])
def test_mul_mat_f8(hip, m, n):
    """Unit weights and tokens of one code: 3 x 448 / 448 x the scale of each."""
    one = np.uint8([0x38, 0x38, 0x38])
    wd, xd, s, y = hip.to_dev(one), hip.to_dev(one), hip.to_dev(np.float32([2.0])), hip.empty(4, fill=0xff)
    args = [G.tensor(G.F8_E4M3, (3, n), wd.ptr, [1, 0, 0, 0]), G.tensor(G.F32, (1, -(-n // 128)), s.ptr, [4, 0, 0, 0]),
            G.tensor(G.F8_E4M3, (3, m), xd.ptr, [1, 0, 0, 0]), G.tensor(G.F32, (1, m), s.ptr, [4, 0, 0, 0])]
    # outputs of a row lie one after the other: a row of few is written by all
    wide = hip.torch.full((n,), 7.0, dtype=hip.torch.float16 if n > 1 << 20 else hip.torch.float32,
                          device=hip.dev)
    t = G.F16 if n > 1 << 20 else G.F32
    size = G.mul_mat_f8_work_size(args[0], args[2])
    work = hip.empty(size)
    print(f"mul_mat_f8 m={m} n={n} work={size}", flush=True)
    G.mul_mat_f8(*args, G.tensor(t, (n, m), wide.data_ptr(), [wide.element_size(), 0, 0, 0]), work.ptr, size)
    done(hip)
    assert bool((wide == 12.0).all()) and y.numpy()[0] == 0xff


@pytest.mark.parametrize("tokens", [MOST, MOST - 2])
def test_head_norm_rope(hip, tokens):
    x = np.float32([3.0, -4.0])
    xd, y, p = hip.to_dev(x), hip.empty(8), hip.to_dev(np.int32([0]))
    print(f"head_norm_rope tokens={tokens}", flush=True)
    G.head_norm_rope(G.tensor(G.F32, (2, 1, tokens), xd.ptr, [4, 0, 0, 0]), None, G.tensor(G.F32, (2, 1, tokens), y.ptr, [4, 0, 0, 0]),
                     None, None, G.head_rope(0), 0.0)
    done(hip)
    assert (np.abs(y.numpy(np.float32) - x / np.sqrt(12.5)) <= 1e-6).all()


@pytest.mark.parametrize("rows", [MOST, MOST - 1])
def test_log_probs(hip, rows):
    x = np.float32([0.0, 1.0])
    xd, ids, lp, e = hip.to_dev(x), hip.empty(4), hip.empty(4), hip.torch.full((1,), 5.0, device=hip.dev)
    lt = G.tensor(G.F32, (2, rows), xd.ptr, [4, 0, 0, 0])
    assert G.log_probs_work_size(lt, 1) == 0
    print(f"log_probs rows={rows}", flush=True)
    G.log_probs(lt, None, None, None, G.tensor(G.I32, (1, rows), ids.ptr, [4, 0, 0, 0]),
                G.tensor(G.F32, (1, rows), lp.ptr, [4, 0, 0, 0]))
    done(hip)
    assert ids.numpy(np.int32)[0] == 1 and abs(lp.numpy(np.float32)[0] + np.log1p(np.exp(-1))) <= 1e-6 and e[0] == 5.0
