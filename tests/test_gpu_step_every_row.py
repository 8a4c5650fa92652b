"""The most rows a call may have (GPU), each row's output of its own: 2^31 - 1 rows that share their inputs and write
one after the other.  A launch that is cut short, or one part of a call at the wrong place, leaves poison."""
from __future__ import annotations

import numpy as np
import pytest

from weft_amd import ggml as G

pytestmark = pytest.mark.gpu
MOST = (1 << 31) - 1
#: rows behind the last, which stay as they were
BEHIND = 4096


def filled(hip, rows, dtype, value):
    t = hip.torch.empty(rows + BEHIND, dtype=dtype, device=hip.dev)
    t.fill_(value)
    return t


def written(hip, out, rows, want, poison):
    hip.torch.cuda.synchronize()
    assert hip.last_error() == 0
    step = 1 << 28  # a comparison's result has a byte an element
    wrong = sum(int((out[i:min(i + step, rows)] != want).sum()) for i in range(0, rows, step))
    assert wrong == 0 and bool((out[rows:] == poison).all())


@pytest.mark.parametrize("rows", [MOST, MOST - 63])
def test_quantize_f8(hip, rows):
    """Rows of one value: its code is that of 448 or -448."""
    x = hip.to_dev(np.float32([-0.3]))
    codes, scales = filled(hip, rows, hip.torch.uint8, 0x7f), hip.empty(4)
    print(f"quantize_f8 rows={rows}", flush=True)
    G.quantize_f8(G.tensor(G.F32, (1, rows), x.ptr, [4, 0, 0, 0]), G.tensor(G.F8_E4M3, (1, rows), codes.data_ptr()),
                  G.tensor(G.F32, (1, rows), scales.ptr, [4, 0, 0, 0]))
    written(hip, codes, rows, 0xfe, 0x7f)
    assert scales.numpy(np.float32)[0] == np.float32(0.3) / np.float32(448)


def test_scales_of_quantize_f8(hip):
    x, codes = hip.to_dev(np.float32([448 * 3.0])), hip.empty(1)
    scales = filled(hip, MOST, hip.torch.float32, -1.0)
    print("quantize_f8's scales", flush=True)
    G.quantize_f8(G.tensor(G.F32, (1, MOST), x.ptr, [4, 0, 0, 0]), G.tensor(G.F8_E4M3, (1, MOST), codes.ptr, [1, 0, 0, 0]),
                  G.tensor(G.F32, (1, MOST), scales.data_ptr(), [4, 4, 0, 0]))
    written(hip, scales, MOST, 3.0, -1.0)


@pytest.mark.parametrize("m,n", [(MOST, 1), (1, MOST), (MOST // 16, 16), (40, MOST // 40)])
def test_mul_mat_f8(hip, m, n):
    one = np.uint8([0x38, 0x38, 0x38])
    w, x, s = hip.to_dev(one), hip.to_dev(one), hip.to_dev(np.float32([2.0]))
    y = filled(hip, m * n, hip.torch.float16, 7.0)
    args = [G.tensor(G.F8_E4M3, (3, n), w.ptr, [1, 0, 0, 0]), G.tensor(G.F32, (1, -(-n // 128)), s.ptr, [4, 0, 0, 0]),
            G.tensor(G.F8_E4M3, (3, m), x.ptr, [1, 0, 0, 0]), G.tensor(G.F32, (1, m), s.ptr, [4, 0, 0, 0])]
    size = G.mul_mat_f8_work_size(args[0], args[2])
    work = hip.empty(size)
    print(f"mul_mat_f8 m={m} n={n} work={size}", flush=True)
    G.mul_mat_f8(*args, G.tensor(G.F16, (n, m), y.data_ptr()), work.ptr, size)
    written(hip, y, m * n, 12.0, 7.0)


@pytest.mark.parametrize("tokens", [MOST, MOST - 2])
def test_head_norm_rope(hip, tokens):
    """Heads of one value, normed: 1 or -1 to 16 bits."""
    x = hip.to_dev(np.float32([-3.0]))
    y = filled(hip, tokens, hip.torch.float16, 7.0)
    print(f"head_norm_rope tokens={tokens}", flush=True)
    G.head_norm_rope(G.tensor(G.F32, (1, 1, tokens), x.ptr, [4, 0, 0, 0]), None, G.tensor(G.F16, (1, 1, tokens), y.data_ptr()),
                     None, None, G.head_rope(0), 0.0)
    written(hip, y, tokens, -1.0, 7.0)


def test_heads_of_head_norm_rope(hip):
    """The most heads of a token, queries and keys."""
    heads = 1 << 28
    x = hip.to_dev(np.float32([-3.0]))
    q, k = (filled(hip, heads, hip.torch.float16, 7.0) for _ in range(2))
    print("head_norm_rope heads", flush=True)
    source = G.tensor(G.F32, (1, heads, 1), x.ptr, [4, 0, 0, 0])
    G.head_norm_rope(source, source, *(G.tensor(G.F16, (1, heads, 1), t.data_ptr()) for t in (q, k)), None, G.head_rope(0), 0.0)
    for t in (q, k):
        written(hip, t, heads, -1.0, 7.0)


@pytest.mark.parametrize("rows", [MOST, MOST - 1])
def test_log_probs(hip, rows):
    x, lp = hip.to_dev(np.float32([0.0, 1.0])), hip.empty(4)
    ids, entropy = filled(hip, rows, hip.torch.int32, -7), filled(hip, rows, hip.torch.float32, 5.0)
    lt = G.tensor(G.F32, (2, rows), x.ptr, [4, 0, 0, 0])
    print(f"log_probs rows={rows}", flush=True)
    G.log_probs(lt, None, None, G.tensor(G.F32, (rows,), entropy.data_ptr()), G.tensor(G.I32, (1, rows), ids.data_ptr()),
                G.tensor(G.F32, (1, rows), lp.ptr, [4, 0, 0, 0]))
    written(hip, ids, rows, 1, -7)
    p = 1 / (1 + np.exp(-1.0))
    first = float(entropy[0])
    assert abs(first + p * np.log(p) + (1 - p) * np.log(1 - p)) <= 1e-6
    written(hip, entropy, rows, first, 5.0)
