"""What the 8-bit float products, the rotation of heads and the log probabilities refuse,
before anything is launched (no GPU): the code raised, and that nothing stays recorded."""
from __future__ import annotations

import pytest

from weft_amd import _lib, ggml as G
from tests.test_layer_refusals import A, INVALID, NOT_SUPPORTED, refused

INF, NAN = float("inf"), float("nan")


def swapped(args, i, value):
    a = list(args)
    a[i] = value
    return a


# ------------------------------------------------------------- the quantizer
def quantize_args(k=300, rows=200, blocks=False, t=G.F32):
    return [G.tensor(t, (k, rows), A[0]), G.tensor(G.F8_E4M3, (k, rows), A[1]),
            G.tensor(G.F32, (-(-k // 128), -(-rows // 128) if blocks else rows), A[2])]


@pytest.mark.parametrize("blocks", [False, True])
def test_quantizer(blocks):
    ok = quantize_args(blocks=blocks)
    for i in range(3):
        assert refused(G.quantize_f8, *swapped(ok, i, None)) == INVALID
        for t in (G.Q8_0, G.I32):
            assert refused(G.quantize_f8, *swapped(ok, i, G.tensor(t, (512, 4), A[i]))) == NOT_SUPPORTED
    rows = ok[2].ne[1]
    for bad in (G.tensor(G.F32, (300, 199), A[0]), G.tensor(G.F32, (299, 200), A[0]), G.tensor(G.F32, (300, 200, 2), A[0]),
                G.tensor(G.F32, (300, 200), A[0] + 2), G.tensor(G.F32, (300, 200), 0),
                G.tensor(G.F32, (300, 200), A[0], [8, 2400, 0, 0]), G.tensor(G.F32, (300, 200), A[0], [4, 1202, 0, 0])):
        assert refused(G.quantize_f8, *swapped(ok, 0, bad)) == INVALID
    for bad in (G.tensor(G.F8_E4M3, (300, 201), A[1]), G.tensor(G.F8_E4M3, (300, 200), 0),
                G.tensor(G.F8_E4M3, (300, 200), A[1], [2, 600, 0, 0]), G.tensor(G.F8_E4M3, (300, 200, 1, 2), A[1])):
        assert refused(G.quantize_f8, *swapped(ok, 1, bad)) == INVALID
    for bad in (G.tensor(G.F32, (2, rows), A[2]), G.tensor(G.F32, (3, 3), A[2]), G.tensor(G.F32, (3, rows), 0),
                G.tensor(G.F32, (3, rows), A[2] + 1), G.tensor(G.F32, (3, rows), A[2], [4, 10, 0, 0])):
        assert refused(G.quantize_f8, *swapped(ok, 2, bad)) == INVALID
    G.quantize_f8(*quantize_args(rows=0))
    assert _lib.load().weft_hip_get_last_error() == 0


# --------------------------------------------------------------- the product
def product_args(m=5, n=200, k=300, t=G.F32, out=G.F32):
    return [G.tensor(G.F8_E4M3, (k, n), A[0]), G.tensor(G.F32, (-(-k // 128), -(-n // 128)), A[1]),
            G.tensor(t, (k, m), A[2]), G.tensor(G.F32, (-(-k // 128), m), A[3]) if t == G.F8_E4M3 else None,
            G.tensor(out, (n, m), A[4]), A[5], 1 << 30]


@pytest.mark.parametrize("t", [G.F32, G.F16, G.F8_E4M3])
def test_product(t):
    ok = product_args(t=t)
    for i in (0, 1, 2, 4):
        assert refused(G.mul_mat_f8, *swapped(ok, i, None)) == INVALID
    for i, types in ((0, (G.F32, G.Q8_0)), (1, (G.F16,)), (2, (G.Q8_K, G.I32)), (4, (G.F8_E4M3, G.I32))):
        for bad in types:
            assert refused(G.mul_mat_f8, *swapped(ok, i, G.tensor(bad, (256, 4), A[i]))) == NOT_SUPPORTED
    scales = G.tensor(G.F32, (3, 5), A[3])
    assert refused(G.mul_mat_f8, *swapped(ok, 3, None if t == G.F8_E4M3 else scales)) == INVALID
    assert refused(G.mul_mat_f8, *swapped(ok, 3, G.tensor(G.F16, (3, 5), A[3]))) == NOT_SUPPORTED
    unit = {G.F32: 4, G.F16: 2, G.F8_E4M3: 1}[t]
    for i, shape, kind, e in ((0, (300, 200), G.F8_E4M3, 1), (2, (300, 5), t, unit), (4, (200, 5), G.F32, 4)):
        for bad in (G.tensor(kind, (shape[0] + 1, shape[1]), A[i]), G.tensor(kind, (*shape, 2), A[i]),
                    G.tensor(kind, (*shape, 1, 2), A[i]), G.tensor(kind, shape, 0),
                    G.tensor(kind, shape, A[i], [2 * e, 2 * e * shape[0], 0, 0])):
            assert refused(G.mul_mat_f8, *swapped(ok, i, bad)) == INVALID
        if e > 1:
            assert refused(G.mul_mat_f8, *swapped(ok, i, G.tensor(kind, shape, A[i] + 1))) == INVALID
            assert refused(G.mul_mat_f8, *swapped(ok, i, G.tensor(kind, shape, A[i], [e, e * shape[0] + 1, 0, 0]))) == INVALID
    for bad in (G.tensor(G.F32, (2, 2), A[1]), G.tensor(G.F32, (3, 200), A[1]), G.tensor(G.F32, (3, 2), A[1] + 2),
                G.tensor(G.F32, (3, 2), 0), G.tensor(G.F32, (3, 2), A[1], [6, 12, 0, 0])):
        assert refused(G.mul_mat_f8, *swapped(ok, 1, bad)) == INVALID
    assert refused(G.mul_mat_f8, *product_args(k=0, t=t)) == INVALID
    if t != G.F8_E4M3:
        size = G.mul_mat_f8_work_size(*product_args(m=400, t=t)[0:3:2])
        assert size >= 400 * 384
        big = product_args(m=400, t=t)
        assert refused(G.mul_mat_f8, *swapped(big, 6, size - 1)) == INVALID
        assert refused(G.mul_mat_f8, *swapped(big, 5, 0)) == INVALID
        assert refused(G.mul_mat_f8, *swapped(big, 5, A[5] + 8)) == INVALID


def test_empty_products_launch_nothing():
    for kw in ({"m": 0}, {"n": 0}):
        a = product_args(**kw)
        assert G.mul_mat_f8_work_size(a[0], a[2]) == 0
        G.mul_mat_f8(*a[:5])
    assert _lib.load().weft_hip_get_last_error() == 0


# -------------------------------------------------------------- the rotation
def rope_args(d=64, heads=4, kv=2, tokens=5, n=64, t=G.F32, out=G.F32, eps=1e-6, **kw):
    return [G.tensor(t, (d, heads, tokens), A[0]), G.tensor(t, (d, kv, tokens), A[1]), G.tensor(out, (d, heads, tokens), A[2]),
            G.tensor(out, (d, kv, tokens), A[3]), G.tensor(G.I32, (tokens,), A[4]), G.head_rope(n, **kw), eps,
            G.tensor(G.F32, (d,), A[5]), G.tensor(G.F32, (d,), A[6]), G.tensor(G.F32, (n // 2,), A[7])]


def test_heads():
    ok = rope_args()
    for i in (0, 1, 2, 3, 4):
        assert refused(G.head_norm_rope, *swapped(ok, i, None)) == INVALID
    for i in (0, 1, 2, 3):
        heads = 4 if i in (0, 2) else 2
        assert refused(G.head_norm_rope, *swapped(ok, i, G.tensor(G.Q8_0, (64, heads, 5), A[i]))) == NOT_SUPPORTED
        for bad in (G.tensor(G.F32, (62, heads, 5), A[i]), G.tensor(G.F32, (64, heads, 6), A[i]),
                    G.tensor(G.F32, (64, heads, 5, 2), A[i]), G.tensor(G.F32, (64, 0, 5), A[i]),
                    G.tensor(G.F32, (64, heads, 5), 0), G.tensor(G.F32, (64, heads, 5), A[i] + 2),
                    G.tensor(G.F32, (64, heads, 5), A[i], [8, 512, 2048, 0]),
                    G.tensor(G.F32, (64, heads, 5), A[i], [4, 258, 2048, 0]),
                    G.tensor(G.F32, (64, heads, 5), A[i], [4, 256, 2050, 0])):
            assert refused(G.head_norm_rope, *swapped(ok, i, bad)) == INVALID
    assert refused(G.head_norm_rope, *swapped(ok, 1, G.tensor(G.F16, (64, 2, 5), A[1]))) == NOT_SUPPORTED
    assert refused(G.head_norm_rope, *swapped(ok, 2, G.tensor(G.F32, (64, 5, 5), A[2]))) == INVALID
    assert refused(G.head_norm_rope, *rope_args(d=258, n=258)) == NOT_SUPPORTED
    assert refused(G.head_norm_rope, *rope_args(d=0, n=0)) == INVALID


def test_rotations():
    for n in (66, 3, -2):
        assert refused(G.head_norm_rope, *swapped(rope_args(), 5, G.head_rope(n))) == INVALID
    for kw in ({"base": 0.0}, {"base": -1.0}, {"base": INF}, {"base": NAN}, {"scale": INF}, {"scale": NAN},
               {"magnitude": INF}, {"magnitude": NAN}):
        assert refused(G.head_norm_rope, *rope_args(**kw)) == INVALID
    for eps in (-1e-6, NAN):
        assert refused(G.head_norm_rope, *rope_args(eps=eps)) == INVALID
    ok = rope_args()
    assert refused(G.head_norm_rope, *swapped(ok, 6, None)) == INVALID  # weights without a norm
    assert refused(G.head_norm_rope, *swapped(ok, 4, G.tensor(G.F32, (5,), A[4]))) == NOT_SUPPORTED
    for bad in (G.tensor(G.I32, (4,), A[4]), G.tensor(G.I32, (5,), A[4] + 2), G.tensor(G.I32, (5,), 0)):
        assert refused(G.head_norm_rope, *swapped(ok, 4, bad)) == INVALID
    for i, n in ((7, 64), (8, 64), (9, 32)):
        assert refused(G.head_norm_rope, *swapped(ok, i, G.tensor(G.F16, (n,), A[i]))) == NOT_SUPPORTED
        for bad in (G.tensor(G.F32, (n - 1,), A[i]), G.tensor(G.F32, (n,), 0), G.tensor(G.F32, (n, 2), A[i])):
            assert refused(G.head_norm_rope, *swapped(ok, i, bad)) == INVALID
    none = swapped(swapped(ok, 1, None), 3, None)
    assert refused(G.head_norm_rope, *none) == INVALID  # a weight for no keys
    assert refused(G.head_norm_rope, *swapped(ok, 5, G.head_rope(0))) == INVALID  # factors for no pairs


def test_no_tokens():
    G.head_norm_rope(*rope_args(tokens=0))
    assert _lib.load().weft_hip_get_last_error() == 0


# ------------------------------------------------------- the log probabilities
def choice_args(v=5000, rows=3, given=2, top=4, t=G.F32):
    return [G.tensor(t, (v, rows), A[0]), G.tensor(G.I32, (given, rows), A[1]), G.tensor(G.F32, (given, rows), A[2]),
            G.tensor(G.F32, (rows,), A[3]), G.tensor(G.I32, (top, rows), A[4]), G.tensor(G.F32, (top, rows), A[5]), 1.0, A[6],
            1 << 30]


def test_choices():
    ok = choice_args()
    for i in (0, 1, 2, 4, 5):
        assert refused(G.log_probs, *swapped(ok, i, None)) == INVALID
    assert refused(G.log_probs, *swapped(ok, 0, G.tensor(G.Q8_0, (5024, 3), A[0]))) == NOT_SUPPORTED
    for i, n, t, wrong in ((1, 2, G.I32, G.F32), (2, 2, G.F32, G.F16), (4, 4, G.I32, G.F32), (5, 4, G.F32, G.I32)):
        assert refused(G.log_probs, *swapped(ok, i, G.tensor(wrong, (n, 3), A[i]))) == NOT_SUPPORTED
        for bad in (G.tensor(t, (n + 1, 3), A[i]), G.tensor(t, (n, 4), A[i]), G.tensor(t, (n, 3, 2), A[i]), G.tensor(t, (n, 3), 0),
                    G.tensor(t, (n, 3), A[i] + 2), G.tensor(t, (n, 3), A[i], [8, 64, 0, 0]), G.tensor(t, (n, 3), A[i], [4, 18, 0, 0])):
            assert refused(G.log_probs, *swapped(ok, i, bad)) == INVALID
    for bad in (G.tensor(G.F32, (4,), A[3]), G.tensor(G.F32, (3,), 0), G.tensor(G.F32, (1, 3), A[3])):
        assert refused(G.log_probs, *swapped(ok, 3, bad)) == INVALID
    for bad in (G.tensor(G.F32, (5000, 3, 2), A[0]), G.tensor(G.F32, (0, 3), A[0]), G.tensor(G.F32, (5000, 3), 0),
                G.tensor(G.F32, (5000, 3), A[0] + 2), G.tensor(G.F32, (5000, 3), A[0], [4, 20002, 0, 0])):
        assert refused(G.log_probs, *swapped(ok, 0, bad)) == INVALID
    assert refused(G.log_probs, *choice_args(top=65)) == INVALID
    assert refused(G.log_probs, *choice_args(v=3)) == INVALID  # more alternatives than logits
    for s in (0.0, -1.0, INF, NAN):
        assert refused(G.log_probs, *swapped(ok, 6, s)) == INVALID
    long = choice_args(v=100000)
    size = G.log_probs_work_size(long[0], 4)
    assert size > 0
    assert refused(G.log_probs, *swapped(long, 8, size - 1)) == INVALID
    assert refused(G.log_probs, *swapped(long, 7, 0)) == INVALID
    assert refused(G.log_probs, *swapped(long, 7, A[6] + 8)) == INVALID


def test_nothing_asked():
    G.log_probs(*choice_args(rows=0))
    G.log_probs(choice_args()[0], None, None, None, None, None)
    assert _lib.load().weft_hip_get_last_error() == 0
