"""The operators of a decoder layer's attention half together (GPU).

Against 64 bits without any rounding of activations: a Q8_K row of normal values
is off by at most 4 / 127 / sqrt(12) = 0.9 % rms, a Q8_0 cache row by 0.8 %.
Scores of unit spread are then off by 1.5 %, the weighted values by 1.5 % and
their own 1.2 %, and the output product's records by 0.9 % again: 2.2 % in all;
5 % is allowed.

Decoded tokens against the same tokens read at once: products of other sums and
16-bit roundings (2^-10) move at most a tenth of the output's records by one
step of 4 / 127, which is 1 % rms; 2 % is allowed."""
from __future__ import annotations

import numpy as np
import pytest

import oracle as o

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, KV_HEADS, D = 512, 8, 2, 64


def plain(layer, x, window=0, sinks=0):
    """One sequence's outputs in 64 bits."""
    w = {n: o.dequantize("q4_k", t.cpu().numpy(), HIDDEN).astype(np.float64) for n, t in layer.weights.items()}
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5)
    n = len(x)
    q = (y @ w["q"].T).reshape(n, KV_HEADS, HEADS // KV_HEADS, D)
    k, v = ((y @ w[i].T).reshape(n, KV_HEADS, D) for i in "kv")
    s = np.einsum("thsd,jhd->hstj", q, k) / np.sqrt(D)
    t, j = np.arange(n)[:, None], np.arange(n)[None, :]
    seen = j <= t
    if window:
        seen &= (j > t - window) | (j < sinks)
    s = np.where(seen, s, -np.inf)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return np.einsum("hstj,jhd->thsd", p, v).reshape(n, HEADS * D) @ w["o"].T


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 3)])
def test_decoded_tokens_are_those_read_at_once(hip, window, sinks):
    from examples.decoder_layer import build, decoded_and_at_once

    prompts, steps = (37, 5, 150), 3
    rng = np.random.default_rng(7)
    host = [rng.standard_normal((n + steps, HIDDEN)).astype(np.float32) for n in prompts]
    x = [torch.from_numpy(h).cuda() for h in host]

    def layer():
        return build(x[0].device, HIDDEN, HEADS, KV_HEADS, D, window=window, sinks=sinks)

    first = layer()
    y, whole = decoded_and_at_once(first, layer(), x, prompts)
    torch.cuda.synchronize()
    assert hip.last_error() == 0
    y, whole = y.double().cpu().numpy(), whole.double().cpu().numpy()
    assert np.isfinite(y).all()
    for s, n in enumerate(prompts):
        assert np.linalg.norm(y[s] - whole[s]) <= 0.02 * np.linalg.norm(whole[s])
        want = plain(first, host[s].astype(np.float64), window, sinks)[n:]
        for got in (y[s], whole[s]):
            assert np.linalg.norm(got - want) <= 0.05 * np.linalg.norm(want)


def test_the_residual_is_added_once(hip):
    from examples.decoder_layer import build

    rng = np.random.default_rng(8)
    a, b = (torch.from_numpy(rng.standard_normal((9, HIDDEN)).astype(np.float32)).cuda() for _ in range(2))
    total, out = build(a.device, HIDDEN, HEADS, KV_HEADS, D).forward(a, b, [9])
    same, whole = build(a.device, HIDDEN, HEADS, KV_HEADS, D).forward(a + b, None, [9])
    torch.cuda.synchronize()
    assert torch.equal(total, a + b) and torch.equal(total, same)
    assert torch.equal(out, whole)
