"""The operators of a step together, from a row to its answer (GPU).

Against 64 bits with the weights as their codes have them, the cache as its records have it and
every activation quantized as the operators do, at the same places.  Two roundings of
numbers that differ by e < a step differ by a step with the chance e / step: by e x step in
the mean square.  e4m3 steps are 2^-4 to 2^-3 of a value, 0.07 of the row's rms for a value of mean size
0.8 of it.  The attention's 16-bit roundings leave 5e-4 of its rows, so their codes differ by
sqrt(0.8 x 5e-4 x 0.07) = 0.5 %; beside the residual of the same size that is 0.4 % of the sum, and the last
product's codes differ by sqrt(0.8 x 0.004 x 0.07) = 1.5 %.  3 % is allowed.  What
log_probs says of the step's own logits is held to 32 bits: 1e-4 (sums of 5003 terms, 6e-8 each at most)."""
from __future__ import annotations

import numpy as np
import pytest

from tests._f8 import BLOCK, quantize, values
from tests._layer import decode, encode

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, KV_HEADS, D, VOCABULARY, EPS = 512, 8, 2, 64, 5003, 1e-5


def norm(x, w):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * w


def through_f8(x):
    codes, scales = quantize(x.astype(np.float32), 1)
    return values(codes, scales, 1)


def turned(x):
    """x (tokens, heads, D) at positions 0, 1, .."""
    t = np.arange(len(x))[:, None] * 10000.0 ** (-2 * np.arange(D // 2) / D)
    c, s = np.cos(t)[:, None], np.sin(t)[:, None]
    a, b = x[..., :D // 2], x[..., D // 2:]
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


def plain(model, x):
    """One sequence's logits."""
    w = {n: values(c.view(torch.uint8).cpu().numpy(), s.cpu().numpy(), BLOCK) for n, (c, s) in model.weights.items()}
    g = {n: t.double().cpu().numpy() for n, t in model.norms.items()}
    n = len(x)
    y = through_f8(norm(x, g["in"]))
    q, k, v = ((y @ w[i].T).reshape(n, -1, D) for i in "qkv")
    q, k = turned(norm(q, g["q"])), turned(norm(k, g["k"]))
    k, v = (decode("q8_0", encode("q8_0", np.ascontiguousarray(c, np.float32))) for c in (k, v))
    s = np.einsum("thsd,jhd->hstj", q.reshape(n, KV_HEADS, -1, D), k) / np.sqrt(D)
    s = np.where(np.arange(n)[None, :] <= np.arange(n)[:, None], s, -np.inf)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    o = np.einsum("hstj,jhd->thsd", p, v).reshape(n, HEADS * D)
    return through_f8(norm(x + through_f8(o) @ w["o"].T, g["out"])) @ w["vocabulary"].T


def model_of(**kw):
    from examples.answer_step import build

    return build(torch.device("cuda:0"), HIDDEN, HEADS, KV_HEADS, D, VOCABULARY, **kw)


def rows(n, seed):
    return np.random.default_rng(seed).standard_normal((n, HIDDEN)).astype(np.float32)


def test_prompts_and_decoded_tokens(hip):
    prompts, steps = (37, 5, 150), 3
    host = [rows(n + steps, n) for n in prompts]
    x = [torch.from_numpy(h).cuda() for h in host]
    model, other = model_of(), model_of()
    given = torch.randint(0, VOCABULARY, (sum(len(h) for h in host), 1), dtype=torch.int32).cuda()
    given[3] = -1
    whole = other.step(torch.cat(x), other.describe([len(h) for h in host]), given, 6)
    first = model.step(torch.cat([a[:n] for a, n in zip(x, prompts)]), model.describe(list(prompts)), given[:sum(prompts)], 6)
    decoded = [model.step(torch.stack([a[n + i] for a, n in zip(x, prompts)]), model.describe([1] * 3), given[:3], 6)
               for i in range(steps)]
    torch.cuda.synchronize()
    assert hip.last_error() == 0
    at = np.cumsum([0] + [len(h) for h in host])
    at_first = np.cumsum([0, *prompts])
    for i, (h, n) in enumerate(zip(host, prompts)):
        want = plain(model, h.astype(np.float64))
        got = [whole[0][at[i]:at[i + 1]], torch.cat([first[0][at_first[i]:at_first[i + 1]], *(d[0][i:i + 1] for d in decoded)])]
        for g in got:
            g = g.double().cpu().numpy()
            assert np.isfinite(g).all()
            assert (np.linalg.norm(g - want, axis=1) <= 0.03 * np.linalg.norm(want, axis=1)).all()
    for logits, lp, entropy, ids, top in [whole, first, *decoded]:
        z = torch.log_softmax(logits.double(), -1)
        ok = (asked := given[:len(z)]) >= 0
        assert (lp - torch.gather(z, 1, asked.long().clamp_min(0)))[ok].abs().max() <= 1e-4
        assert (entropy + (z.exp() * z).sum(-1)).abs().max() <= 1e-4
        order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :6]
        assert torch.equal(ids.long(), order) and (top - torch.gather(z, 1, order)).abs().max() <= 1e-4


def test_a_decode_step_replayed_from_a_graph(hip):
    """Captured once, replayed with other rows, positions and lengths in the same memory: bit for bit the eager steps."""
    prompts = [20, 33]
    eager, captured = model_of(), model_of()
    prompt = torch.from_numpy(rows(sum(prompts), 5)).cuda()
    told = torch.full((sum(prompts), 1), 17, dtype=torch.int32, device="cuda")
    for m in (eager, captured):
        m.step(prompt, m.describe(prompts), told, 4)
    x = torch.from_numpy(rows(2, 6)).cuda()
    batch = list(captured.describe([1, 1]))
    # room for the pages that later steps need
    pages = torch.full((2, 8), -1, dtype=torch.int32, device="cuda")
    pages[:, :batch[0].shape[1]] = batch[0]
    batch[0] = pages
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        out = captured.step(x, batch, told[:2], 4)
    hip._lib.set_stream(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        row = torch.from_numpy(rows(2, 60 + i)).cuda()
        b = list(eager.describe([1, 1]))
        wide = torch.full_like(pages, -1)
        wide[:, :b[0].shape[1]] = b[0]
        b[0] = wide
        want = [t.clone() for t in eager.step(row, b, told[:2], 4)]
        x.copy_(row)
        for kept, now in zip(batch, (b if i == 0 else [wide, *b[1:]])):
            kept.copy_(now)
        if i > 0:
            captured.describe([1, 1])
        graph.replay()
        torch.cuda.synchronize()
        for a, w in zip(out, want):
            assert torch.equal(a, w)
