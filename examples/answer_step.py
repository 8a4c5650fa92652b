"""A decoder step from its input row to an answer, out of the library's operators with
8-bit float weights:

    add_rms_norm -> quantize_f8 -> mul_mat_f8 (q, k, v) -> head_norm_rope -> kv_write
      -> attention -> mul_mat_f8 (o) -> add_rms_norm -> mul_mat_f8 (vocabulary) -> log_probs

The layer's input is quantized once for its three products (the others quantize theirs on the
way); queries and keys are normed and turned where the products left them; the step ends
with the log probability of a token of each row, the row's entropy and its likeliest tokens.

Run on a GPU: ``python -m examples.answer_step`` reads two prompts and continues both with
their likeliest tokens, one by one.
"""
from __future__ import annotations

import math

import torch

from examples.decoder_layer import EPS, DecoderAttention
from weft_amd import _lib, ggml as G

TYPES = {torch.float32: G.F32, torch.float16: G.F16, torch.int32: G.I32, torch.float8_e4m3fn: G.F8_E4M3}


def dense(x):
    return G.tensor(TYPES[x.dtype], (*reversed(x.shape),), x.data_ptr())


def f8_weights(w):
    """Codes and block scales of float32 weights (out, in) on the GPU."""
    codes = torch.empty(w.shape, dtype=torch.float8_e4m3fn, device=w.device)
    scales = torch.empty(-(-w.shape[0] // 128), -(-w.shape[1] // 128), device=w.device)
    G.quantize_f8(dense(w), dense(codes), dense(scales))
    return codes, scales


class AnswerStep(DecoderAttention):
    """One layer's attention half and a vocabulary over it.  weights: "q", "k", "v", "o" and
    "vocabulary" as float32 rows (out, in) on the GPU; norms: "in", "out" (hidden) and "q", "k"
    (head size)."""

    def __init__(self, hidden, heads, kv_heads, head_size, weights, norms, *, base=10000.0, **kw):
        super().__init__(hidden, heads, kv_heads, head_size, {n: f8_weights(w) for n, w in weights.items()}, norms["in"], **kw)
        self.norms, self.rope = norms, G.head_rope(head_size, base=base)
        self.vocabulary = weights["vocabulary"].shape[0]

    def _f8(self, name, x, x_scales=None):
        codes, scales = self.weights[name]
        y = torch.empty(x.shape[0], codes.shape[0], device=x.device)
        w, xt = dense(codes), dense(x)
        work = torch.empty(G.mul_mat_f8_work_size(w, xt), dtype=torch.uint8, device=x.device)
        G.mul_mat_f8(w, dense(scales), xt, None if x_scales is None else dense(x_scales), dense(y), work.data_ptr(),
                     work.numel())
        return y

    def describe(self, new):
        """Pages for the new tokens, and what a step reads of the batch, on the GPU: (pages, starts, lengths,
        positions); a decode step that is replayed from a graph finds them in the same memory."""
        before = list(self.lengths[:len(new)])
        _, kept = self._batch(new, self.norm.device)
        positions = torch.cat([torch.arange(b, b + n, dtype=torch.int32) for b, n in zip(before, new)])
        return (*kept, positions.to(self.norm.device))

    def step(self, x, batch, tokens, n_top):
        """x: (tokens, hidden) float32; tokens: (tokens, 1) int32, whose log probabilities are asked for
        (-1: none).  Returns logits, the given tokens' log probabilities, entropies, ids and log
        probabilities of the n_top likeliest."""
        _lib.set_stream(torch.cuda.current_stream().cuda_stream)
        pages, starts, lengths, positions = batch
        kv = G.kv_batch(dense(pages), dense(starts), dense(lengths))
        n, d, device = x.shape[0], self.d, x.device

        total, y = torch.empty_like(x), torch.empty_like(x)
        G.add_rms_norm(dense(x), None, dense(self.norms["in"]), dense(total), dense(y), EPS)
        codes = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=device)
        scales = torch.empty(n, -(-self.hidden // 128), device=device)
        G.quantize_f8(dense(y), dense(codes), dense(scales))
        q, k, v = (self._f8(i, codes, scales).view(n, -1, d) for i in "qkv")
        G.head_norm_rope(dense(q), dense(k), dense(q), dense(k), dense(positions), self.rope, EPS, dense(self.norms["q"]),
                         dense(self.norms["k"]))

        pool = (d, self.page_size, self.kv_heads, self.k_cache.shape[0])
        k_cache, v_cache = (G.tensor(G.Q8_0, pool, c.data_ptr()) for c in (self.k_cache, self.v_cache))
        G.kv_write(dense(k), dense(v), kv, k_cache, v_cache)
        o = torch.empty_like(q)
        work = torch.empty(G.attention_work_size(dense(q), k_cache, v_cache, kv), dtype=torch.uint8, device=device)
        G.attention(dense(q), k_cache, v_cache, kv, dense(o), 1.0 / math.sqrt(d), self.window, self.sinks, work.data_ptr(),
                    work.numel())
        out = self._f8("o", o.view(n, -1))
        G.add_rms_norm(dense(total), dense(out), dense(self.norms["out"]), dense(total), dense(y), EPS)

        logits = self._f8("vocabulary", y)
        lp, entropy = torch.empty(n, 1, device=device), torch.empty(n, device=device)
        ids, top = torch.empty(n, n_top, dtype=torch.int32, device=device), torch.empty(n, n_top, device=device)
        work = torch.empty(G.log_probs_work_size(dense(logits), n_top), dtype=torch.uint8, device=device)
        G.log_probs(dense(logits), dense(tokens), dense(lp), dense(entropy), dense(ids), dense(top), 1.0, work.data_ptr(),
                    work.numel())
        return logits, lp, entropy, ids, top


def build(device, hidden=1024, heads=16, kv_heads=4, head_size=64, vocabulary=5003, seed=0, **kw):
    g = torch.Generator().manual_seed(seed)

    def rows(out, k, spread=1.0):
        return (torch.randn(out, k, generator=g) * (spread / math.sqrt(k))).to(device)

    weights = {"q": rows(heads * head_size, hidden), "k": rows(kv_heads * head_size, hidden),
               "v": rows(kv_heads * head_size, hidden), "o": rows(hidden, heads * head_size),
               "vocabulary": rows(vocabulary, hidden, 2.0)}
    norms = {n: (1 + 0.1 * torch.randn(k, generator=g)).to(device)
             for n, k in (("in", hidden), ("out", hidden), ("q", head_size), ("k", head_size))}
    return AnswerStep(hidden, heads, kv_heads, head_size, weights, norms, **kw)


def main():
    device = torch.device("cuda:0")
    model = build(device)
    words = torch.randn(model.vocabulary, model.hidden, generator=torch.Generator().manual_seed(1)).to(device)
    prompts = [torch.arange(7, 44), torch.arange(100, 300)]
    told = torch.full((sum(len(p) for p in prompts), 1), -1, dtype=torch.int32, device=device)
    _, _, _, ids, _ = model.step(words[torch.cat(prompts).to(device)], model.describe([len(p) for p in prompts]), told, 5)
    last = torch.tensor([len(prompts[0]) - 1, -1])
    for _ in range(4):
        token = ids[last, 0]
        _, _, entropy, ids, top = model.step(words[token.long()], model.describe([1, 1]), told[:2], 5)
        last = torch.arange(2)
        print("tokens %s, entropy of the next %s nats, likeliest %s (log probabilities %s)" % (
            token.tolist(), ["%.2f" % e for e in entropy.tolist()], ids[:, 0].tolist(), ["%.2f" % t for t in top[:, 0].tolist()]))


if __name__ == "__main__":
    main()
