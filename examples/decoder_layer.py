"""The attention half of a decoder layer out of the library's operators:

    add_rms_norm -> mul_mat (q, k, v) -> kv_write -> attention -> mul_mat (o)

with Q4_K weights and a paged Q8_0 cache.  The norm adds the layer before's
output and writes the Q8_K records that the products take, so the activations are
quantized once and never read in 32 bits again.  Queries and keys are used as the
products give them; a model with rotary positions turns them before kv_write.

Run on a GPU: ``python -m examples.decoder_layer`` reads two prompts, decodes a
few tokens of both, and compares them with the same tokens read at once.
"""
from __future__ import annotations

import math

import torch

from weft_amd import _lib, ggml as G

EPS = 1e-5


class DecoderAttention:
    """total = x + delta, out = o(attention(q, k, v of norm(total))), for a batch of
    sequences whose new tokens' rows lie one sequence after the other; the next
    half layer takes (total, out) as its (x, delta)."""

    def __init__(self, hidden, heads, kv_heads, head_size, weights, norm, *, page_size=16, pages=64, max_seqs=8,
                 window=0, sinks=0):
        """weights: "q", "k", "v", "o" as Q4_K rows (out, bytes), uint8 on the GPU;
        norm: (hidden) float32."""
        self.hidden, self.heads, self.kv_heads, self.d = hidden, heads, kv_heads, head_size
        self.page_size, self.window, self.sinks = page_size, window, sinks
        self.weights, self.norm = weights, norm
        shape = (pages, kv_heads, page_size, G.row_size(G.Q8_0, head_size))
        self.k_cache = torch.zeros(shape, dtype=torch.uint8, device=norm.device)
        self.v_cache = torch.zeros_like(self.k_cache)
        self.free = list(range(pages))
        self.table = torch.full((max_seqs, pages), -1, dtype=torch.int32)
        self.lengths = [0] * max_seqs

    def _product(self, name, rows_out, src1, tokens, like):
        w = G.tensor(G.Q4_K, (src1.ne[0], rows_out), self.weights[name].data_ptr())
        y = torch.empty(tokens, rows_out, dtype=torch.float32, device=like.device)
        size = G.mul_mat_work_size(w, src1)  # 0 for records
        work = torch.empty(size, dtype=torch.uint8, device=like.device)
        G.mul_mat(w, src1, G.tensor(G.F32, (rows_out, tokens), y.data_ptr()), work.data_ptr(), size)
        return y

    def _batch(self, new, device):
        """Gives the new tokens pages and describes the batch; the tensors are kept
        by the caller until the work is done."""
        for s, n in enumerate(new):
            have, need = -(-self.lengths[s] // self.page_size), -(-(self.lengths[s] + n) // self.page_size)
            for i in range(have, need):
                self.table[s, i] = self.free.pop()
            self.lengths[s] += n
        seqs = len(new)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        longest = max(1, max(-(-x // self.page_size) for x in self.lengths[:seqs]))
        kept = (self.table[:seqs, :longest].contiguous().to(device),
                torch.tensor(starts, dtype=torch.int32).to(device),
                torch.tensor(self.lengths[:seqs], dtype=torch.int32).to(device))
        t = [G.tensor(G.I32, (*reversed(x.shape),), x.data_ptr()) for x in kept]
        return G.kv_batch(*t), kept

    def forward(self, x, delta, new):
        """x, delta (or None): (tokens, hidden) float32, new[s] rows of sequence s.
        Returns (total, out)."""
        _lib.set_stream(torch.cuda.current_stream().cuda_stream)
        tokens, hidden, d = x.shape[0], self.hidden, self.d
        batch, kept = self._batch(new, x.device)

        y = torch.empty(tokens, G.row_size(G.Q8_K, hidden), dtype=torch.uint8, device=x.device)
        records = G.tensor(G.Q8_K, (hidden, tokens), y.data_ptr())
        total = torch.empty_like(x)
        rows = (hidden, tokens)
        G.add_rms_norm(G.tensor(G.F32, rows, x.data_ptr()),
                       None if delta is None else G.tensor(G.F32, rows, delta.data_ptr()),
                       G.tensor(G.F32, (hidden,), self.norm.data_ptr()), G.tensor(G.F32, rows, total.data_ptr()),
                       records, EPS)
        q = self._product("q", self.heads * d, records, tokens, x)
        k = self._product("k", self.kv_heads * d, records, tokens, x)
        v = self._product("v", self.kv_heads * d, records, tokens, x)

        pool = (d, self.page_size, self.kv_heads, self.k_cache.shape[0])
        k_cache = G.tensor(G.Q8_0, pool, self.k_cache.data_ptr())
        v_cache = G.tensor(G.Q8_0, pool, self.v_cache.data_ptr())
        rows = (d, self.kv_heads, tokens)
        G.kv_write(G.tensor(G.F32, rows, k.data_ptr()), G.tensor(G.F32, rows, v.data_ptr()), batch, k_cache, v_cache)

        o = torch.empty(tokens, self.heads * d, dtype=torch.float32, device=x.device)
        queries = G.tensor(G.F32, (d, self.heads, tokens), q.data_ptr())
        size = G.attention_work_size(queries, k_cache, v_cache, batch)
        work = torch.empty(size, dtype=torch.uint8, device=x.device)
        G.attention(queries, k_cache, v_cache, batch, G.tensor(G.F32, (d, self.heads, tokens), o.data_ptr()),
                    1.0 / math.sqrt(d), self.window, self.sinks, work.data_ptr(), size)
        return total, self._product("o", hidden, G.tensor(G.F32, (self.heads * d, tokens), o.data_ptr()), tokens, x)


def random_weights(out, k, seed, device):
    """Q4_K rows of random codes: d (6-bit scale) code - dmin (6-bit min), with
    d and dmin such that the values have a variance of about 1 / k."""
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(0, 256, (out, k // 256, 144), dtype=torch.uint8, generator=g)
    step = 1.0 / (258 * math.sqrt(k))
    w[..., :4] = torch.tensor([step, 7.5 * step]).half().view(torch.uint8)
    return w.view(out, -1).to(device)


def build(device, hidden=1024, heads=16, kv_heads=4, head_size=64, seed=0, **kw):
    weights = {"q": random_weights(heads * head_size, hidden, seed, device),
               "k": random_weights(kv_heads * head_size, hidden, seed + 1, device),
               "v": random_weights(kv_heads * head_size, hidden, seed + 2, device),
               "o": random_weights(hidden, heads * head_size, seed + 3, device)}
    norm = torch.ones(hidden, device=device)
    return DecoderAttention(hidden, heads, kv_heads, head_size, weights, norm, **kw)


def decoded_and_at_once(layer, other, x, prompts):
    """Outputs of the tokens after each prompt: decoded one by one, and read with it."""
    steps = len(x[0]) - prompts[0]
    layer.forward(torch.cat([a[:n] for a, n in zip(x, prompts)]), None, prompts)
    y = torch.stack([layer.forward(torch.stack([a[n + i] for a, n in zip(x, prompts)]), None, [1] * len(x))[1]
                     for i in range(steps)], 1)
    whole = other.forward(torch.cat(x), None, [len(a) for a in x])[1].split([len(a) for a in x])
    return y, torch.stack([w[n:] for w, n in zip(whole, prompts)])


def main():
    device = torch.device("cuda:0")
    prompts, steps = (37, 200), 4
    x = [torch.randn(n + steps, 1024, generator=torch.Generator().manual_seed(n)).to(device) for n in prompts]
    a, b = decoded_and_at_once(build(device), build(device), x, prompts)
    for s, n in enumerate(prompts):
        print("prompt of %d tokens: the next %d, decoded, differ from those read at once by %.1e of their size"
              % (n, steps, ((a[s] - b[s]).norm() / b[s].norm()).item()))


if __name__ == "__main__":
    main()
