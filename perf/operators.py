"""What is measured of the operators around a quantized product in a decoder layer.

``norm``   the residual sum and its root-mean-square norm, written in the 8-bit
           records that the products take (or in 32 or 16 bits);
``cache``  new tokens' keys and values quantized into a paged cache, and the
           sequences read back from it;
``attend`` attention of new tokens over that cache: one token a sequence or a
           chunk, causal, with an optional sliding window beside first tokens
           that stay visible.

The cache is a pool of pages, (pages, kv heads, slots of a page, head values)
with the values of a head as GGML records; a sequence's pages come from a table
in any order.  Keys and values are N(0, 1), each key channel at a scale of its
own; the scores' spread is then about one, as trained heads have it.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
#: bytes of a record of 32 (q8_k: 256) values
RECORD = {"f32": 0, "f16": 0, "q4_0": 18, "q8_0": 34, "q8_1": 36, "q8_k": 292}
EPS = 1e-5


# ------------------------------------------------------------------ the cases
def listed():
    def norm(name, rows, k, dst):
        return {"name": name, "op": "norm", "rows": rows, "k": k, "dst": dst}

    def cache(name, kind, seqs, longest, new, page, kv_heads, d, src="f32", ragged=1):
        return {"name": name, "op": "cache", "kind": kind, "seqs": seqs, "longest": longest, "new": new, "page": page,
                "kv_heads": kv_heads, "d": d, "src": src, "ragged": ragged}

    def attend(name, kind, seqs, longest, new, page, heads, kv_heads, d, src="f32", window=0, sinks=0, ragged=1):
        return {"name": name, "op": "attend", "kind": kind, "seqs": seqs, "longest": longest, "new": new, "page": page,
                "heads": heads, "kv_heads": kv_heads, "d": d, "src": src, "window": window, "sinks": sinks,
                "ragged": ragged}

    return [
        # one token's row between two products of a decode step (their batch-1 kernels quantize it themselves)
        norm("norm_decode_row", 1, 4096, "f32"),
        # a chunk of odd length in front of a Q4_0 or MXFP4 product
        norm("norm_chunk_q8_0", 509, 11008, "q8_0"),
        # a long prefill in front of a K-quant product: the largest
        norm("norm_prefill_q8_k", 16384, 8192, "q8_k"),
        # one step of a chat that has just begun
        cache("cache_one_token", "q8_0", 1, 131, 1, 16, 8, 128),
        # four prompts that are stored whole, the smallest records
        cache("cache_prompts_q4_0", "q4_0", 4, 2048, 2048, 64, 8, 128, ragged=3),
        # a full batch's decode step and the transfer of its caches to a program that wants plain values
        cache("cache_batch_read", "q8_0", 32, 16384, 1, 64, 8, 128, ragged=5),
        # decode: a short chat, one user
        attend("decode_short", "q8_0", 1, 1023, 1, 16, 32, 8, 128),
        # decode: a server's batch of uneven chats
        attend("decode_batch", "q8_0", 48, 8192, 1, 64, 32, 8, 128, ragged=7),
        # decode: one user deep in a long document, the cache in 4 bits
        attend("decode_long_q4_0", "q4_0", 1, 131072, 1, 256, 32, 8, 128),
        # a whole prompt on an empty cache in 16 bits
        attend("prefill_prompt_f16", "f16", 1, 4096, 4096, 64, 32, 8, 128, src="f16"),
        # a chunk late in a long context, each head with a window and four sinks
        attend("chunk_window_sinks", "q8_0", 1, 32768, 512, 64, 64, 8, 64, window=4096, sinks=4),
        # chunked prefill beside decodes in one batch, a head size between powers of two, no shared heads
        attend("mixed_batch_d96", "q4_0", 9, 3001, 640, 32, 16, 16, 96, ragged=11),
    ]


def draw(rng):
    """A case of the same ranges: sizes spread over their logarithm, odd ones among them."""
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    top = {}
    for c in listed():
        w = work(c)
        top[c["op"]] = [max(a, b) for a, b in zip(top.get(c["op"], (0, 0)), (w["bytes"], w["flops"]))]
    while True:
        op = rng.choice(["norm", "cache", "attend", "attend"])
        if op == "norm":
            dst = rng.choice(["f32", "f16", "q8_0", "q8_1", "q8_k"])
            c = {"op": op, "rows": log(1, 16384), "k": 256 * log(1, 64) if dst == "q8_k" else 32 * log(4, 512),
                 "dst": dst}
        else:
            new = rng.choice([1, 1, log(2, 4096)]) if op == "attend" else rng.choice([1, log(2, 4096)])
            seqs = log(1, 64)
            c = {"op": op, "kind": rng.choice(["f16", "q8_0", "q4_0"]), "seqs": seqs,
                 "longest": max(new, log(16, 131072 if new == 1 else 32768)), "new": new,
                 "page": rng.choice([16, 24, 32, 64, 256]), "kv_heads": rng.choice([1, 2, 4, 8, 16]),
                 "d": rng.choice([64, 96, 128, 128, 256]), "src": rng.choice(["f32", "f16"]),
                 "ragged": rng.randrange(1, 1 << 30)}
            if op == "attend":
                c["heads"] = c["kv_heads"] * rng.choice([1, 2, 4, 5, 8])
                c["window"] = rng.choice([0, 0, log(16, 8192)])
                c["sinks"] = rng.choice([0, 4, log(1, 64)]) if c["window"] else 0
                # the plain form keeps every score
                if seqs * c["heads"] * new * c["longest"] > 1 << 30:
                    continue
            if seqs * c["longest"] * c["kv_heads"] * c["d"] > 1 << 29:
                continue
        if 3072 in c.values():  # no width or length of this framework's workloads
            continue
        w = work(c)
        if w["bytes"] <= top[op][0] and w["flops"] <= max(1, top[op][1]):
            return c


def lengths_of(case):
    """([cache length], [new tokens]) of a case's sequences; the first is the longest."""
    r = random.Random(case["ragged"])
    ls, ns = [], []
    for i in range(case["seqs"]):
        n = case["new"] if i == 0 or case["new"] == 1 else r.randint(1, case["new"])
        ls.append(case["longest"] if i == 0 else max(n, r.randint((case["longest"] + 3) // 4, case["longest"])))
        ns.append(n)
    return ls, ns


def row_bytes(kind, n):
    if kind in ("f32", "f16"):
        return n * (4 if kind == "f32" else 2)
    return RECORD[kind] * (n // (256 if kind == "q8_k" else 32))


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["k"]
        return {"bytes": 12.0 * n + 4.0 * case["k"] + case["rows"] * row_bytes(case["dst"], case["k"]), "flops": 5.0 * n}
    ls, ns = lengths_of(case)
    kv = 2 * case["kv_heads"] * row_bytes(case["kind"], case["d"])  # a token's keys and values
    src = 4 if case["src"] == "f32" else 2
    if case["op"] == "cache":
        values = 2 * case["kv_heads"] * case["d"]
        # the new rows are read, written as records, and with the rest read back as 16-bit values
        return {"bytes": float(sum(ns) * (values * src + kv) + sum(ls) * (kv + 2 * values)), "flops": float(sum(ns) * values)}
    pairs = keys = 0
    for n_keys, n in zip(ls, ns):
        first = n_keys - n
        w, s = case["window"], case["sinks"]
        if not w:
            pairs += n * first + n * (n + 1) // 2
            keys += n_keys
        else:
            for p in range(first, n_keys):
                lo = max(0, p - w + 1)
                pairs += p + 1 - lo + min(s, lo)
            lo = max(0, first - w + 1)
            keys += n_keys - lo + min(s, lo)
    q = sum(ns) * case["heads"] * case["d"]
    return {"bytes": float(keys * kv + q * (src + 2)), "flops": 4.0 * pairs * case["heads"] * case["d"]}


# ------------------------------------------------------------- GGML's records
def first_largest(b):
    """The value of largest magnitude in each block, the first where several are."""
    a = b.abs()
    at = torch.arange(b.shape[-1], device=b.device)
    first = torch.where(a == a.amax(-1, keepdim=True), at, b.shape[-1]).amin(-1, keepdim=True)
    return torch.gather(b, -1, first.clamp_max(b.shape[-1] - 1))


def reciprocal(d):
    return torch.where(d != 0, 1.0 / torch.where(d != 0, d, torch.ones_like(d)), torch.zeros_like(d))


def half_away(t):
    whole = t.trunc()
    return torch.where((t - whole).abs() == 0.5, whole + t.sign(), t.round())


def codes_q8_0(x):
    """(scale in 32 bits, codes) of blocks of 32."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    d = b.abs().amax(-1, keepdim=True) / 127.0
    return d, half_away(b * reciprocal(d))


def codes_q4_0(x):
    b = x.reshape(*x.shape[:-1], -1, 32)
    d = first_largest(b) / -8.0
    return d, (b * reciprocal(d) + 8.5).trunc().clamp_max(15)


def codes_q8_k(x):
    b = x.reshape(*x.shape[:-1], -1, 256)
    top = first_largest(b)
    some = top != 0
    scale = torch.where(some, -127.0 / torch.where(some, top, torch.ones_like(top)), torch.zeros_like(top))
    return reciprocal(scale), (b * scale).round().clamp_max(127)


def to_records(x, kind):
    """The rows of x (..., n) as a cache of that kind holds them: bytes, or 16-bit values."""
    if kind == "f16":
        return x.half()
    if kind == "q8_0":
        d, q = codes_q8_0(x.float())
        body = q.to(torch.int8).view(torch.uint8)
    else:
        d, q = codes_q4_0(x.float())
        q = q.to(torch.uint8)
        body = q[..., :16] | (q[..., 16:] << 4)
    return torch.cat([d.half().view(torch.uint8), body], -1).flatten(-2)


def from_records(r, kind):
    """Their values in 32 bits."""
    if kind == "f16":
        return r.float()
    b = r.reshape(*r.shape[:-1], -1, RECORD[kind])
    d = b[..., :2].contiguous().view(torch.float16).float()
    if kind == "q8_0":
        q = b[..., 2:].view(torch.int8).float()
    else:
        q = torch.cat([b[..., 2:] & 15, b[..., 2:] >> 4], -1).float() - 8.0
    return (d * q).flatten(-2)


# ---------------------------------------------------------------- the inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    s = {"case": case, "op": case["op"]}
    if case["op"] == "norm":
        rows, k, dst = case["rows"], case["k"], case["dst"]
        s["x"], s["residual"] = normal(rows, k), normal(rows, k) * 3.0
        s["weight"] = 1.0 + 0.1 * normal(k)
        s["total"] = torch.empty(rows, k, device=DEV)
        if RECORD[dst]:
            s["y"] = torch.empty(rows, row_bytes(dst, k), dtype=torch.uint8, device=DEV)
        else:
            s["y"] = torch.empty(rows, k, dtype=torch.float32 if dst == "f32" else torch.float16, device=DEV)
        if dst == "q8_k":
            s["sums"] = torch.empty(rows, k // 256, 16, dtype=torch.float16, device=DEV)
        s["values"] = torch.empty(rows, k, dtype=torch.float16, device=DEV)
    else:
        ls, ns = lengths_of(case)
        page, kind, kvh, d = case["page"], case["kind"], case["kv_heads"], case["d"]
        width = -(-max(ls) // page)
        used = [-(-n // page) for n in ls]
        order = torch.randperm(sum(used) + 2, generator=torch.Generator().manual_seed(int(seed))).tolist()
        table = torch.full((len(ls), width), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(used):
            table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        s["pages"] = table.to(DEV)
        s["starts"] = torch.tensor([sum(ns[:i]) for i in range(len(ns) + 1)], dtype=torch.int32).to(DEV)
        s["lengths"] = torch.tensor(ls, dtype=torch.int32).to(DEV)
        s["longest"], s["new"], s["tokens"] = max(ls), max(ns), sum(ns)
        spread = 0.5 + torch.rand(d, generator=g, device=DEV)
        src = torch.float32 if case["src"] == "f32" else torch.float16
        for name, scale in (("k", spread), ("v", 1.0)):
            pool = torch.empty(len(order), kvh, page, row_bytes(kind, d) // (2 if kind == "f16" else 1),
                               dtype=torch.float16 if kind == "f16" else torch.uint8, device=DEV)
            step = max(1, (1 << 25) // (kvh * page * d))
            for p in range(0, len(order), step):
                pool[p:p + step] = to_records(normal(min(step, len(order) - p), kvh, page, d) * scale, kind)
            s[name + "_cache"] = pool
            if case["op"] == "cache":
                s[name + "_new"] = (normal(sum(ns), kvh, d) * scale).to(src)
                s[name + "_out"] = torch.empty(len(ls), max(ls), kvh, d, dtype=torch.float16, device=DEV)
        if case["op"] == "attend":
            s["q"] = normal(sum(ns), case["heads"], d).to(src)
            s["out"] = torch.empty(sum(ns), case["heads"], d, dtype=torch.float16, device=DEV)
    if own:
        s["plan"] = plan(s)
    return s


def plan(s):
    """The descriptors (and the work buffer) that a program keeps beside its buffers."""
    from weft_amd import ggml as G

    t = {"f32": G.F32, "f16": G.F16, "q4_0": G.Q4_0, "q8_0": G.Q8_0, "q8_1": G.Q8_1, "q8_k": G.Q8_K,
         torch.float32: G.F32, torch.float16: G.F16, torch.int32: G.I32}
    case = s["case"]

    def dense(x):
        return G.tensor(t[x.dtype], tuple(reversed(x.shape)), x.data_ptr())

    if s["op"] == "norm":
        y = G.tensor(t[case["dst"]], (case["k"], case["rows"]), s["y"].data_ptr())
        return [dense(s[n]) for n in ("x", "residual", "weight", "total")] + [y]
    batch = G.kv_batch(dense(s["pages"]), dense(s["starts"]), dense(s["lengths"]))
    pools = [G.tensor(t[case["kind"]], (case["d"], case["page"], case["kv_heads"], s[n].shape[0]), s[n].data_ptr())
             for n in ("k_cache", "v_cache")]
    if s["op"] == "cache":
        return [dense(s[n]) for n in ("k_new", "v_new")] + pools + [batch] + [dense(s[n]) for n in ("k_out", "v_out")]
    q, out = dense(s["q"]), dense(s["out"])
    size = G.attention_work_size(q, pools[0], pools[1], batch)
    s["work"] = torch.empty(max(size, 16), dtype=torch.uint8, device=DEV)
    return [q] + pools + [batch, out, size]


# --------------------------------------------------------------- the operators
def run(s):
    if own:
        return run_own(s)
    if s["op"] == "norm":
        return plain_norm(s)
    return plain_cache(s) if s["op"] == "cache" else plain_attend(s)


def run_own(s):
    from weft_amd import _lib, ggml as G

    _lib.set_stream(torch.cuda.current_stream().cuda_stream)
    case, p = s["case"], s["plan"]
    if s["op"] == "norm":
        G.add_rms_norm(p[0], p[1], p[2], p[3], p[4], EPS)
        return norm_values(s)
    if s["op"] == "cache":
        G.kv_write(p[0], p[1], p[4], p[2], p[3])
        G.kv_read(p[2], p[3], p[4], p[5], p[6])
        return {"k": s["k_out"], "v": s["v_out"]}
    G.attention(p[0], p[1], p[2], p[3], p[4], 1.0 / math.sqrt(case["d"]), case["window"], case["sinks"],
                s["work"].data_ptr(), p[5])
    return s["out"]


def norm_values(s):
    """The sum, and what the records in y stand for (in 16 bits, as they are read)."""
    dst, y = s["case"]["dst"], s["y"]
    if not RECORD[dst]:
        return {"total": s["total"], "y": y}
    rows = y.shape[0]
    if dst == "q8_k":
        d = y.view(torch.float32).view(rows, -1, 73)[..., :1]
        q = y.view(torch.int8).view(rows, -1, 292)[..., 4:260]
        torch.mul(q, d, out=s["values"].view(q.shape))
        torch.mul(y.view(torch.int16).view(rows, -1, 146)[..., 130:], d, out=s["sums"])
        return {"total": s["total"], "y": s["values"], "sums": s["sums"]}
    h = y.view(torch.float16).view(rows, -1, RECORD[dst] // 2)
    q = y.view(torch.int8).view(rows, -1, RECORD[dst])[..., RECORD[dst] - 32:]
    torch.mul(q, h[..., :1], out=s["values"].view(q.shape))
    out = {"total": s["total"], "y": s["values"]}
    if dst == "q8_1":
        out["sums"] = h[..., 1]
    return out


def plain_norm(s):
    dst = s["case"]["dst"]
    total = s["x"] + s["residual"]
    y = total * torch.rsqrt((total * total).mean(-1, keepdim=True) + EPS) * s["weight"]
    out = {"total": total}
    if dst == "f32":
        out["y"] = y
    elif dst == "f16":
        out["y"] = y.half()
    elif dst == "q8_k":
        d, q = codes_q8_k(y)
        out["y"] = (d * q).half().flatten(-2)
        out["sums"] = (d * q.unflatten(-1, (16, 16)).sum(-1)).half()
    else:
        d, q = codes_q8_0(y)
        out["y"] = (d.half() * q).half().flatten(-2)
        if dst == "q8_1":
            out["sums"] = (d * q.sum(-1, keepdim=True)).half().squeeze(-1)
    return out


def places(s):
    """(sequence, position in it, index among its new tokens) of each new token."""
    token = torch.arange(s["tokens"], device=DEV)
    seq = (token[:, None] >= s["starts"][None, 1:]).sum(1)
    index = token - s["starts"][seq]
    count = s["starts"][1:] - s["starts"][:-1]
    return seq, s["lengths"][seq] - count[seq] + index, index


def gather(s, name):
    """A pool's sequences as (sequences, longest, kv heads, values) in 32 bits, zeros past their lengths."""
    page = s["case"]["page"]
    at = torch.arange(s["longest"], device=DEV)
    there = at[None, :] < s["lengths"][:, None]
    p = torch.where(there, s["pages"][:, at // page], 0).long()
    rows = s[name][p, :, (at % page)[None, :].expand_as(p)]
    values = from_records(rows, s["case"]["kind"])
    return torch.where(there[:, :, None, None], values, 0.0), there


def plain_cache(s):
    kind, page = s["case"]["kind"], s["case"]["page"]
    seq, pos, _ = places(s)
    p = s["pages"][seq, pos // page].long()
    s["k_cache"][p, :, pos % page] = to_records(s["k_new"], kind)
    s["v_cache"][p, :, pos % page] = to_records(s["v_new"], kind)
    return {"k": gather(s, "k_cache")[0].half(), "v": gather(s, "v_cache")[0].half()}


def plain_attend(s):
    case = s["case"]
    kvh, d = case["kv_heads"], case["d"]
    share = case["heads"] // kvh
    k, there = gather(s, "k_cache")
    v, _ = gather(s, "v_cache")
    seqs, longest = there.shape
    seq, pos, index = places(s)
    q = torch.zeros(seqs, s["new"], case["heads"], d, device=DEV)
    q[seq, index] = s["q"].float() * (1.0 / math.sqrt(d))
    q = q.view(seqs, s["new"], kvh, share, d).permute(0, 2, 1, 3, 4).reshape(seqs, kvh, s["new"] * share, d)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(seqs, kvh, s["new"], share, longest)
    # visible: at most the token's own position, and inside its window or among the sinks
    at = torch.arange(longest, device=DEV)
    own_pos = torch.full((seqs, s["new"]), -1, device=DEV, dtype=pos.dtype)
    own_pos[seq, index] = pos
    seen = at <= own_pos[..., None]
    if case["window"]:
        seen = seen & ((at > own_pos[..., None] - case["window"]) | (at < case["sinks"]))
    seen = (seen & there[:, None, :])[:, None, :, None, :]
    scores = torch.where(seen, scores, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -torch.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(seqs, kvh, s["new"] * share, longest), v.permute(0, 2, 1, 3).contiguous())
    out = out.view(seqs, kvh, s["new"], share, d) / torch.where(total > 0, total, 1.0)
    return out.permute(0, 2, 1, 3, 4).reshape(seqs, s["new"], case["heads"], d)[seq, index].half()


# ------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s["x"].double() + s["residual"].double()
        y = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / case["k"] + EPS) * s["weight"].double()
        dst = case["dst"]
        if dst in ("f32", "f16"):
            return {"total": x, "y": y}
        size = 256 if dst == "q8_k" else 32
        b = y.view(case["rows"], -1, size)
        if dst == "q8_k":
            low, high = b.amin(-1, keepdim=True), b.amax(-1, keepdim=True)
            step = torch.where(high >= -low, high, low) / -127.0
            step32 = step
        else:
            step = b.abs().amax(-1, keepdim=True) / 127.0
            step32 = step.half().double()
        q = torch.round(b / step)
        out = {"total": x, "y": (q * step32).view(case["rows"], -1)}
        if dst == "q8_k":
            out["sums"] = q.view(case["rows"], -1, 16, 16).sum(-1) * step32
        elif dst == "q8_1":
            out["sums"] = q.sum(-1) * step[..., 0]
        return out
    kind, page, kvh, d = case["kind"], case["page"], case["kv_heads"], case["d"]
    ls, ns = lengths_of(case)
    pages = s["pages"].tolist()

    def stored(name, i):
        """A sequence's rows (length, kv heads, values) in 64 bits."""
        rows = torch.cat([s[name][p].transpose(0, 1) for p in pages[i][:-(-ls[i] // page)]])[:ls[i]]
        if kind == "f16":
            return rows.double()
        rec = rows.view(ls[i], kvh, d // 32, RECORD[kind])
        step = rec[..., 0:2].contiguous().view(torch.float16).double()
        if kind == "q8_0":
            return (step * rec[..., 2:34].contiguous().view(torch.int8).double()).flatten(2)
        nibbles = rec[..., 2:18].to(torch.int16)
        return (step * (torch.cat([nibbles % 16, nibbles // 16], 3) - 8).double()).flatten(2)

    if case["op"] == "cache":
        out, at = {}, 0
        for name in ("k", "v"):
            out[name] = torch.zeros(len(ls), max(ls), kvh, d, dtype=torch.float64, device=DEV)
        for i, (length, n) in enumerate(zip(ls, ns)):
            for name in ("k", "v"):
                out[name][i, :length] = stored(name + "_cache", i)
                x = s[name + "_new"][at:at + n].double()
                if kind != "f16":
                    b = x.view(n, kvh, d // 32, 32)
                    if kind == "q8_0":
                        step = b.abs().amax(-1, keepdim=True) / 127
                        x = (torch.round(b / step) * step.half().double()).flatten(2)
                    else:
                        low, high = b.amin(-1, keepdim=True), b.amax(-1, keepdim=True)
                        step = torch.where(high > -low, high, low) / -8
                        x = ((torch.floor(b / step + 8.5).clamp_max(15) - 8) * step.half().double()).flatten(2)
                out[name][i, length - n:length] = x
            at += n
        return out
    share = case["heads"] // kvh
    out = torch.zeros(sum(ns), case["heads"], d, dtype=torch.float64, device=DEV)
    at = 0
    for i, (length, n) in enumerate(zip(ls, ns)):
        k, v = stored("k_cache", i), stored("v_cache", i)
        own_pos = torch.arange(length - n, length, device=DEV)[:, None]
        key = torch.arange(length, device=DEV)[None, :]
        hidden = key > own_pos
        if case["window"]:
            hidden = hidden | ((own_pos - key >= case["window"]) & (key >= case["sinks"]))
        for h in range(case["heads"]):
            sc = s["q"][at:at + n, h].double() @ k[:, h // share].T / math.sqrt(d)
            sc = sc.masked_fill(hidden, -math.inf)
            out[at:at + n, h] = torch.softmax(sc, 1) @ v[:, h // share]
        at += n
    return out
