"""What is measured of the operators that take a decoder step from 8-bit float products to an answer.

``quantize``  rows or weight blocks as 8-bit floats (e4m3) with a 32-bit scale for
              each 128 values of a row, or for each block of 128 x 128 weights;
``product``   the product of such weights with activations, which come as plain rows
              (quantized within the call) or with their scales;
``rotate``    the norm of each query and key head and the rotation by its token's
              position, between those products and the cache;
``choose``    what a step answers with: the log probabilities of given tokens, the
              entropy of each row of logits and its top alternatives.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-6
BLOCK = 128
#: the largest e4m3 value, and the smallest magnitude that a scale is made from
TOP, LEAST = 448.0, 2.0 ** -100
TYPES = {"f32": torch.float32, "f16": torch.float16, "f8": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "f8": 1}


# ------------------------------------------------------------------ the cases
def listed():
    def quantize(name, rows, k, src, blocks):
        return {"name": name, "op": "quantize", "rows": rows, "k": k, "src": src, "blocks": blocks}

    def product(name, m, n, k, src, dst):
        return {"name": name, "op": "product", "m": m, "n": n, "k": k, "src": src, "dst": dst}

    def rotate(name, tokens, heads, kv_heads, d, n_rot, neighbours, src, dst, base, first, factors=False):
        return {"name": name, "op": "rotate", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "d": d,
                "n_rot": n_rot, "neighbours": neighbours, "src": src, "dst": dst, "base": base, "first": first,
                "factors": factors}

    def choose(name, rows, v, given, top, src, scale=1.0):
        return {"name": name, "op": "choose", "rows": rows, "v": v, "given": given, "top": top, "src": src,
                "scale": scale}

    return [
        # a long prompt's activations, once for the products that share them
        quantize("quantize_prompt", 2048, 11008, "f16", False),
        # a checkpoint's weights as they are loaded; rows that no block divides
        quantize("quantize_weights", 11008, 4101, "f32", True),
        # decode: one token through one projection, where latency counts
        product("product_row", 1, 4096, 4096, "f32", "f32"),
        # decode: a server's batch through an up projection
        product("product_batch", 24, 11008, 4096, "f32", "f32"),
        # a short prompt through a down projection of odd width
        product("product_prompt", 509, 4101, 11008, "f16", "f16"),
        # a long prefill, its activations quantized before: the largest
        product("product_prefill", 8192, 8192, 8192, "f8", "f16"),
        # one step of a chat
        rotate("rotate_token", 1, 32, 8, 128, 128, False, "f32", "f16", 10000.0, 1023),
        # a batch deep in long documents, part of each head turned, pairs of neighbours, stretched frequencies
        rotate("rotate_batch_far", 48, 16, 16, 96, 64, True, "f32", "f32", 500000.0, 1000003, True),
        # a long prefill in 16 bits
        rotate("rotate_prefill", 16384, 64, 8, 128, 128, False, "f16", "f16", 10000.0, 0),
        # one step of a chat: the token and five alternatives
        choose("choose_token", 1, 32000, 1, 5, "f32"),
        # a server's batch with a large vocabulary, at a temperature
        choose("choose_batch", 48, 131072, 4, 20, "f32", 1.25),
        # the perplexity of a document, 16-bit logits of an odd vocabulary
        choose("choose_document", 4096, 50021, 1, 0, "f16"),
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
        op = rng.choice(["quantize", "product", "product", "product", "rotate", "rotate", "choose", "choose"])
        if op == "quantize":
            c = {"op": op, "rows": log(1, 16384), "k": rng.choice([log(1, 16384), 16 * log(1, 1024)]),
                 "src": rng.choice(["f32", "f16"]), "blocks": rng.choice([False, True])}
        elif op == "product":
            c = {"op": op, "m": log(1, 8192), "n": rng.choice([log(1, 16384), 128 * log(1, 128)]),
                 "k": rng.choice([log(1, 16384), 128 * log(1, 128), 128 * log(1, 128)]),
                 "src": rng.choice(["f32", "f16", "f8"]), "dst": rng.choice(["f32", "f16"])}
        elif op == "rotate":
            d = rng.choice([64, 80, 96, 128, 128, 192, 256])
            kv_heads = rng.choice([1, 2, 4, 8, 16])
            c = {"op": op, "tokens": log(1, 16384), "heads": kv_heads * rng.choice([1, 2, 4, 5, 8]),
                 "kv_heads": kv_heads, "d": d, "n_rot": rng.choice([d, d, d // 2, 2 * rng.randint(1, d // 2)]),
                 "neighbours": rng.choice([False, True]), "src": rng.choice(["f32", "f16"]),
                 "dst": rng.choice(["f32", "f16"]), "base": rng.choice([10000.0, 500000.0, 1000000.0]),
                 "first": rng.choice([0, log(1, 1 << 21)]), "factors": rng.choice([False, False, True])}
        else:
            v = log(2, 262144)
            c = {"op": op, "rows": log(1, 4096), "v": v, "given": rng.choice([0, 1, 1, log(1, 16)]),
                 "top": min(v, rng.choice([0, 1, 5, 20, log(1, 64)])), "src": rng.choice(["f32", "f16"]),
                 "scale": rng.choice([1.0, 1.0, 0.5, 1.25])}
            # the plain form sorts whole rows
            if c["top"] and c["rows"] * v > 1 << 27:
                continue
        w = work(c)
        if w["bytes"] <= top[op][0] and w["flops"] <= top[op][1]:
            return c


def up(n):
    return -(-n // BLOCK)


def work(case):
    if case["op"] == "quantize":
        n = case["rows"] * case["k"]
        scales = up(case["k"]) * (up(case["rows"]) if case["blocks"] else case["rows"])
        return {"bytes": n * (SIZE[case["src"]] + 1.0) + 4.0 * scales, "flops": 3.0 * n}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        x = m * k * SIZE[case["src"]] + (4 * m * up(k) if case["src"] == "f8" else 0)
        return {"bytes": float(n * k + 4 * up(n) * up(k) + x + m * n * SIZE[case["dst"]]), "flops": 2.0 * m * n * k}
    if case["op"] == "rotate":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["d"]
        more = 8.0 * case["d"] + 4.0 * case["tokens"] + (2.0 * case["n_rot"] if case["factors"] else 0)
        return {"bytes": n * (SIZE[case["src"]] + SIZE[case["dst"]]) + more, "flops": 7.0 * n}
    n = case["rows"] * case["v"]
    return {"bytes": n * float(SIZE[case["src"]]) + case["rows"] * (4.0 + 8.0 * (case["given"] + case["top"])),
            "flops": 5.0 * n}


# --------------------------------------------------------- 8-bit floats in blocks
def blocks_of(x, rows):
    """x (r, k) as (r blocks, rows, k blocks, 128), zeros past its ends."""
    r, k = x.shape
    wide = torch.nn.functional.pad(x, (0, up(k) * BLOCK - k, 0, -(-r // rows) * rows - r))
    return wide.view(-1, rows, up(k), BLOCK)


def to_f8(x, rows):
    """(codes (r, k), scales (r blocks, k blocks)), one scale for each ``rows`` x 128 values."""
    b = blocks_of(x.float(), rows)
    most = b.abs().amax((1, 3)).clamp_min(LEAST)
    top = torch.full_like(most, TOP)
    codes = (b * torch.div(top, most)[:, None, :, None]).to(torch.float8_e4m3fn)
    return codes.view(b.shape[0] * rows, -1)[:x.shape[0], :x.shape[1]].contiguous(), torch.div(most, top)


def from_f8(codes, scales, rows):
    """Their values in 32 bits, (r, k)."""
    b = blocks_of(codes.float(), rows) * scales[:, None, :, None]
    return b.view(b.shape[0] * rows, -1)[:codes.shape[0], :codes.shape[1]]


# ---------------------------------------------------------------- the inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def empty(kind, *shape):
        return torch.empty(*shape, dtype=TYPES[kind], device=DEV)

    def rows(r, k):
        # channels of uneven size, as activations have them
        return normal(r, k) * torch.exp(0.7 * normal(k))

    s = {"case": case}
    if case["op"] == "quantize":
        r, k = case["rows"], case["k"]
        s["x"] = (normal(r, k) * 0.02 if case["blocks"] else rows(r, k)).to(TYPES[case["src"]])
        s["codes"] = empty("f8", r, k)
        s["scales"] = empty("f32", up(r) if case["blocks"] else r, up(k))
    elif case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        s["w"], s["w_scales"] = to_f8(normal(n, k) * (0.02 * torch.exp(0.3 * normal(n)))[:, None], BLOCK)
        x = rows(m, k)
        if case["src"] == "f8":
            s["x"], s["x_scales"] = to_f8(x, 1)
        else:
            s["x"] = x.to(TYPES[case["src"]])
        s["y"] = empty(case["dst"], m, n)
    elif case["op"] == "rotate":
        t, d, src = case["tokens"], case["d"], TYPES[case["src"]]
        for name, heads in (("q", case["heads"]), ("k", case["kv_heads"])):
            s[name] = normal(t, heads, d).mul_(3.0).to(src)
            s[name + "_weight"] = 1.0 + 0.1 * normal(d)
            s[name + "_out"] = empty(case["dst"], t, heads, d)
        s["positions"] = torch.arange(case["first"], case["first"] + t, device=DEV, dtype=torch.int32)
        if case["factors"]:
            s["factors"] = 1.0 + 7.0 * torch.rand(case["n_rot"] // 2, generator=g, device=DEV)
    else:
        r, v = case["rows"], case["v"]
        x = normal(r, v) * 2.5
        if v > 100:  # words that a grammar bars
            x.scatter_(1, torch.randint(0, v, (r, v // 50), generator=g, device=DEV), -math.inf)
        # the token that the step took, and others asked for
        s["tokens"] = torch.randint(0, v, (r, case["given"]), generator=g, device=DEV, dtype=torch.int32)
        if case["given"]:
            x.scatter_(1, s["tokens"][:, :1].long(), 9.0 + normal(r, 1))
        s["logits"] = x.to(TYPES[case["src"]])
        s["token_lp"] = empty("f32", r, case["given"])
        s["entropy"] = empty("f32", r)
        s["top_ids"] = torch.empty(r, case["top"], dtype=torch.int32, device=DEV)
        s["top_lp"] = empty("f32", r, case["top"])
    if own:
        s["plan"] = plan(s)
    return s


def plan(s):
    """The descriptors (and the work buffer) that a program keeps beside its buffers."""
    from weft_amd import ggml as G

    case = s["case"]
    t = {torch.float32: G.F32, torch.float16: G.F16, torch.int32: G.I32, torch.float8_e4m3fn: G.F8_E4M3}

    def dense(name):
        x = s.get(name)
        return None if x is None or x.numel() == 0 else G.tensor(t[x.dtype], tuple(reversed(x.shape)), x.data_ptr())

    def workspace(size):
        s["work"] = torch.empty(size, dtype=torch.uint8, device=DEV)
        return s["work"].data_ptr(), size

    if case["op"] == "quantize":
        return [dense(n) for n in ("x", "codes", "scales")]
    if case["op"] == "product":
        p = [dense(n) for n in ("w", "w_scales", "x", "x_scales", "y")]
        return [*p, *workspace(G.mul_mat_f8_work_size(p[0], p[2]))]
    if case["op"] == "rotate":
        how = G.head_rope(n_rot=case["n_rot"], neighbours=case["neighbours"], base=case["base"])
        return [*(dense(n) for n in ("q", "k", "q_out", "k_out", "positions")), how,
                *(dense(n) for n in ("q_weight", "k_weight", "factors"))]
    p = [dense(n) for n in ("logits", "tokens", "token_lp", "entropy", "top_ids", "top_lp")]
    return [*p, case["scale"], *workspace(G.log_probs_work_size(p[0], case["top"]))]


# --------------------------------------------------------------- the operators
def run(s):
    op = s["case"]["op"]
    if own:
        return run_own(s, op)
    return {"quantize": plain_quantize, "product": plain_product, "rotate": plain_rotate, "choose": plain_choose}[op](s)


def run_own(s, op):
    from weft_amd import _lib, ggml as G

    _lib.set_stream(torch.cuda.current_stream().cuda_stream)
    p = s["plan"]
    if op == "quantize":
        G.quantize_f8(*p)
        return {"codes": s["codes"], "scales": s["scales"]}
    if op == "product":
        G.mul_mat_f8(*p)
        return s["y"]
    if op == "rotate":
        q, k, q_out, k_out, positions, how, q_weight, k_weight, factors = p
        G.head_norm_rope(q, k, q_out, k_out, positions, how, EPS, q_weight, k_weight, factors)
        return {"q": s["q_out"], "k": s["k_out"]}
    G.log_probs(*p)
    return {n: s[n] for n in ("token_lp", "entropy", "top_ids", "top_lp")}


def plain_quantize(s):
    codes, scales = to_f8(s["x"], BLOCK if s["case"]["blocks"] else 1)
    return {"codes": codes, "scales": scales}


def plain_product(s):
    x, x_scales = (s["x"], s["x_scales"]) if s["case"]["src"] == "f8" else to_f8(s["x"], 1)
    y = torch.matmul(from_f8(x, x_scales, 1), from_f8(s["w"], s["w_scales"], BLOCK).T)
    return y.to(TYPES[s["case"]["dst"]])


def plain_rotate(s):
    case = s["case"]
    n = case["n_rot"]
    i = torch.arange(n // 2, device=DEV, dtype=torch.float64)
    speed = torch.pow(torch.full_like(i, case["base"]), -2.0 * i / n)
    if case["factors"]:
        speed = speed / s["factors"].double()
    angle = s["positions"].double()[:, None] * speed
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turn(x, weight):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
        r, rest = x[..., :n], x[..., n:]
        if case["neighbours"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        else:
            a, b = r[..., :n // 2], r[..., n // 2:]
            r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        return torch.cat([r, rest], -1).to(TYPES[case["dst"]])

    return {"q": turn(s["q"], s["q_weight"]), "k": turn(s["k"], s["k_weight"])}


def plain_choose(s):
    case = s["case"]
    x = s["logits"].float()
    d = (x - x.amax(-1, keepdim=True)) * case["scale"]
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    out = {"entropy": (torch.where(e > 0, e * (log_total - d), 0.0).sum(-1, keepdim=True) / total).squeeze(-1),
           "token_lp": torch.gather(d, 1, s["tokens"].long()) - log_total}
    if case["top"]:
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
    else:
        ids = torch.empty(case["rows"], 0, dtype=torch.int64, device=DEV)
    out["top_ids"], out["top_lp"] = ids.int(), torch.gather(d, 1, ids) - log_total
    return out


# ------------------------------------------------------ the definition in 64 bits
def nearest_f8(v):
    """The nearest e4m3 values, halfway cases to the even code: three bits past the leading one, steps of 2^-9 at least."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def exact(case, seed):
    s = prepare(case, seed)

    def quantized(x, rows):
        """Codes and scales in 64 bits; the factor and its product are those that 32 bits give, so that codes are the same."""
        r, k = x.shape
        wide = torch.zeros(-(-r // rows) * rows, up(k) * BLOCK, dtype=torch.float64, device=DEV)
        wide[:r, :k] = x.double()
        wide = wide.view(-1, rows, up(k), BLOCK)
        most = torch.maximum(wide.amax((1, 3)), -wide.amin((1, 3))).clamp_min(LEAST)
        factor = (TOP / most).float().double()[:, None, :, None]
        return nearest_f8((wide * factor).float().double()), most / TOP

    if case["op"] == "quantize":
        codes, scales = quantized(s["x"], BLOCK if case["blocks"] else 1)
        r, k = case["rows"], case["k"]
        return {"codes": codes.view(-1, up(k) * BLOCK)[:r, :k], "scales": scales}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        w = s["w"].double() * s["w_scales"].double().repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
        if case["src"] == "f8":
            x = s["x"].double() * s["x_scales"].double().repeat_interleave(BLOCK, 1)[:, :k]
        else:
            codes, scales = quantized(s["x"], 1)
            x = (codes * scales.float().double()[:, None, :, None]).view(m, -1)[:, :k]
        return x @ w.T
    if case["op"] == "rotate":
        n, d = case["n_rot"], case["d"]
        out = {}
        for name in ("q", "k"):
            x = s[name].double()
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / d + EPS) * s[name + "_weight"].double()
            out[name] = x.clone()
            for i in range(n // 2):
                angle = s["positions"].double() * math.exp(-2 * i / n * math.log(case["base"]))
                if case["factors"]:
                    angle = angle / s["factors"][i].double()
                a, b = (2 * i, 2 * i + 1) if case["neighbours"] else (i, i + n // 2)
                z = torch.polar(torch.ones_like(angle), angle)[:, None] * torch.complex(x[..., a], x[..., b])
                out[name][..., a], out[name][..., b] = z.real, z.imag
        return out
    x = s["logits"].double() * case["scale"]
    lp = torch.log_softmax(x, -1)
    p = lp.exp()
    return {"entropy": -torch.where(p > 0, p * lp, 0.0).sum(-1), "token_lp": torch.gather(lp, 1, s["tokens"].long()),
            "top_ids": None, "top_lp": torch.topk(lp, case["top"], dim=-1).values}
