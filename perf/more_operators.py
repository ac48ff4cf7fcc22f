"""Performance cases of microscaled 4-bit tensors and of log probabilities: quantisation to blocks of
4-bit floats and back, products with such weights, the score of given tokens under such an output head,
and log probabilities, entropy, rank and top alternatives out of logits.

A microscaled row holds blocks of 32 values: each is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign, times
the block's power of two, 2^e: e = floor(log2(largest magnitude)) - 2 (rule "floor"; what then lies past 6
becomes 6) or the smallest e that no value of the block exceeds 6 2^e (rule "ceil").  Values are rounded to
the nearest, ties to the even code.
"""

import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one token's activations, as they are made ready for a product: all latency
        {"name": "quantize_token", "op": "quantize", "x": "f16", "rows": 1, "cols": 1024, "rule": "floor"},
        # a checkpoint's table
        {"name": "quantize_table", "op": "quantize", "x": "bf16", "rows": 151936, "cols": 1024, "rule": "ceil"},
        # one generated token through the q, k and v projections of a layer
        {"name": "linear_token", "op": "linear", "x": "bf16", "y": "bf16", "m": 1, "n": 4096, "k": 1024},
        # a step of 48 users through a layer's output projection
        {"name": "linear_batch", "op": "linear", "x": "f16", "y": "f32", "m": 48, "n": 1024, "k": 2048},
        # a prompt through the gate and up projections
        {"name": "linear_prompt", "op": "linear", "x": "bf16", "y": "bf16", "m": 2000, "n": 6144, "k": 1024},
        # a few proposed tokens with 4-bit activations
        {"name": "linear4_check", "op": "linear4", "x": "f16", "y": "f16", "m": 5, "n": 6144, "k": 1024},
        # a wide layer with 4-bit activations: all matrix rate
        {"name": "linear4_prompt", "op": "linear4", "x": "bf16", "y": "bf16", "m": 4096, "n": 8192, "k": 4096},
        # how likely an answer of 21 tokens is
        {"name": "score_answer", "op": "score", "x": "bf16", "m": 21, "n": 151936, "k": 1024},
        # the tokens of a whole prompt
        {"name": "score_prompt", "op": "score", "x": "f16", "m": 1999, "n": 151936, "k": 1024},
        # a generated token with its five best alternatives
        {"name": "logprobs_token", "op": "logprobs", "x": "f32", "rows": 1, "vocab": 151936, "pad": 0, "top": 5, "masked": 0.0},
        # a step of 64 users under a grammar that leaves half of the vocabulary
        {"name": "logprobs_batch", "op": "logprobs", "x": "f32", "rows": 64, "vocab": 151936, "pad": 0, "top": 20, "masked": 0.5},
        # a prompt's tokens, logits in rows padded to a multiple of 256
        {"name": "logprobs_prompt", "op": "logprobs", "x": "bf16", "rows": 1100, "vocab": 151669, "pad": 139, "top": 1, "masked": 0.0},
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    op = rng.choice(("quantize", "linear", "linear", "linear4", "linear4", "score", "logprobs", "logprobs"))
    if op == "quantize":
        cols = 32 * _log(rng, 1, 256)
        return {"op": op, "x": rng.choice(("f16", "bf16", "f32")), "rows": _log(rng, 1, 100_000_000 // cols), "cols": cols,
                "rule": rng.choice(("floor", "ceil"))}
    if op in ("linear", "linear4"):
        m, n, k = _log(rng, 1, 4096), _log(rng, 1, 16384), 32 * _log(rng, 1, 256)
        while m * n * k > 130_000_000_000:
            n = (n + 1) // 2
        x = rng.choice(("f16", "bf16"))
        return {"op": op, "x": x, "y": rng.choice((x, "f32")), "m": m, "n": n, "k": k}
    if op == "score":
        n, k = _log(rng, 100, 151936), 32 * _log(rng, 2, 128)
        return {"op": op, "x": rng.choice(("f16", "bf16")), "m": _log(rng, 1, max(1, min(2000, 300_000_000_000 // (n * k)))), "n": n, "k": k}
    vocab = _log(rng, 2, 262144)
    return {"op": op, "x": rng.choice(("f32", "f16", "bf16")), "rows": _log(rng, 1, min(4096, max(1, 100_000_000 // vocab))), "vocab": vocab,
            "pad": rng.choice((0, 0, rng.randrange(1, 300))), "top": rng.randrange(0, min(vocab, 32) + 1),
            "masked": rng.choice((0.0, 0.0, 0.3, 0.98))}


# ---------------------------------------------------------------- what a case holds
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _targets(g, rows, n):
    return torch.randint(0, n, (rows,), generator=g, device="cuda", dtype=torch.int32)


def prepare(case, seed):
    g, op, s = _gen(seed), case["op"], {"case": case}
    kind = DTYPES[case["x"]]
    if op == "quantize":
        # rows of unlike size, as a table's or a layer's activations are
        x = torch.empty(case["rows"], case["cols"], dtype=kind, device="cuda").normal_(generator=g)
        s["x"] = x.mul_((0.05 * _randn(g, case["rows"], 1).exp()).to(kind))
        return s
    if op == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.empty(rows, vocab + case["pad"], dtype=kind, device="cuda").normal_(generator=g).mul_(3)
        s["targets"] = _targets(g, rows, vocab)
        if case["masked"]:
            keep = x[torch.arange(rows, device="cuda"), s["targets"].long()].clone()
            for row in x.split(max(1, 50_000_000 // x.shape[1])):
                row[torch.rand(row.shape, generator=g, device="cuda") < case["masked"]] = -math.inf
            x[torch.arange(rows, device="cuda"), s["targets"].long()] = keep
        s["logits"] = x[:, :vocab]
        return s
    m, n, k = case["m"], case["n"], case["k"]
    s["x"] = _randn(g, m, k).to(kind)
    if op == "score":
        s["targets"] = _targets(g, m, n)
    # weights of a trained size, in blocks of unlike size; a user's program has them quantised
    w = torch.empty(n, k, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    w.mul_(((2.5 if op == "score" else 1.0) / math.sqrt(k) * (0.3 * _randn(g, n, 1)).exp()).to(torch.bfloat16))
    codes, e = _codes(w.float(), "floor")
    s["packed"] = (codes[:, 0::2] | codes[:, 1::2] << 4).to(torch.uint8)
    s["scale"] = (e + 127).to(torch.uint8)
    if own:
        from llm_accelerator_amd.mx import MXTensor
        s["w"] = MXTensor(s["packed"], s["scale"])
    return s


# ---------------------------------------------------------------- plain forms
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _codes(x, rule):
    """fp32 [rows, cols] -> (codes 0 .. 15, exponents of the blocks)."""
    rows, cols = x.shape
    b = x.view(rows, cols // 32, 32)
    mant, exp = torch.frexp(b.abs().amax(-1))  # mant 2^exp, 0.5 <= mant < 1
    e = exp - 3
    if rule == "ceil":
        e = e + (mant > 0.75).int()  # the largest lies past 6 2^(exp - 3)
    e = e.clamp(-127, 127)
    a = torch.ldexp(b, -e[..., None]).abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    v = (torch.round(a / step) * step).clamp(max=6.0)  # half to even
    code = torch.where(v < 2, 2 * v, torch.where(v < 4, v + 2, v / 2 + 4)).int()
    return (code | (b < 0).int() << 3).view(rows, cols), e


def _values(codes, e):
    """The fp32 values that codes and exponents stand for."""
    rows, cols = codes.shape
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    return torch.ldexp(level[codes.long()].view(rows, cols // 32, 32), e[..., None]).view(rows, cols)


def _weights(s):
    p = s["packed"].int()
    return _values(torch.stack((p & 15, p >> 4), -1).flatten(1), s["scale"].int() - 127)


def _quantize(s):
    case = s["case"]
    out = torch.empty_like(s["x"])
    step = max(1, 40_000_000 // case["cols"])
    for i in range(0, case["rows"], step):
        out[i:i + step] = _values(*_codes(s["x"][i:i + step].float(), case["rule"]))
    return {"values": out}


def _linear(s):
    x = s["x"].float()
    if s["case"]["op"] == "linear4":
        x = _values(*_codes(x, "floor"))
    return {"y": (x @ _weights(s).T).to(DTYPES[s["case"]["y"]])}


def _score(s):
    w, got = _weights(s), []
    for x, t in zip(s["x"].float().split(512), s["targets"].long().split(512)):
        z = x @ w.T
        z -= z.amax(-1, keepdim=True)
        total = z.exp().sum(-1)
        got.append((z.gather(1, t[:, None])[:, 0] - total.log(), total.log() - (z.exp() * z).sum(-1) / total, -total.log()))
    return {name: torch.cat(v) for name, v in zip(("logprob", "entropy", "best"), zip(*got))}


def _logprobs(s):
    top, got = s["case"]["top"], []
    for x, t in zip(s["logits"].split(256), s["targets"].long().split(256)):
        x = x.float()
        z = x - x.amax(-1, keepdim=True)
        p = z.exp()
        total = p.sum(-1, keepdim=True)
        z -= total.log()
        entropy = -(p / total * torch.where(p > 0, z, 0)).sum(-1)
        mine = x.gather(1, t[:, None])
        at = torch.arange(x.shape[1], device="cuda")
        rank = ((x > mine) | ((x == mine) & (at < t[:, None]))).sum(-1).int()
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top] if top else t[:, None][:, :0]
        got.append((z.gather(1, t[:, None])[:, 0], rank, entropy, z.gather(1, order), order.int()))
    return {name: torch.cat(v) for name, v in zip(("logprob", "rank", "entropy", "top_logprobs", "top_ids"), zip(*got))}


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"quantize": _quantize, "linear": _linear, "linear4": _linear, "score": _score, "logprobs": _logprobs}[op](s)
    from llm_accelerator_amd.logprobs import token_logprobs
    from llm_accelerator_amd.mx import mx_linear, mx_quantize, mx_score
    if op == "quantize":
        return {"values": mx_quantize(s["x"], rule=s["case"]["rule"]).dequantize(s["x"].dtype)}
    if op == "linear":
        return {"y": mx_linear(s["x"], s["w"], out_dtype=DTYPES[s["case"]["y"]])}
    if op == "linear4":
        return {"y": mx_linear(mx_quantize(s["x"]), s["w"], out_dtype=DTYPES[s["case"]["y"]])}
    if op == "score":
        got = mx_score(s["x"], s["w"], s["targets"])
        return {"logprob": got.logprob, "entropy": got.entropy, "best": got.best}
    got = token_logprobs(s["logits"], s["targets"], top=s["case"]["top"])
    return {"logprob": got.logprob, "rank": got.rank, "entropy": got.entropy, "top_logprobs": got.top_logprobs, "top_ids": got.top_ids}


# ---------------------------------------------------------------- the least work
def work(case):
    op, size = case["op"], DTYPES[case["x"]].itemsize
    if op == "quantize":
        count = case["rows"] * case["cols"]
        return {"bytes": count * (2 * size + 0.5 + 1 / 32), "flops": 0}  # in, the 4-bit form, the values out
    if op == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": rows * (vocab * size + 16 + 8 * case["top"]), "flops": 4 * rows * vocab}
    m, n, k = case["m"], case["n"], case["k"]
    held = m * k * size + n * k * (0.5 + 1 / 32)
    return {"bytes": held + (16 * m if op == "score" else m * n * DTYPES[case["y"]].itemsize), "flops": 2 * m * n * k}


# ---------------------------------------------------------------- the definition in 64 bits
def _nearest(x, rule):
    """Doubles [rows, cols] as microscaled values: of the eight magnitudes the nearest, of two as near the one of the even code."""
    level = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    out = torch.empty_like(x)
    for j in range(0, x.shape[1], 32):
        b = x[:, j:j + 32]
        most = b.abs().max(-1, keepdim=True).values
        lg = torch.log2(torch.where(most > 0, most, 1.0)).floor()
        lg = torch.where(torch.exp2(lg) > most, lg - 1, torch.where(torch.exp2(lg + 1) <= most, lg + 1, lg))  # log2 may be off by a rounding
        e = lg - 2
        if rule == "ceil":
            e = torch.where(6 * torch.exp2(e) < most, e + 1, e)
        scale = torch.exp2(e.clamp(-127, 127))
        a = b.abs() / scale
        hi = torch.searchsorted(level, a.contiguous()).clamp(max=7)
        lo = (hi - 1).clamp(min=0)
        up, down = (level[hi] - a).abs(), (a - level[lo]).abs()
        pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
        out[:, j:j + 32] = torch.copysign(level[pick] * scale, b)
    return out


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "quantize":
        return {"values": torch.cat([_nearest(x.double(), case["rule"]) for x in s["x"].split(max(1, 20_000_000 // case["cols"]))])}
    if op == "logprobs":
        names, parts = ("logprob", "entropy", "top_logprobs"), []
        for x, t in zip(s["logits"].split(128), s["targets"].long().split(128)):
            lp = torch.log_softmax(x.double(), -1)
            best = lp.topk(case["top"], -1).values if case["top"] else lp[:, :0]
            parts.append((lp[torch.arange(len(t), device="cuda"), t], -torch.special.xlogy(lp.exp(), lp.exp()).sum(-1), best))
        got = {name: torch.cat(v) for name, v in zip(names, zip(*parts))}
        return {"logprob": got["logprob"], "rank": None, "entropy": got["entropy"], "top_logprobs": got["top_logprobs"], "top_ids": None}
    # byte by byte out of a table of the two values that it holds
    signed = [v for half in (LEVELS, [-v for v in LEVELS]) for v in half]
    pairs = torch.tensor([(signed[i % 16], signed[i // 16]) for i in range(256)], dtype=torch.float64, device="cuda")
    # (some rows at a time: torch's indexing gave other rows' values past 2^30 bytes of output here)
    w = torch.cat([pairs[p.long()].flatten(1) * torch.exp2(e.double() - 127).repeat_interleave(32, 1)
                   for p, e in zip(s["packed"].split(4096), s["scale"].split(4096))])
    x = s["x"].double()
    if op == "linear4":
        x = _nearest(x, "floor")
    if op != "score":
        return {"y": x @ w.T}
    parts = []
    for x, t in zip(x.split(128), s["targets"].long().split(128)):
        lp = torch.log_softmax(x @ w.T, -1)
        parts.append((lp[torch.arange(len(t), device="cuda"), t], -(lp.exp() * lp).sum(-1), lp.max(-1).values))
    return {name: torch.cat(v) for name, v in zip(("logprob", "entropy", "best"), zip(*parts))}
