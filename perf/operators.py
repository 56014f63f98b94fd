"""What the low-bit operators are measured on: the cache held in 4 bits (append and attention) and the
product in 8-bit integers.

    append   s1kv.Batch.append into a pool of dtype "q4", and the rows read back as the cache holds them
    attend   s1kv.Batch.attention over such a pool: decode rows, prompt chunks over cached prefixes, prompts
    product  s1kv.matmul_w8a8 / matmul_w8a8_group: tokens quantised, 8-bit product, one scale a token and channel

The 4-bit format.  A row is the D values of one token and KV head, lo and hi its least and greatest value:

    m = bf16(fp32((7 lo + 8 hi) / 15))                         (both roundings to nearest even)
    s = fp32(max((hi - m) / 7, (m - lo) / 8)), rounded up to bf16
    code = 8 + the integer nearest to (x - m) / s, ties to even, 8 where s = 0: 0 .. 15
    value = fp32(m + s (code - 8))

The 8-bit tokens: s = fp32(max |x| / 127), 1 for a row of zeros; code = the integer nearest to x / s, ties to even.

`own` False: plain torch operations.  `own` True: the framework's calls.
"""
import math
import os
import random
import sys

import torch

own = False

BLOCK = 16  # tokens a block of the cache


def _s1kv():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "s1-infer_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import s1kv
    return s1kv


# ------------------------------------------------------------------- cases --

def listed():
    return [
        # one decode step of 64 sequences: a token each, 8 KV heads of 128
        {"name": "append step", "op": "append", "seqs": 64, "low": 1, "high": 1, "kv": 8, "dim": 128, "mix": 1},
        # the prompts of a step, ragged
        {"name": "append prompts", "op": "append", "seqs": 5, "low": 1000, "high": 6000, "kv": 8, "dim": 128, "mix": 2},
        # small heads and an odd number of them
        {"name": "append small heads", "op": "append", "seqs": 37, "low": 1, "high": 301, "kv": 3, "dim": 64, "mix": 3},
        # one short conversation, 16 query heads on 8 KV heads: latency
        {"name": "decode one", "op": "attend", "seqs": 1, "low": 777, "high": 777, "qlow": 1, "qhigh": 1, "heads": 16, "kv": 8, "dim": 128, "mix": 4},
        # a serving batch, 32 query heads on 8 KV heads, ragged contexts
        {"name": "decode batch", "op": "attend", "seqs": 64, "low": 300, "high": 8192, "qlow": 1, "qhigh": 1, "heads": 32, "kv": 8, "dim": 128, "mix": 5},
        # two long documents, 64 query heads on 8 KV heads
        {"name": "decode long", "op": "attend", "seqs": 2, "low": 100001, "high": 131072, "qlow": 1, "qhigh": 1, "heads": 64, "kv": 8, "dim": 128, "mix": 6},
        # heads of 64, seven query heads on each KV head, contexts from one token
        {"name": "decode small heads", "op": "attend", "seqs": 33, "low": 1, "high": 2049, "qlow": 1, "qhigh": 1, "heads": 28, "kv": 4, "dim": 64, "mix": 7},
        # new turns over cached prefixes: ragged chunks
        {"name": "chunks", "op": "attend", "seqs": 12, "low": 1500, "high": 2500, "qlow": 37, "qhigh": 400, "heads": 32, "kv": 8, "dim": 128, "mix": 8},
        # one whole prompt from an empty cache
        {"name": "prompt", "op": "attend", "seqs": 1, "low": 4001, "high": 4001, "qlow": 4001, "qhigh": 4001, "heads": 32, "kv": 8, "dim": 128, "mix": 9},
        # q, k and v projections of one token
        {"name": "product token", "op": "product", "rows": 1, "k": 1024, "n": 2048, "n2": 1024, "n3": 1024},
        # the same of a decode batch, larger model
        {"name": "product step", "op": "product", "rows": 64, "k": 4096, "n": 4096, "n2": 1024, "n3": 1024},
        # an MLP projection of a long prompt, odd number of tokens
        {"name": "product prompt", "op": "product", "rows": 8001, "k": 4096, "n": 14336, "n2": 0, "n3": 0},
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    what = rng.choice(["append", "decode", "chunks", "product", "product"])
    dim, mix = rng.choice([64, 128, 128]), rng.randrange(1 << 30)
    if what == "append":
        seqs = _log(rng, 1, 64)
        high = _log(rng, 1, 24000 // seqs)
        return {"op": "append", "seqs": seqs, "low": rng.randint(1, high), "high": high, "kv": rng.choice([1, 2, 3, 4, 8]), "dim": dim, "mix": mix}
    kv = rng.choice([1, 2, 4, 8])
    if what == "decode":
        seqs = _log(rng, 1, 64)
        high = _log(rng, 1, min(131072, 262144 // seqs))
        return {"op": "attend", "seqs": seqs, "low": _log(rng, 1, high), "high": high, "qlow": 1, "qhigh": 1, "heads": kv * rng.choice([1, 2, 4, 7, 8]), "kv": kv, "dim": dim, "mix": mix}
    if what == "chunks":
        seqs = _log(rng, 1, 12)
        qhigh = _log(rng, 2, 4000 // seqs)
        high = qhigh + _log(rng, 1, 2500)
        return {"op": "attend", "seqs": seqs, "low": rng.randint(qhigh, high), "high": high, "qlow": rng.randint(1, qhigh), "qhigh": qhigh, "heads": kv * rng.choice([1, 2, 4]), "kv": kv, "dim": dim, "mix": mix}
    group = rng.random() < 0.4
    rows = _log(rng, 1, 8000)
    k, n = _log(rng, 256, 4096), _log(rng, 256, 8192)
    return {"op": "product", "rows": rows, "k": k, "n": n, "n2": _log(rng, 64, 2048) if group else 0, "n3": _log(rng, 64, 2048) if group else 0}


def _lengths(c):
    """(tokens, query rows) of each sequence; the first takes the longest of both."""
    r = random.Random(c["mix"])
    lens = [c["high"]] + [r.randint(c["low"], c["high"]) for _ in range(c["seqs"] - 1)]
    if c["op"] == "append":
        return lens, [0] * c["seqs"]
    rows = [c["qhigh"]] + [r.randint(c["qlow"], c["qhigh"]) for _ in range(c["seqs"] - 1)]
    return lens, [min(a, b) for a, b in zip(rows, lens)]


def work(c):
    if c["op"] == "product":
        n = c["n"] + c["n2"] + c["n3"]
        return {"bytes": 4 * c["rows"] * c["k"] + n * (c["k"] + 4) + 4 * c["rows"] * n, "flops": 2 * c["rows"] * c["k"] * n}
    lens, rows = _lengths(c)
    held = 2 * c["kv"] * (c["dim"] // 2 + 4)  # bytes a token
    if c["op"] == "append":  # fp32 in, the cache written and read back, fp32 out
        return {"bytes": sum(lens) * (2 * 8 * c["kv"] * c["dim"] + 2 * held), "flops": 2 * 10 * sum(lens) * c["kv"] * c["dim"]}
    seen = sum(r * (n - r) + r * (r + 1) // 2 for n, r in zip(lens, rows))
    return {"bytes": sum(lens) * held + sum(rows) * 8 * c["heads"] * c["dim"] + 4 * sum(-(-n // BLOCK) for n in lens),
            "flops": 4 * c["heads"] * c["dim"] * seen}


# ------------------------------------------------------------------ inputs --

def _normal(shape, gen):
    return torch.randn(shape, device="cuda", dtype=torch.float32, generator=gen)


def _inputs(c, seed):
    """What the seed alone makes: tokens' K and V (and queries), or rows and weights."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + 17)
    if c["op"] == "product":
        k = c["k"]
        x = _normal((c["rows"], k), gen)
        x *= 0.5 + 4.0 * torch.rand((1, k), device="cuda", generator=gen) ** 8  # a few large channels
        made = {"x": x, "w": []}
        for n in (c["n"], c["n2"], c["n3"]):
            if n:  # 8-bit weights, a row for each channel, rows padded with zeros to whole 16 bytes
                w = torch.zeros((n, -(-k // 16) * 16), dtype=torch.int8, device="cuda")
                w[:, :k] = (_normal((n, k), gen) * 36).round().clamp(-127, 127).to(torch.int8)
                made["w"].append((w, 1e-4 + 1e-3 * torch.rand((n,), device="cuda", generator=gen)))
        return made
    lens, rows = _lengths(c)
    total, shape = sum(lens), (sum(lens), c["kv"], c["dim"])
    k, v = _normal(shape, gen), _normal(shape, gen)
    k *= 0.5 + 2.5 * torch.rand((1,) + shape[1:], device="cuda", generator=gen) ** 6  # keys have channels that stand out
    v += 0.3 * _normal((1,) + shape[1:], gen)
    made = {"k": k, "v": v, "lens": lens, "rows": rows, "total": total}
    if c["op"] == "attend":
        made["q"] = _normal((sum(rows), c["heads"], c["dim"]), gen)
    blocks = sum(-(-n // BLOCK) for n in lens)
    made["blocks"] = blocks + 3
    made["order"] = random.Random(seed).sample(range(blocks + 3), blocks + 3)  # blocks lie where the allocator left them
    return made


def prepare(c, seed):
    s = _inputs(c, seed)
    s["case"] = c
    if c["op"] == "product":
        return s
    lens, rows = s["lens"], s["rows"]
    if own:
        # the cache of a running program: a pool, its sequences, and the step's batch, which serves every layer
        S = _s1kv()
        pool = S.Pool(1, c["kv"], c["dim"], s["blocks"], BLOCK, dtype="q4", max_seqs=c["seqs"], initial_free_list=s["order"])
        seqs = list(range(c["seqs"]))
        fill = pool.batch(seqs, lens, rows)
        if c["op"] == "attend":
            fill.append(0, s.pop("k"), s.pop("v"))
            fill.end()
            fill = pool.batch(seqs, None, rows)
        s["pool"], s["batch"] = pool, fill
        return s
    if c["op"] == "append":
        return s
    # the same cache in tensors: packed codes, two to a byte, their s and m, blocks in the same scattered order
    ids = list(reversed(s["order"]))
    table, width, t0 = [], -(-max(lens) // BLOCK), 0
    for n in lens:
        b = -(-n // BLOCK)
        table.append(ids[t0:t0 + b] + [0] * (width - b))
        t0 += b
    s["table"] = torch.tensor(table, device="cuda")
    s["lens_t"] = torch.tensor(lens, device="cuda")
    s["rows_t"] = torch.tensor(rows, device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), s["lens_t"])
    pos = torch.arange(s["total"], device="cuda") - (torch.cumsum(s["lens_t"], 0) - s["lens_t"])[seq]
    at = s["table"][seq, pos // BLOCK] * BLOCK + pos % BLOCK
    for name in ("k", "v"):
        code, scale, mid = _quantise(s.pop(name))
        code = code.to(torch.uint8)
        held = torch.zeros((s["blocks"] * BLOCK, c["kv"], c["dim"] // 2), dtype=torch.uint8, device="cuda")
        held[at] = code[..., 0::2] | (code[..., 1::2] << 4)
        params = torch.zeros((s["blocks"] * BLOCK, c["kv"], 2), dtype=torch.bfloat16, device="cuda")
        params[at] = torch.stack([scale, mid], -1)
        s[name + "_codes"], s[name + "_params"] = held, params
    s["row_seq"] = torch.repeat_interleave(torch.arange(len(rows), device="cuda"), s["rows_t"])
    s["row_at"] = torch.arange(sum(rows), device="cuda") - (torch.cumsum(s["rows_t"], 0) - s["rows_t"])[s["row_seq"]]
    return s


# ------------------------------------------------------------ plain forms --

def _quantise(x):
    """(codes 0 .. 15 as float, s, m as bfloat16) of the rows in x's last dimension; 64 bits, where values lie next to a border."""
    lo, hi = x.amin(-1).double(), x.amax(-1).double()
    m = ((7 * lo + 8 * hi) / 15).float().bfloat16()
    d = m.double()
    top = torch.maximum((hi - d) / 7, (d - lo) / 8).float()
    s = ((top.view(torch.int32) + 0xFFFF) & -65536).view(torch.float32).bfloat16()
    e = s.double()
    near = ((x.double() - d[..., None]) / torch.where(e > 0, e, torch.ones_like(e))[..., None]).round().clamp(-8, 7)
    return near.float() + 8, s, m


def _attend(s):
    c = s["case"]
    b, width = s["table"].shape
    kv, dim, heads = c["kv"], c["dim"], c["heads"]
    slots = (s["table"][:, :, None] * BLOCK + torch.arange(BLOCK, device="cuda")).reshape(b, width * BLOCK)

    def values(name):  # [b, kv, tokens, dim]
        code = s[name + "_codes"][slots]
        code = torch.stack([code & 15, code >> 4], -1).reshape(b, width * BLOCK, kv, dim).float() - 8
        p = s[name + "_params"][slots].float()
        return (p[..., 1:] + p[..., :1] * code).transpose(1, 2)

    most, g = c["qhigh"], heads // kv
    q = torch.zeros((b, most, heads, dim), device="cuda")
    q[s["row_seq"], s["row_at"]] = s["q"]
    q = q.reshape(b, most, kv, g, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, g * most, dim)
    x = (q @ values("k").transpose(2, 3)) / math.sqrt(dim)
    last = (s["lens_t"] - s["rows_t"])[:, None] + torch.arange(most, device="cuda")  # the last token that a row sees
    hidden = torch.arange(width * BLOCK, device="cuda") > last[:, :, None]
    hidden = hidden[:, None].expand(b, g, most, width * BLOCK).reshape(b, 1, g * most, width * BLOCK)
    x.masked_fill_(hidden, float("-inf"))
    x = torch.exp(x - x.amax(-1, keepdim=True))
    v = values("v").masked_fill((torch.arange(width * BLOCK, device="cuda") >= s["lens_t"][:, None])[:, None, :, None], 0)
    o = (x @ v) / x.sum(-1, keepdim=True)
    o = o.reshape(b, kv, g, most, dim).permute(0, 3, 1, 2, 4).reshape(b, most, heads, dim)
    return o[s["row_seq"], s["row_at"]]


def _product(s):
    x = s["x"]
    top = x.abs().amax(1, keepdim=True)
    scale = torch.where(top > 0, (top.double() / 127).float(), torch.ones_like(top))
    code = (x.double() / scale.double()).round()
    k = x.shape[1]
    # sums up to 127 * 127 * k pass 24 bits: 64-bit products
    return [((code @ w[:, :k].double().t()) * scale.double() * ws.double()).float() for w, ws in s["w"]]


def run(s):
    op = s["case"]["op"]
    if own:
        S = _s1kv()
        if op == "append":
            s["batch"].append(0, s["k"], s["v"])
            return s["batch"].gather(0, S.K), s["batch"].gather(0, S.V)
        if op == "attend":
            return s["batch"].attention(0, s["q"])
        weights = [S.ChannelQuantizedTensor(w, ws, s["x"].shape[1]) for w, ws in s["w"]]
        return S.matmul_w8a8_group(s["x"], weights)
    if op == "append":
        made = []
        for x in (s["k"], s["v"]):
            code, scale, mid = _quantise(x)
            made.append(mid.float()[..., None] + scale.float()[..., None] * (code - 8))
        return tuple(made)
    return _attend(s) if op == "attend" else _product(s)


# ---------------------------------------------------------------- in 64 bits --

def _held64(x):
    """The values that the 4-bit cache holds for the rows of x, from the format's definition."""
    x = x.to(torch.float64)
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    mid = (low * 7 + high * 8).div(15).to(torch.float32).to(torch.bfloat16).to(torch.float64)
    need = torch.maximum(high.sub(mid).div(7), mid.sub(low).div(8)).to(torch.float32)
    step = need.to(torch.bfloat16)  # to nearest; one bfloat16 further where that is below
    step = torch.where(step.to(torch.float32) < need, torch.nextafter(step, torch.full_like(step, float("inf"))), step).to(torch.float64)
    code = torch.where(step > 0, x.sub(mid).div(step), torch.zeros_like(x)).round().clamp(-8, 7)
    return mid + step * code


def exact(c, seed):
    s = _inputs(c, seed)
    if c["op"] == "append":
        return _held64(s["k"]), _held64(s["v"])
    if c["op"] == "product":
        x = s["x"].to(torch.float64)
        step = x.abs().max(1, keepdim=True).values.div(127).to(torch.float32).to(torch.float64)
        held = torch.where(step > 0, x.div(step), x).round() * step
        return [held @ (w[:, :c["k"]].to(torch.float64) * ws.to(torch.float64)[:, None]).T for w, ws in s["w"]]
    made, t0, r0, g = [], 0, 0, c["heads"] // c["kv"]
    for n, r in zip(s["lens"], s["rows"]):
        k, v = _held64(s["k"][t0:t0 + n]), _held64(s["v"][t0:t0 + n])
        q = s["q"][r0:r0 + r].to(torch.float64)
        t0, r0 = t0 + n, r0 + r
        after = torch.arange(n, device="cuda")[None] > (n - r + torch.arange(r, device="cuda"))[:, None]
        heads = []
        for h in range(c["heads"]):
            a = q[:, h] @ k[:, h // g].T * c["dim"] ** -0.5
            heads.append(torch.softmax(a.masked_fill(after, -math.inf), 1) @ v[:, h // g])
        made.append(torch.stack(heads, 1))
    return torch.cat(made)
