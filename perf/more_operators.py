"""The operators of a 4-bit KV cache and of beam search whose speed and exactness are measured.

  store    K and V of a step's or a prompt's rows into a cache of 4-bit values
           (ops.kv_update_fp4), and the same rows read back (ops.kv_read_fp4).
  attend   causal attention of packed rows on such a cache: single tokens, drafted
           tokens, prompts (ops.fp4_attention).
  select   the best continuations of each request's beams (ops.beam_select).
  reorder  the caches of all layers after a selection: every beam takes the rows of
           the beam that it goes on from (ops.kv_reorder).

A 4-bit cache here is one layer's slice: values [rows][kv heads][head dim / 2] bytes,
two e2m1 values each, the first in the low half, and scales [rows][kv heads][head dim /
32] bytes, one for each block of 32 values: byte b stands for 2^(b - 127). A sequence's
positions lie in consecutive rows from its row base on. Head layouts and vocabularies
are those of the Llama-3-8B, Llama-2-7B and tiny models of the benchmark and tests, and
generic ones.
"""
from __future__ import annotations

import math
import random

import torch

own = False   # False: plain torch operations; True: the framework's operators

DEV = "cuda:0"
DTYPES = {"f16": torch.float16, "f32": torch.float32}


# ---- cases ---------------------------------------------------------------------

def listed():
    return [
        # one decode step of a batch: the launches are what counts
        {"name": "store_step", "op": "store", "rows": 32, "kv_heads": 8, "hd": 128, "in": "f32", "out": "f16",
         "max_seq": 2048, "mix": 1},
        # the packed prompts of several requests
        {"name": "store_prompts", "op": "store", "rows": 8192, "kv_heads": 8, "hd": 128, "in": "f16", "out": "f16",
         "max_seq": 4096, "mix": 2},
        # three short prompts on the tiny model, the reference's types
        {"name": "attend_tiny", "op": "attend", "seqs": 3, "least": 1, "most": 13, "context": 0, "heads": 4,
         "kv_heads": 2, "hd": 64, "type": "f32", "mix": 3},
        # a decode step of one request with a long context, binary32 rows as the decode step has them
        {"name": "attend_one", "op": "attend", "seqs": 1, "least": 1, "most": 1, "context": 8191, "heads": 32,
         "kv_heads": 8, "hd": 128, "type": "f32", "mix": 4},
        # a decode step of 64 requests, contexts of a few hundred positions to 8000
        {"name": "attend_batch", "op": "attend", "seqs": 64, "least": 1, "most": 1, "context": 8000, "heads": 32,
         "kv_heads": 8, "hd": 128, "type": "f16", "mix": 5},
        # drafted tokens of 16 requests, every head with its own K and V
        {"name": "attend_drafts", "op": "attend", "seqs": 16, "least": 5, "most": 5, "context": 2500, "heads": 32,
         "kv_heads": 32, "hd": 128, "type": "f32", "mix": 6},
        # chat prompts of 20 requests, from a word to a page
        {"name": "attend_chats", "op": "attend", "seqs": 20, "least": 3, "most": 611, "context": 0, "heads": 32,
         "kv_heads": 8, "hd": 128, "type": "f16", "mix": 7},
        # one long document
        {"name": "attend_long", "op": "attend", "seqs": 1, "least": 6000, "most": 6000, "context": 0, "heads": 32,
         "kv_heads": 8, "hd": 128, "type": "f16", "mix": 8},
        # one request of four beams
        {"name": "select_one", "op": "select", "batch": 1, "beams": 4, "vocab": 128256, "n": 8, "first": False, "mix": 9},
        # sixteen requests of eight beams
        {"name": "select_batch", "op": "select", "batch": 16, "beams": 8, "vocab": 128256, "n": 16, "first": False,
         "mix": 10},
        # four beams of one request in all layers of the Llama-2-7B model
        {"name": "reorder_one", "op": "reorder", "groups": 1, "beams": 4, "layers": 32, "max_seq": 512, "most": 200,
         "kv_heads": 32, "hd": 128, "kv": "f16", "mix": 11},
        # eight requests of eight beams in all layers of the Llama-3-8B model
        {"name": "reorder_batch", "op": "reorder", "groups": 8, "beams": 8, "layers": 32, "max_seq": 300, "most": 300,
         "kv_heads": 8, "hd": 128, "kv": "f16", "mix": 12},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    heads, kv_heads, hd = rng.choice([(32, 8, 128), (32, 32, 128), (4, 2, 64), (24, 8, 64), (16, 1, 128), (40, 8, 128)])
    mix = rng.randrange(100, 1 << 30)
    op = rng.choice(["store", "attend", "attend", "attend", "select", "reorder"])
    if op == "store":
        rows = _log(rng, 1, 8000 * 8 // max(8, kv_heads))
        return {"op": op, "rows": rows, "kv_heads": kv_heads, "hd": hd, "in": rng.choice(["f16", "f32"]),
                "out": rng.choice(["f16", "f32"]), "max_seq": _log(rng, 64, 4096), "mix": mix}
    if op == "select":
        beams = _log(rng, 1, 16)
        return {"op": op, "batch": _log(rng, 1, 128 // beams), "beams": beams, "vocab": _log(rng, 500, 128256),
                "n": rng.choice([beams, 2 * beams]), "first": rng.random() < 0.15, "mix": mix}
    if op == "reorder":
        beams, layers = _log(rng, 2, 16), _log(rng, 1, 32)
        most = _log(rng, 1, 300)
        groups = _log(rng, 1, max(1, 8 * 8 * 32 * 8 * 128 // (beams * layers * kv_heads * hd)))
        return {"op": op, "groups": min(64, groups), "beams": beams, "layers": layers, "max_seq": most + rng.randrange(50),
                "most": most, "kv_heads": kv_heads, "hd": hd, "kv": "f16", "mix": mix}
    typ = rng.choice(["f16", "f32"])
    case = {"op": op, "heads": heads, "kv_heads": kv_heads, "hd": hd, "type": typ, "mix": mix}
    if rng.random() < 0.6:   # decode steps and drafted tokens
        seqs = _log(rng, 1, 64)
        rows = rng.choice([1, 1, 1, rng.randint(2, 8)])
        return {**case, "seqs": seqs, "least": rows, "most": rows,
                "context": _log(rng, 1, min(16000, 500000 // seqs) * 8 // max(8, kv_heads))}
    seqs = _log(rng, 1, 32)
    most = _log(rng, 1, 4000 // seqs)
    return {**case, "seqs": seqs, "least": max(1, most // 20), "most": most,
            "context": rng.choice([0, _log(rng, 1, 4000 // seqs + 64)])}


def _attend_sizes(case):
    """(rows, context before them) of each sequence; one has the most rows, one the longest context."""
    rng = random.Random(case["mix"])
    rows = [rng.randint(case["least"], case["most"]) for _ in range(case["seqs"])]
    rows[rng.randrange(len(rows))] = case["most"]
    ctx = [rng.randint(case["context"] // 20, case["context"]) for _ in rows]
    ctx[rng.randrange(len(ctx))] = case["context"]
    return rows, ctx


def _reorder_plan(case):
    """Positions of each group, and for each of its beams the one that it goes on from."""
    rng = random.Random(case["mix"])
    lens = [rng.randint(case["most"] // 4, case["most"]) for _ in range(case["groups"])]
    lens[rng.randrange(len(lens))] = case["most"]
    return lens, [[rng.randrange(case["beams"]) for _ in range(case["beams"])] for _ in lens]


# ---- inputs --------------------------------------------------------------------

def _rand(gen, shape, dtype, sigma=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * sigma).to(dtype)


def _index(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _places(case):
    """Row bases and positions of a "store" case's rows: runs of rows that follow
    each other in a sequence (prompts), or single ones (a decode step)."""
    rng = random.Random(case["mix"])
    rows, cap = case["rows"], case["max_seq"]
    base, pos = [], []
    while len(base) < rows:
        n = 1 if rows <= 64 else min(rows - len(base), rng.randint(1, cap))
        first = rng.randint(0, cap - n)
        slot = len(pos) and max(base) // cap + 1
        base += [slot * cap] * n
        pos += range(first, first + n)
    return base, pos


def _inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "select":
        rows = case["batch"] * case["beams"]
        logits = _rand(gen, (rows, case["vocab"]), torch.float32, 3.0)
        logits[:, -40:] = -math.inf   # tokens that the model does not use
        if case["first"]:   # all beams start alike: only the first counts
            scores = torch.full((case["batch"], case["beams"]), -math.inf, device=DEV)
            scores[:, 0] = 0
        else:
            scores = -20 - 2 * torch.rand(case["batch"], case["beams"], generator=gen, device=DEV)
        n = (case["batch"], case["n"])
        return {"logits": logits, "scores": scores, "out": torch.empty(n, device=DEV),
                "parents": torch.empty(n, dtype=torch.int32, device=DEV),
                "tokens": torch.empty(n, dtype=torch.int32, device=DEV)}
    kvh, hd = case["kv_heads"], case["hd"]
    if case["op"] == "reorder":
        lens, parents = _reorder_plan(case)
        beams, cap = case["beams"], case["max_seq"]
        slots = list(range(len(lens) * beams))
        random.Random(case["mix"] + 1).shuffle(slots)
        shape = (case["layers"], len(slots) * cap, kvh, hd)
        return {"k": _rand(gen, shape, DTYPES[case["kv"]]), "v": _rand(gen, shape, DTYPES[case["kv"]]),
                "base": _index([s * cap for s in slots]), "lens": _index([n for n in lens for _ in range(beams)]),
                "parents": _index([p for row in parents for p in row])}
    if case["op"] == "store":
        base, pos = _places(case)
        total = max(base) + case["max_seq"]
        kv = _rand(gen, (case["rows"], 2 * kvh, hd), DTYPES[case["in"]], 1.5)   # the end of a fused product's rows
        kv = kv * torch.exp(_rand(gen, (1, 2 * kvh, hd), kv.dtype))             # some channels are larger than others
        caches = {name: torch.zeros(total, kvh, hd // d, dtype=torch.uint8, device=DEV)
                  for name, d in (("kc", 2), ("ks", 32), ("vc", 2), ("vs", 32))}
        out = torch.empty(2, case["rows"], kvh, hd, dtype=DTYPES[case["out"]], device=DEV)
        return {"k": kv[:, :kvh], "v": kv[:, kvh:], **caches, "base": _index(base), "pos": _index(pos),
                "rows": _index([b + p for b, p in zip(base, pos)]), "k_out": out[0], "v_out": out[1]}
    rows, ctx = _attend_sizes(case)
    lens = [r + c for r, c in zip(rows, ctx)]
    cap = max(lens)
    slots = list(range(len(rows)))
    random.Random(case["mix"] + 1).shuffle(slots)
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    got = {"start": _index(starts), "lens": _index(lens), "base": _index([s * cap for s in slots]), "cap": cap,
           "most_rows": max(rows), "q": _rand(gen, (starts[-1], case["heads"], hd), DTYPES[case["type"]], 1.5)}
    for name in "kv":
        parts = [_pack(_rand(gen, (min(16384, len(rows) * cap - r), kvh, hd), torch.float32))
                 for r in range(0, len(rows) * cap, 16384)]
        got[name + "c"], got[name + "s"] = (torch.cat([p[i] for p in parts]) for i in (0, 1))
    got["out"] = torch.zeros_like(got["q"])
    return got


_engine = None


def prepare(case, seed):
    global _engine
    if own and _engine is None:
        from janus_amd import ops
        _engine = ops.ComputeEngine(0)
    return {"case": case, **_inputs(case, seed)}


# ---- the operators ---------------------------------------------------------------

def _pack(x):
    """x [rows, kv heads, hd] as (values, scales) in bytes. A block's scale 2^e: e =
    floor(log2 max) - 2, one more where max is above 7/8 of the next power of two,
    within [-23, 13]; a block with an infinity or NaN has scale byte 255. Values go to the
    nearest e2m1 value (0, 0.5, 1, 1.5, 2, 3, 4, 6), ties to the even code."""
    rows, kvh, hd = x.shape
    x = x.float().reshape(rows, kvh, hd // 32, 32)
    top = x.abs().amax(-1, keepdim=True)
    odd = ~torch.isfinite(x).all(-1, keepdim=True)
    m, e = torch.frexp(top.masked_fill(odd, 1.0))
    e = (e - 3 + (m > 0.875).int()).clamp(-23, 13).masked_fill(top == 0, -23)
    y = torch.ldexp(x.abs(), -e)
    code = (y > 0.25).byte() + (y >= 0.75).byte() + (y > 1.25).byte() + (y >= 1.75).byte() + (y > 2.5).byte() \
        + (y >= 3.5).byte() + (y > 5).byte() + 8 * torch.signbit(x).byte()
    code = code.masked_fill(odd, 0).view(rows, kvh, hd // 2, 2)
    return code[..., 0] | code[..., 1] << 4, (e + 127).masked_fill(odd, 255).byte().view(rows, kvh, hd // 32)


def _values(codes, scales):
    """The values that such bytes stand for, in 32 bits."""
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=DEV)
    levels = torch.cat([levels, -levels])
    code = torch.stack([codes & 15, codes >> 4], -1).int()
    x = levels[code].view(*scales.shape, 32)
    scale = torch.exp2(scales.float().clamp(min=104) - 127).masked_fill(scales > 140, math.nan)
    return (x * scale[..., None]).view(*codes.shape[:2], -1)


def _plain_store(s):
    at = s["base"].long() + s["pos"].long()
    for name in "kv":
        s[name + "c"][at], s[name + "s"][at] = _pack(s[name])
        s[name + "_out"][:] = _values(s[name + "c"][at], s[name + "s"][at]).to(s[name + "_out"].dtype)
    return {"k": s["k_out"], "v": s["v_out"]}


def _plain_attend(s):
    q, lens, start = s["q"], s["lens"].long(), s["start"].long()
    rows, heads, hd = q.shape
    kvh = s["kc"].shape[1]
    rep = heads // kvh
    count = start[1:] - start[:-1]
    b, n, cap = len(lens), s["most_rows"], s["cap"]
    i = torch.arange(n, device=DEV)
    j = torch.arange(cap, device=DEV)
    there = i[None] < count[:, None]
    at = torch.where(there, start[:-1, None] + i[None], rows)
    kv_at = s["base"].long()[:, None] + j[None]
    seen = j[None, None] < (lens[:, None] - count[:, None] + i[None] + 1)[..., None]            # [b, n, cap]
    k = _values(s["kc"], s["ks"])[kv_at].permute(0, 2, 3, 1).contiguous()
    v = _values(s["vc"], s["vs"])[kv_at].permute(0, 2, 1, 3).contiguous()
    qs = q[at.clamp(max=rows - 1)].float().view(b, n, kvh, rep, hd).permute(0, 2, 1, 3, 4).reshape(b, kvh, n * rep, hd)
    score = (torch.matmul(qs, k) * (1.0 / math.sqrt(hd))).view(b, kvh, n, rep, cap)
    score = score.masked_fill(~seen[:, None, :, None, :], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, kvh, n * rep, cap), v).view(b, kvh, n, rep, hd) / total.clamp(min=1e-30)
    whole = torch.empty(rows + 1, heads, hd, dtype=q.dtype, device=DEV)
    whole[at] = out.permute(0, 2, 1, 3, 4).reshape(b, n, heads, hd).to(q.dtype)
    return whole[:rows]


def _plain_select(s):
    case = s["case"]
    n, vocab = case["n"], case["vocab"]
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    logp = x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True)))
    value = (s["scores"].double().view(-1, 1) + logp).view(case["batch"], -1)
    # the n best, ties to the lowest index: those above the n-th value, and the first ones equal to it
    best, at = value.topk(n, -1)
    last = best[:, -1:]
    far = value.shape[1]
    index = torch.arange(far, device=DEV, dtype=torch.int32)
    equal = torch.where(value == last, index, far).topk(n, -1, largest=False).values
    at = torch.cat([torch.where(best > last, at, far), equal], -1).sort(-1).values
    found = value.gather(1, at.clamp(max=far - 1)).masked_fill(at == far, -math.inf)
    found, order = found.sort(stable=True, dim=-1, descending=True)
    at = at.gather(1, order)[:, :n]
    return {"scores": found[:, :n].float(), "parents": (at // vocab).int(), "tokens": (at % vocab).int()}


def _plain_reorder(s):
    case = s["case"]
    beams = case["beams"]
    base, lens = s["base"].long().view(-1, beams), s["lens"].long().view(-1, beams)
    source = base.gather(1, s["parents"].long().view(-1, beams))
    j = torch.arange(case["max_seq"], device=DEV)
    there = j < lens[..., None]
    to = (base[..., None] + j).flatten()
    at = torch.where(there, source[..., None] + j, base[..., None] + j).flatten()
    s["k"][:, to] = s["k"][:, at]
    s["v"][:, to] = s["v"][:, at]
    return {"k": s["k"], "v": s["v"]}


def _own(s):
    from janus_amd import ops
    case = s["case"]
    if case["op"] == "store":
        ops.kv_update_fp4(_engine, s["k"], s["v"], s["kc"], s["ks"], s["vc"], s["vs"], case["max_seq"],
                          row_base=s["base"], positions=s["pos"])
        ops.kv_read_fp4(_engine, s["kc"], s["ks"], s["vc"], s["vs"], s["k_out"], s["v_out"], rows=s["rows"])
        return {"k": s["k_out"], "v": s["v_out"]}
    if case["op"] == "attend":
        ops.fp4_attention(_engine, s["q"], s["kc"], s["ks"], s["vc"], s["vs"], s["out"], case["seqs"], s["cap"],
                          q_start=s["start"], row_base=s["base"], seq_lens=s["lens"])
        return s["out"]
    if case["op"] == "select":
        ops.beam_select(_engine, s["logits"], s["scores"], s["out"], s["parents"], s["tokens"])
        return {"scores": s["out"], "parents": s["parents"], "tokens": s["tokens"]}
    ops.kv_reorder(_engine, [s["k"], s["v"]], case["beams"], case["max_seq"], s["base"], s["parents"],
                   seq_lens=s["lens"], layers=case["layers"])
    return {"k": s["k"], "v": s["v"]}


def run(state):
    if own:
        return _own(state)
    return {"store": _plain_store, "attend": _plain_attend, "select": _plain_select,
            "reorder": _plain_reorder}[state["case"]["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------

def _size(name):
    return 2 if name == "f16" else 4


def work(case):
    if case["op"] == "select":
        rows = case["batch"] * case["beams"]
        alive = case["batch"] if case["first"] else rows   # beams that have ended before they began are not looked at
        return {"bytes": 4 * alive * case["vocab"] + 4 * rows + 12 * case["batch"] * case["n"],
                "flops": 4 * alive * case["vocab"]}
    kvh, hd = case["kv_heads"], case["hd"]
    if case["op"] == "reorder":
        lens, parents = _reorder_plan(case)
        rows = 0
        for n, row in zip(lens, parents):
            moved = [p for i, p in enumerate(row) if p != i]
            rows += n * (len(moved) + len(set(moved)))
        return {"bytes": 2 * case["layers"] * rows * kvh * hd * _size(case["kv"]) + 12 * case["groups"] * case["beams"],
                "flops": 0}
    row = 2 * kvh * (hd // 2 + hd // 32)   # K and V of one position
    if case["op"] == "store":
        # the rows once, the cache written and read, the values written
        per = 2 * kvh * hd * (_size(case["in"]) + _size(case["out"])) + 2 * row + 12
        return {"bytes": case["rows"] * per, "flops": 8 * case["rows"] * kvh * hd}
    rows, ctx = _attend_sizes(case)
    pairs = sum(r * c + r * (r + 1) // 2 for r, c in zip(rows, ctx))
    return {"bytes": sum(rows) * 2 * case["heads"] * hd * _size(case["type"]) + sum(r + c for r, c in zip(rows, ctx)) * row,
            "flops": 4 * hd * case["heads"] * pairs}


# ---- the definitions in 64 bits ----------------------------------------------------

def _rounded(x):
    """The values of a cache that x was stored in."""
    shape = x.shape
    x = x.double().reshape(-1, 32)
    top = x.abs().max(-1, keepdim=True).values
    e = torch.floor(torch.log2(top.clamp(min=1e-30)))
    e = torch.where(torch.pow(2.0, e) > top, e - 1, e)            # log2 may have gone to the next whole number
    e = torch.where(top > 1.75 * torch.pow(2.0, e), e + 1, e) - 2
    scale = torch.pow(2.0, e.clamp(-23, 13))
    y = x.abs() / scale
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0)).double()
    y = (torch.round(y / step) * step).clamp(max=6.0)
    return (torch.sign(x) * y * scale).view(shape)


def _looked_up(codes, scales):
    """Codes and scales as 64-bit values, by a table of all bytes."""
    one = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device=DEV)
    pair = torch.stack([one.repeat(16), one.repeat_interleave(16)], -1)
    x = pair[codes.long()].flatten(-2)
    return x * torch.pow(2.0, scales.double() - 127).repeat_interleave(32, -1)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "store":
        return {"k": _rounded(s["k"]), "v": _rounded(s["v"])}
    if case["op"] == "select":
        logp = torch.log_softmax(s["logits"].double(), -1)
        value = (s["scores"].double().view(-1, 1) + logp).view(case["batch"], -1)
        found, at = torch.sort(value, stable=True, dim=-1, descending=True)
        at = at[:, :case["n"]]
        return {"scores": found[:, :case["n"]], "parents": torch.div(at, case["vocab"], rounding_mode="floor"),
                "tokens": at.remainder(case["vocab"])}
    if case["op"] == "reorder":
        base, lens, beams = s["base"].tolist(), s["lens"].tolist(), case["beams"]
        res = {}
        for name in "kv":
            new = s[name].clone()
            for i, p in enumerate(s["parents"].tolist()):
                src = base[i // beams * beams + p]
                new[:, base[i]:base[i] + lens[i]] = s[name][:, src:src + lens[i]]
            res[name] = new.double()
        return res
    heads, kvh, hd = case["heads"], case["kv_heads"], case["hd"]
    rep = heads // kvh
    parts = []
    start = s["start"].tolist()
    for b, n, i, j in zip(s["base"].tolist(), s["lens"].tolist(), start[:-1], start[1:]):
        k, v = (_looked_up(s[c + "c"][b:b + n], s[c + "s"][b:b + n]).permute(1, 0, 2).contiguous() for c in "kv")
        out = torch.empty(j - i, heads, hd, dtype=torch.float64, device=DEV)
        for r in range(i, j, 2048):
            m = min(2048, j - r)
            ahead = torch.arange(n, device=DEV)[None] >= torch.arange(n - (j - r) + 1, n - (j - r) + 1 + m, device=DEV)[:, None]
            for h in range(kvh):   # the rows of a KV head's queries one behind the other
                q = s["q"][r:r + m, h * rep:(h + 1) * rep].double().reshape(m * rep, hd)
                score = torch.mm(q, k[h].t().contiguous()).view(m, rep, n) / math.sqrt(hd)
                p = torch.softmax(score.masked_fill(ahead[:, None], -math.inf), -1)
                out[r - i:r - i + m, h * rep:(h + 1) * rep] = torch.mm(p.view(m * rep, n), v[h]).view(m, rep, hd)
        parts.append(out)
    return torch.cat(parts)
