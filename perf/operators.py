"""The operators around a shared KV cache whose speed and exactness are measured.

  heads   norms of the query and key heads, their rotation and the append of K
          and V to the cache, from the rows of a fused QKV product
          (ops.qk_norm_rope).
  prompt  causal attention of packed rows: whole prompts, chunks of a prompt
          behind a cached context, drafted tokens (ops.prompt_attention).
  prefix  decode attention of a batch whose sequences share a prefix, which is
          stored once (ops.prefix_attention).

A cache here is one layer's slice, [rows][kv heads][head dim]; a sequence's
positions lie in consecutive rows from its row base on. Head layouts are those
of the Llama-3-8B, Llama-2-7B and tiny models of the benchmark and tests, and
generic ones.
"""
from __future__ import annotations

import math
import random

import torch

own = False   # False: plain torch operations; True: the framework's operators

DEV = "cuda:0"
EPS = 1e-5
THETA = 500000.0
DTYPES = {"f16": torch.float16, "f32": torch.float32}


# ---- cases ---------------------------------------------------------------------

def listed():
    return [
        # one decode step of one request: the launch is what counts
        {"name": "heads_step", "op": "heads", "rows": 1, "heads": 32, "kv_heads": 8, "hd": 128, "in": "f32",
         "out": "f32", "kv": "f16", "norm": True, "max_seq": 2048, "mix": 1},
        # one decode step of a batch, every head with its own K and V
        {"name": "heads_batch", "op": "heads", "rows": 48, "heads": 32, "kv_heads": 32, "hd": 128, "in": "f32",
         "out": "f32", "kv": "f32", "norm": True, "max_seq": 512, "mix": 2},
        # the packed prompts of several requests
        {"name": "heads_prompts", "op": "heads", "rows": 8192, "heads": 32, "kv_heads": 8, "hd": 128, "in": "f16",
         "out": "f16", "kv": "f16", "norm": True, "max_seq": 2048, "mix": 3},
        # three short prompts on the tiny model, the reference's types
        {"name": "prompt_tiny", "op": "prompt", "seqs": 3, "least": 1, "most": 13, "context": 0, "heads": 4,
         "kv_heads": 2, "hd": 64, "type": "f32", "kv": "f32", "mix": 4},
        # drafted tokens of 16 requests against their contexts
        {"name": "prompt_drafts", "op": "prompt", "seqs": 16, "least": 5, "most": 5, "context": 4000, "heads": 32,
         "kv_heads": 8, "hd": 128, "type": "f16", "kv": "f16", "mix": 5},
        # chat prompts of 24 requests, from a word to a page
        {"name": "prompt_chats", "op": "prompt", "seqs": 24, "least": 3, "most": 700, "context": 0, "heads": 32,
         "kv_heads": 8, "hd": 128, "type": "f16", "kv": "f16", "mix": 6},
        # one long document
        {"name": "prompt_long", "op": "prompt", "seqs": 1, "least": 8192, "most": 8192, "context": 0, "heads": 32,
         "kv_heads": 8, "hd": 128, "type": "f16", "kv": "f16", "mix": 7},
        # prompts in the reference's types, every head with its own K and V
        {"name": "prompt_mha_f32", "op": "prompt", "seqs": 6, "least": 33, "most": 512, "context": 0, "heads": 32,
         "kv_heads": 32, "hd": 128, "type": "f32", "kv": "f32", "mix": 8},
        # the last chunk of a long prompt: binary32 rows on a binary16 cache
        {"name": "prompt_chunk", "op": "prompt", "seqs": 1, "least": 512, "most": 512, "context": 7680, "heads": 32,
         "kv_heads": 8, "hd": 128, "type": "f32", "kv": "f16", "mix": 9},
        # few requests, a short system prompt
        {"name": "prefix_short", "op": "prefix", "batch": 4, "prefix": 500, "most": 40, "heads": 32, "kv_heads": 8,
         "hd": 128, "type": "f32", "kv": "f16", "mix": 10},
        # a batch of chats behind one system prompt with its documents
        {"name": "prefix_system", "op": "prefix", "batch": 32, "prefix": 4096, "most": 512, "heads": 32, "kv_heads": 8,
         "hd": 128, "type": "f16", "kv": "f16", "mix": 11},
        # 64 samples of one long context, binary32 rows as the decode step has them
        {"name": "prefix_long", "op": "prefix", "batch": 64, "prefix": 16384, "most": 1024, "heads": 32, "kv_heads": 8,
         "hd": 128, "type": "f32", "kv": "f16", "mix": 12},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    heads, kv_heads, hd = rng.choice([(32, 8, 128), (32, 32, 128), (4, 2, 64), (24, 8, 64), (16, 1, 128), (40, 8, 128)])
    typ, kv = rng.choice([("f16", "f16"), ("f32", "f16"), ("f32", "f32")])
    case = {"heads": heads, "kv_heads": kv_heads, "hd": hd, "kv": kv, "mix": rng.randrange(100, 1 << 30)}
    op = rng.choice(["heads", "prompt", "prompt", "prefix"])
    if op == "heads":
        rows = _log(rng, 1, 6000)
        return {"op": op, "rows": rows, "in": typ, "out": rng.choice(["f16", "f32"]), "norm": rng.random() < 0.8,
                "max_seq": _log(rng, 64, 4096 if rows > 64 else 65536 // max(16, rows)), **case}
    if op == "prefix":
        batch, most = _log(rng, 1, 64), _log(rng, 1, 800)
        return {"op": op, "type": typ, "batch": batch, "prefix": _log(rng, 64, 12000), "most": most, **case}
    seqs = _log(rng, 1, 32)
    most = _log(rng, 1, 4000 // seqs)
    return {"op": op, "type": typ, "seqs": seqs, "least": max(1, most // 20), "most": most,
            "context": rng.choice([0, _log(rng, 1, 4000 // seqs + 64)]), **case}


def _prompt_sizes(case):
    """(rows, context before them) of each sequence; one has the most rows."""
    rng = random.Random(case["mix"])
    rows = [rng.randint(case["least"], case["most"]) for _ in range(case["seqs"])]
    rows[rng.randrange(len(rows))] = case["most"]
    ctx = [rng.randint(case["context"] // 20, case["context"]) if case["seqs"] > 1 else case["context"] for _ in rows]
    return rows, ctx


def _prefix_sizes(case):
    """Own positions of each sequence, the step's token among them."""
    rng = random.Random(case["mix"])
    own_len = [rng.randint(1, case["most"]) for _ in range(case["batch"])]
    own_len[rng.randrange(len(own_len))] = case["most"]
    return own_len


# ---- inputs --------------------------------------------------------------------

def _places(case):
    """Row bases and positions of the rows of a "heads" case: runs of rows that
    follow each other in a sequence (prompts), or single ones (a decode step)."""
    rng = random.Random(case["mix"])
    rows, cap = case["rows"], case["max_seq"]
    base, pos = [], []
    while len(base) < rows:
        left = rows - len(base)
        n = 1 if rows <= 64 else min(left, rng.randint(1, cap))
        first = rng.randint(0, cap - n)
        slot = len(pos) and max(base) // cap + 1
        base += [slot * cap] * n
        pos += range(first, first + n)
    return base, pos


def _rand(gen, shape, dtype, sigma=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * sigma).to(dtype)


def _inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    heads, kvh, hd = case["heads"], case["kv_heads"], case["hd"]
    kv = DTYPES[case["kv"]]

    def index(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    if case["op"] == "heads":
        base, pos = _places(case)
        total = base[-1] + case["max_seq"]
        qkv = _rand(gen, (case["rows"], heads + 2 * kvh, hd), DTYPES[case["in"]], 2.0)
        ang = torch.arange(case["max_seq"], device=DEV, dtype=torch.float64)[:, None] * \
            THETA ** (-torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)
        return {"q": qkv[:, :heads], "k": qkv[:, heads:heads + kvh], "v": qkv[:, heads + kvh:],
                "q_gamma": 1 + _rand(gen, (hd,), torch.float32, 0.3) if case["norm"] else None,
                "k_gamma": 1 + _rand(gen, (hd,), torch.float32, 0.3) if case["norm"] else None,
                "table": torch.stack([ang.cos(), ang.sin()], -1).float().contiguous(),
                "base": index(base), "pos": index(pos),
                "k_cache": _rand(gen, (total, kvh, hd), kv), "v_cache": _rand(gen, (total, kvh, hd), kv),
                "out": torch.zeros(case["rows"], heads, hd, dtype=DTYPES[case["out"]], device=DEV)}
    if case["op"] == "prompt":
        rows, ctx = _prompt_sizes(case)
        lens = [r + c for r, c in zip(rows, ctx)]
        cap = max(lens)
        slots = list(range(len(rows)))
        random.Random(case["mix"] + 1).shuffle(slots)
        starts = [0]
        for r in rows:
            starts.append(starts[-1] + r)
        got = {"start": index(starts), "lens": index(lens), "base": index([s * cap for s in slots]), "cap": cap,
               "most_rows": max(rows), "q": _rand(gen, (starts[-1], heads, hd), DTYPES[case["type"]], 1.5)}
        total = len(rows) * cap
    else:
        lens = _prefix_sizes(case)
        cap = case["most"]
        slots = list(range(len(lens)))
        random.Random(case["mix"] + 1).shuffle(slots)
        got = {"lens": index(lens), "base": index([case["prefix"] + s * cap for s in slots]), "cap": cap,
               "q": _rand(gen, (len(lens), heads, hd), DTYPES[case["type"]], 1.5)}
        total = case["prefix"] + len(lens) * cap
    got["k_cache"] = _rand(gen, (total, kvh, hd), kv)
    got["v_cache"] = _rand(gen, (total, kvh, hd), kv)
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

def _normed_rotated(x, gamma, table, pos):
    x = x.float()
    if gamma is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma
    half = x.shape[-1] // 2
    cs = table[pos]
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _plain_heads(s):
    pos = s["pos"].long()
    at = s["base"].long() + pos
    s["out"][:] = _normed_rotated(s["q"], s["q_gamma"], s["table"], pos).to(s["out"].dtype)
    s["k_cache"][at] = _normed_rotated(s["k"], s["k_gamma"], s["table"], pos).to(s["k_cache"].dtype)
    s["v_cache"][at] = s["v"].to(s["v_cache"].dtype)
    return {"q": s["out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _grouped(q, k, v, seen):
    """q [b, n, heads, hd] on k, v [b, len, kv heads, hd], seen [b, n, len]: out [b, n, heads, hd] in 32 bits."""
    b, n, heads, hd = q.shape
    kvh = k.shape[2]
    rep = heads // kvh
    q = q.float().view(b, n, kvh, rep, hd).permute(0, 2, 1, 3, 4).reshape(b, kvh, n * rep, hd)
    k = k.float().permute(0, 2, 3, 1).contiguous()
    v = v.float().permute(0, 2, 1, 3).contiguous()
    score = (torch.matmul(q, k) * (1.0 / math.sqrt(hd))).view(b, kvh, n, rep, -1)
    score = score.masked_fill(~seen[:, None, :, None, :], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, kvh, n * rep, -1), v).view(b, kvh, n, rep, hd) / total.clamp(min=1e-30)
    return out.permute(0, 2, 1, 3, 4).reshape(b, n, heads, hd)


def _plain_prompt(s):
    q, lens, start = s["q"], s["lens"].long(), s["start"].long()
    rows = q.shape[0]
    count = start[1:] - start[:-1]
    i = torch.arange(s["most_rows"], device=DEV)
    j = torch.arange(s["cap"], device=DEV)
    there = i[None] < count[:, None]
    at = torch.where(there, start[:-1, None] + i[None], rows)
    kv_at = s["base"].long()[:, None] + j[None]
    seen = j[None, None] < (lens[:, None] - count[:, None] + i[None] + 1)[..., None]
    out = _grouped(q[at.clamp(max=rows - 1)], s["k_cache"][kv_at], s["v_cache"][kv_at], seen)
    whole = torch.empty(rows + 1, *q.shape[1:], dtype=q.dtype, device=DEV)
    whole[at] = out.to(q.dtype)
    return whole[:rows]


def _plain_prefix(s):
    q, n = s["q"], s["case"]["prefix"]
    batch, heads, hd = q.shape
    k, v = s["k_cache"], s["v_cache"]
    kvh = k.shape[1]
    rep = heads // kvh
    scale = 1.0 / math.sqrt(hd)
    q = q.float().view(batch, kvh, rep, hd)
    j = torch.arange(s["cap"], device=DEV)
    at = s["base"].long()[:, None] + j[None]
    # the prefix once for all queries of a KV head
    qh = q.permute(1, 0, 2, 3).reshape(kvh, batch * rep, hd)
    s1 = torch.matmul(qh, k[:n].float().permute(1, 2, 0).contiguous()) * scale                   # [kvh, batch rep, n]
    s2 = torch.matmul(q, k[at].float().permute(0, 2, 3, 1).contiguous()) * scale                 # [batch, kvh, rep, cap]
    s2 = s2.masked_fill((j[None] >= s["lens"].long()[:, None])[:, None, None], -math.inf)
    s1 = s1.view(kvh, batch, rep, n)
    m = torch.maximum(s1.amax(-1).transpose(0, 1), s2.amax(-1))                                  # [batch, kvh, rep]
    p1 = torch.exp(s1 - m.transpose(0, 1)[..., None])
    p2 = torch.exp(s2 - m[..., None])
    total = p1.sum(-1).transpose(0, 1) + p2.sum(-1)
    o1 = torch.matmul(p1.view(kvh, batch * rep, n), v[:n].float().transpose(0, 1).contiguous())
    o2 = torch.matmul(p2, v[at].float().permute(0, 2, 1, 3).contiguous())
    out = (o1.view(kvh, batch, rep, hd).transpose(0, 1) + o2) / total[..., None]
    return out.reshape(batch, heads, hd).to(s["out"].dtype)


def _own(s):
    from janus_amd import ops
    case = s["case"]
    if case["op"] == "heads":
        ops.qk_norm_rope(_engine, s["q"], s["k"], s["v"], s["q_gamma"], s["k_gamma"], EPS, s["table"], s["out"],
                         s["k_cache"], s["v_cache"], case["max_seq"], row_base=s["base"], positions=s["pos"])
        return {"q": s["out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if case["op"] == "prompt":
        ops.prompt_attention(_engine, s["q"], s["k_cache"], s["v_cache"], s["out"], case["seqs"], s["cap"],
                             q_start=s["start"], row_base=s["base"], seq_lens=s["lens"])
    else:
        ops.prefix_attention(_engine, s["q"], s["k_cache"], s["v_cache"], s["out"], 0, case["prefix"], s["cap"],
                             row_base=s["base"], seq_lens=s["lens"])
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return {"heads": _plain_heads, "prompt": _plain_prompt, "prefix": _plain_prefix}[state["case"]["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------

def _size(name):
    return 2 if name == "f16" else 4


def work(case):
    heads, kvh, hd = case["heads"], case["kv_heads"], case["hd"]
    kv_row = 2 * kvh * hd * _size(case["kv"])   # K and V of one position
    if case["op"] == "heads":
        rows = case["rows"]
        per = (heads + 2 * kvh) * hd * _size(case["in"]) + heads * hd * _size(case["out"]) + kv_row + 8
        _, pos = _places(case)
        return {"bytes": rows * per + len(set(pos)) * hd * 4 + 2 * hd * 4 * case["norm"],
                "flops": rows * (heads + kvh) * hd * (7 if case["norm"] else 3)}
    q_row = 2 * heads * hd * _size(case["type"])   # a row of q and of the output
    if case["op"] == "prompt":
        rows, ctx = _prompt_sizes(case)
        pairs = sum(r * c + r * (r + 1) // 2 for r, c in zip(rows, ctx))
        return {"bytes": sum(rows) * q_row + sum(r + c for r, c in zip(rows, ctx)) * kv_row,
                "flops": 4 * hd * heads * pairs}
    lens = _prefix_sizes(case)
    return {"bytes": len(lens) * q_row + (case["prefix"] + sum(lens)) * kv_row,
            "flops": 4 * hd * heads * (len(lens) * case["prefix"] + sum(lens))}


# ---- the definitions in 64 bits ----------------------------------------------------

def _softmax_rows(q, k, v, seen):
    """q [n, heads, hd], k and v [len, kv heads, hd]; row r sees the first seen[r] positions."""
    n, heads, hd = q.shape
    out = torch.zeros(n, heads, hd, dtype=torch.float64, device=DEV)
    rep = heads // k.shape[1]
    there = torch.arange(k.shape[0], device=DEV)
    for h in range(heads):
        kh, vh = k[:, h // rep].double().contiguous(), v[:, h // rep].double().contiguous()
        for r in range(0, n, 4096):
            score = torch.mm(q[r:r + 4096, h].double(), kh.t().contiguous()) / math.sqrt(hd)
            score[there[None] >= seen[r:r + 4096, None]] = -math.inf
            out[r:r + 4096, h] = torch.mm(torch.softmax(score, -1), vh)
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "heads":
        hd = case["hd"]
        half = hd // 2
        pos = s["pos"].long()
        turn = torch.view_as_complex(s["table"].double())[pos][:, None]
        res = {}
        for name in ("q", "k"):
            x = s[name].double()
            if case["norm"]:
                x = x * s[name + "_gamma"].double() * (x.pow(2).sum(-1, keepdim=True) / hd + EPS).rsqrt()
            z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
            res[name] = torch.cat([z.real, z.imag], -1)
        at = s["base"].long() + pos
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        kc[at], vc[at] = res["k"], s["v"].double()
        return {"q": res["q"], "k_cache": kc, "v_cache": vc}
    base, lens = s["base"].tolist(), s["lens"].tolist()
    if case["op"] == "prompt":
        start, parts = s["start"].tolist(), []
        for b, n, i, j in zip(base, lens, start[:-1], start[1:]):
            seen = torch.arange(n - (j - i) + 1, n + 1, device=DEV)
            parts.append(_softmax_rows(s["q"][i:j], s["k_cache"][b:b + n], s["v_cache"][b:b + n], seen))
        return torch.cat(parts)
    p = case["prefix"]
    parts = []
    for r, (b, n) in enumerate(zip(base, lens)):
        k = torch.cat([s["k_cache"][:p], s["k_cache"][b:b + n]])
        v = torch.cat([s["v_cache"][:p], s["v_cache"][b:b + n]])
        # one row: the products of all heads at once
        q = s["q"][r].double().view(case["kv_heads"], -1, case["hd"])
        score = torch.bmm(q, k.double().permute(1, 2, 0).contiguous()) / math.sqrt(case["hd"])
        o = torch.bmm(torch.softmax(score, -1), v.double().permute(1, 0, 2).contiguous())
        parts.append(o.reshape(1, case["heads"], case["hd"]))
    return torch.cat(parts)
