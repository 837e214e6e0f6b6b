"""Cases of the batched-serving operators: the q/k norm with rotation and cache
append, the paged decode attention, and the logits rules.

With `own` false, run() computes each operator in its plain form (elementary
torch operations in 32 bits, rounded once at the end); with `own` true it
calls chpe_qwen_engine_b200.ops.  exact() computes the same outputs in 64
bits, one sequence or row at a time.

Cache: [pages][page positions][kv heads][head dim], as the engine lays out one
layer's pool.  Head counts are those of the three architectures (16/2/128,
16/4/256, 64/8/128) and generic ones.
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
DEV = "cuda"
LIMIT = {"attention": 64 * 8192 // 3 * 8 * 128, "qk": 16384 * 80 * 128, "logits": 256 * 151936}


def listed():
    return [
        # a chat's first tokens on the 3B's heads, f32 activations and the engine's FP16 cache: latency
        {"name": "attn_one_short", "op": "attention", "heads": 16, "kv_heads": 2, "head_dim": 128, "act": "f32",
         "cache": "f16", "batch": 1, "longest": 77, "ragged": False, "page": 64},
        # one user with a very long document on the 72B's heads: split over the length
        {"name": "attn_one_long", "op": "attention", "heads": 64, "kv_heads": 8, "head_dim": 128, "act": "bf16",
         "cache": "bf16", "batch": 1, "longest": 131071, "ragged": False, "page": 64},
        # a server's mixed batch on the 9B's heads, one slot empty, small pages
        {"name": "attn_mixed", "op": "attention", "heads": 16, "kv_heads": 4, "head_dim": 256, "act": "f16",
         "cache": "f16", "batch": 37, "longest": 4093, "ragged": True, "page": 16},
        # a full server on the 72B's heads
        {"name": "attn_full", "op": "attention", "heads": 64, "kv_heads": 8, "head_dim": 128, "act": "bf16",
         "cache": "bf16", "batch": 64, "longest": 8192, "ragged": True, "page": 64},
        # one decoded token on the 9B's heads: norm, rotation of 64 of 256 dimensions, f32
        {"name": "qk_one_token", "op": "qk", "heads": 16, "kv_heads": 4, "head_dim": 256, "rope_dim": 64, "act": "f32",
         "cache": "f16", "tokens": 1, "norm": True, "theta": 1e7, "first": 100003, "prefill": False, "page": 64},
        # one step of a batch on the 72B's heads (no norm), every token at a position of its own
        {"name": "qk_step", "op": "qk", "heads": 64, "kv_heads": 8, "head_dim": 128, "rope_dim": 128, "act": "bf16",
         "cache": "bf16", "tokens": 61, "norm": False, "theta": 1e6, "first": 1000, "prefill": False, "page": 64},
        # a chunk of a long prompt on the 3B's heads with q/k norms
        {"name": "qk_chunk", "op": "qk", "heads": 16, "kv_heads": 2, "head_dim": 128, "rope_dim": 128, "act": "f16",
         "cache": "f16", "tokens": 2049, "norm": True, "theta": 1e6, "first": 30000, "prefill": True, "page": 64},
        # a whole long prompt on the 72B's heads
        {"name": "qk_prompt", "op": "qk", "heads": 64, "kv_heads": 8, "head_dim": 128, "rope_dim": 128, "act": "bf16",
         "cache": "bf16", "tokens": 16384, "norm": True, "theta": 1e6, "first": 0, "prefill": True, "page": 64},
        # one chat of the 3B: penalties over a few hundred tokens and a few biases
        {"name": "logits_one", "op": "logits", "vocab": 151936, "dtype": "f32", "batch": 1, "history": 211,
         "biases": 12, "mask": False, "penalties": True},
        # tool calls of the 9B: a grammar's mask for each row and nothing else
        {"name": "logits_grammar", "op": "logits", "vocab": 248320, "dtype": "bf16", "batch": 7, "history": 0,
         "biases": 0, "mask": True, "penalties": False},
        # a full server of the 72B: everything at once, ragged histories
        {"name": "logits_server", "op": "logits", "vocab": 152064, "dtype": "f32", "batch": 64, "history": 2048,
         "biases": 300, "mask": True, "penalties": True},
        # a large offline batch with long contexts, bf16 logits
        {"name": "logits_offline", "op": "logits", "vocab": 151936, "dtype": "bf16", "batch": 256, "history": 8191,
         "biases": 0, "mask": False, "penalties": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("attention", "qk", "logits"))
    heads, kv, hd = rng.choice(((16, 2, 128), (16, 4, 256), (64, 8, 128), (32, 32, 64), (12, 4, 128), (24, 2, 64)))
    act = rng.choice(("f32", "f16", "bf16"))
    cache = rng.choice(("f16", "bf16")) if act == "f32" else act
    if op == "attention":
        batch = _log(rng, 1, 64)
        longest = _log(rng, 1, max(1, min(131071, LIMIT["attention"] // (batch * kv * hd))))
        return {"op": op, "heads": heads, "kv_heads": kv, "head_dim": hd, "act": act, "cache": cache, "batch": batch,
                "longest": longest, "ragged": rng.random() < 0.6, "page": rng.choice((16, 64, 128))}
    if op == "qk":
        tokens = _log(rng, 1, min(16384, LIMIT["qk"] // ((heads + 2 * kv) * hd * (2 if act == "f32" else 1))))
        return {"op": op, "heads": heads, "kv_heads": kv, "head_dim": hd,
                "rope_dim": rng.choice([d for d in (32, 64, 128, 256) if d <= hd]), "act": act, "cache": cache,
                "tokens": tokens, "norm": rng.random() < 0.7, "theta": rng.choice((1e4, 1e6, 1e7)),
                "first": _log(rng, 1, 200000), "prefill": rng.random() < 0.5, "page": 64}
    vocab = rng.choice((151936, 152064, 248320, 32001, 50257))
    mask, penalties = rng.random() < 0.5, rng.random() < 0.7
    return {"op": op, "vocab": vocab, "dtype": rng.choice(("f32", "f16", "bf16")),
            "batch": _log(rng, 1, min(256, LIMIT["logits"] // vocab // 2)), "history": _log(rng, 1, 8191) if penalties else 0,
            "biases": rng.choice((0, _log(rng, 1, 300))), "mask": mask, "penalties": penalties}


def _lengths(n, longest, ragged):
    """n lengths up to `longest`: all alike, or the first 0 and the others on a square curve."""
    if not ragged or n == 1:
        return [longest] * n
    return [0] + [max(1, round(longest * (i / (n - 1)) ** 2)) for i in range(1, n)]


def work(case):
    if case["op"] == "attention":
        n = sum(_lengths(case["batch"], case["longest"], case["ragged"]))
        h, kv, d, b = case["heads"], case["kv_heads"], case["head_dim"], case["batch"]
        moved = n * kv * d * 2 * SIZE[case["cache"]] + 2 * b * h * d * SIZE[case["act"]] + 4 * b * h
        return {"bytes": moved, "flops": 4 * n * h * d}
    if case["op"] == "qk":
        t, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
        moved = t * d * ((2 * h + 2 * kv) * SIZE[case["act"]] + 2 * kv * SIZE[case["cache"]]) + 12 * t
        return {"bytes": moved, "flops": t * (h + kv) * (4 * d * case["norm"] + 3 * case["rope_dim"])}
    b, v = case["batch"], case["vocab"]
    n = sum(_lengths(b, case["history"], True))
    moved = b * v * (SIZE[case["dtype"]] + 4) + 4 * n + 8 * b * case["biases"] + (b * ((v + 31) // 32) * 4 if case["mask"] else 0)
    return {"bytes": moved, "flops": b * v + 4 * n}


# ---- inputs ---------------------------------------------------------------
def _gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def _prepare_attention(c, seed):
    g = _gen(seed)
    b, page, kv, d = c["batch"], c["page"], c["kv_heads"], c["head_dim"]
    lens = torch.tensor(_lengths(b, c["longest"], c["ragged"]), device=DEV)
    lens = lens[torch.randperm(b, generator=g, device=DEV)].to(torch.int32)
    each = (c["longest"] + page - 1) // page
    # pages in a shuffled order, as a server's free list leaves them
    table = torch.randperm(b * each, generator=g, device=DEV).to(torch.int32).view(b, each)
    kc = torch.randn(b * each, page, kv, d, generator=g, device=DEV, dtype=DT[c["cache"]])
    vc = torch.randn(b * each, page, kv, d, generator=g, device=DEV, dtype=DT[c["cache"]])
    q = torch.randn(b, c["heads"], d, generator=g, device=DEV).to(DT[c["act"]])
    s = {"case": c, "q": q, "k_cache": kc, "v_cache": vc, "table": table, "lens": lens, "scale": 1.0 / math.sqrt(d)}
    s["out"], s["lse"] = torch.empty_like(q), torch.empty(b, c["heads"], device=DEV)
    if own:
        from chpe_qwen_engine_b200 import ops
        s["workspace"] = ops.attention_workspace(d, DEV)
    return s


def _prepare_qk(c, seed):
    g = _gen(seed)
    t, h, kv, d, page = c["tokens"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    # the fused projection's output: q, k and v of a token side by side
    qkv = torch.randn(t, (h + 2 * kv) * d, generator=g, device=DEV).to(DT[c["act"]])
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split((h * d, kv * d, kv * d), 1))
    rows = -(-t // page) * page + page
    if c["prefill"]:
        pos = torch.arange(c["first"], c["first"] + t, device=DEV, dtype=torch.int32)
        # whole pages of a shuffled list, filled in order
        order = torch.randperm(rows // page, generator=g, device=DEV)
        at = torch.arange(t, device=DEV)
        slots = order[at // page] * page + at % page
    else:
        pos = torch.randint(0, 2 * c["first"], (t,), generator=g, device=DEV, dtype=torch.int32)
        slots = torch.randperm(rows, generator=g, device=DEV)[:t]
    weight = lambda: 1 + 0.1 * torch.randn(d, generator=g, device=DEV) if c["norm"] else None  # noqa: E731
    s = {"case": c, "q": q, "k": k, "v": v, "positions": pos, "slots": slots, "q_weight": weight(), "k_weight": weight(), "eps": 1e-6}
    for name in ("k_cache", "v_cache"):
        s[name] = torch.zeros(rows // page, page, kv, d, device=DEV, dtype=DT[c["cache"]])
    i = torch.arange(0, c["rope_dim"], 2, dtype=torch.float64)
    s["inv_freq"] = torch.pow(torch.tensor(c["theta"], dtype=torch.float64), -i / c["rope_dim"])
    s["inv_freq_device"] = s["inv_freq"].to(DEV)
    s["q_out"] = torch.empty(t, h, d, device=DEV, dtype=DT[c["act"]])
    return s


def _prepare_logits(c, seed):
    g = _gen(seed)
    b, v, n = c["batch"], c["vocab"], c["history"]
    s = {"case": c, "logits": (3 * torch.randn(b, v, generator=g, device=DEV)).to(DT[c["dtype"]])}
    for name in ("history", "prompt_lens", "total_lens", "repetition", "frequency", "presence", "bias_ids", "bias_values", "mask"):
        s[name] = None
    if c["penalties"]:
        # text repeats itself: low ids are much more frequent than high ones
        u = torch.rand(b, n, generator=g, device=DEV)
        s["history"] = ((u ** 4) * v).to(torch.int32).clamp_(max=v - 1)
        total = torch.tensor(_lengths(b, n, True), device=DEV)[torch.randperm(b, generator=g, device=DEV)]
        s["total_lens"] = total.to(torch.int32)
        s["prompt_lens"] = (total * 2 // 3).to(torch.int32)
        s["repetition"] = 1 + 0.3 * torch.rand(b, generator=g, device=DEV)
        s["frequency"] = 0.5 * torch.rand(b, generator=g, device=DEV)
        s["presence"] = 0.5 * torch.rand(b, generator=g, device=DEV)
    if c["biases"]:
        s["bias_ids"] = torch.randint(0, v, (b, c["biases"]), generator=g, device=DEV, dtype=torch.int32)
        s["bias_values"] = 4 * torch.randn(b, c["biases"], generator=g, device=DEV)
    if c["mask"]:
        words = (v + 31) // 32
        # a grammar allows stretches of tokens: three words in four are all ones or all zeros
        some = torch.randint(-2**31, 2**31, (b, words), generator=g, device=DEV, dtype=torch.int64)
        kind = torch.randint(0, 4, (b, words), generator=g, device=DEV)
        some = torch.where(kind == 0, some, torch.where(kind == 1, torch.full_like(some, -1), torch.zeros_like(some)))
        s["mask"] = some.to(torch.int32)
    s["out"] = torch.empty(b, v, device=DEV)
    s["argmax"] = torch.empty(b, device=DEV, dtype=torch.int32)
    return s


def prepare(case, seed):
    return {"attention": _prepare_attention, "qk": _prepare_qk, "logits": _prepare_logits}[case["op"]](case, seed)


# ---- the plain forms ------------------------------------------------------
def _plain_attention(s):
    c, table, lens = s["case"], s["table"].long(), s["lens"].long()
    b, kv, d = c["batch"], c["kv_heads"], c["head_dim"]
    k, v = (s[name][table].reshape(b, -1, kv, d).float() for name in ("k_cache", "v_cache"))
    inside = torch.arange(k.shape[1], device=DEV) < lens[:, None]
    q = s["q"].float().view(b, kv, -1, d)
    score = torch.matmul(q, k.permute(0, 2, 3, 1)) * s["scale"]
    score = torch.where(inside[:, None, None, :], score, -torch.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    v = torch.where(inside[:, :, None, None], v, 0.0)
    out = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total)).view(b, -1)
    return {"out": out.reshape(b, -1, d).to(s["q"].dtype), "lse": lse}


def _plain_qk(s):
    c = s["case"]
    half = c["rope_dim"] // 2
    angle = s["positions"].double()[:, None] * s["inv_freq_device"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(x, weight):
        x = x.float()
        if c["norm"]:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * weight
        lo, hi, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin, rest), -1)

    kc, vc = (s[name].flatten(0, 1) for name in ("k_cache", "v_cache"))
    kc[s["slots"]] = turned(s["k"], s["k_weight"]).to(kc.dtype)
    vc[s["slots"]] = s["v"].float().to(vc.dtype)
    return {"q": turned(s["q"], s["q_weight"]).to(s["q"].dtype), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_logits(s):
    c = s["case"]
    b, v = c["batch"], c["vocab"]
    x = s["logits"].float()
    if c["penalties"]:
        at = torch.arange(c["history"], device=DEV)
        ids, kept = s["history"].long(), at < s["total_lens"][:, None]
        written = (kept & (at >= s["prompt_lens"][:, None])).int()
        seen = torch.zeros(b, v, device=DEV, dtype=torch.int32).scatter_add_(1, ids, kept.int())
        count = torch.zeros(b, v, device=DEV, dtype=torch.int32).scatter_add_(1, ids, written).float()
        r = s["repetition"][:, None]
        x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
        x = torch.where(count > 0, x - s["frequency"][:, None] * count - s["presence"][:, None], x)
    if c["biases"]:
        # of entries with the same id the last one counts
        nth = torch.arange(1, c["biases"] + 1, device=DEV).expand(b, -1)
        last = torch.zeros(b, v, device=DEV, dtype=torch.int64).scatter_reduce_(1, s["bias_ids"].long(), nth, "amax")
        x = torch.where(last > 0, x + s["bias_values"].gather(1, (last - 1).clamp(min=0)), x)
    if c["mask"]:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        x = torch.where(bits.view(b, -1)[:, :v] > 0, x, -torch.inf)
    y = torch.where(torch.isnan(x), -torch.inf, x)
    top = y.amax(1, keepdim=True)
    first = torch.where(y == top, torch.arange(v, device=DEV, dtype=torch.int32), v).amin(1)
    return {"logits": x, "argmax": torch.where(top[:, 0] > -torch.inf, first, -1).to(torch.int32)}


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"attention": _plain_attention, "qk": _plain_qk, "logits": _plain_logits}[op](s)
    from chpe_qwen_engine_b200 import ops
    if op == "attention":
        ops.attention_decode_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], scale=s["scale"],
                                   out=s["out"], lse=s["lse"], workspace=s["workspace"])
        return {"out": s["out"], "lse": s["lse"]}
    if op == "qk":
        ops.qk_norm_rope(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], q_weight=s["q_weight"],
                         k_weight=s["k_weight"], eps=s["eps"], k_cache=s["k_cache"], v_cache=s["v_cache"],
                         slots=s["slots"], q_out=s["q_out"])
        return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    ops.logits_process(s["logits"], history=s["history"], prompt_lens=s["prompt_lens"], total_lens=s["total_lens"],
                       repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                       bias_ids=s["bias_ids"], bias_values=s["bias_values"], mask=s["mask"], out=s["out"],
                       argmax=s["argmax"])
    return {"logits": s["out"], "argmax": s["argmax"]}


# ---- the definitions in 64 bits -------------------------------------------
def _exact_attention(s):
    c = s["case"]
    b, h, kv, d, page = c["batch"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    out = torch.zeros(b, h, d, device=DEV, dtype=torch.float64)
    lse = torch.full((b, h), -math.inf, device=DEV, dtype=torch.float64)
    for i, n in enumerate(s["lens"].tolist()):
        for head in range(kv if n else 0):
            pages = s["table"][i, : -(-n // page)].long()
            k = s["k_cache"][pages, :, head].reshape(-1, d)[:n].double()
            v = s["v_cache"][pages, :, head].reshape(-1, d)[:n].double()
            mine = slice(head * (h // kv), (head + 1) * (h // kv))
            score = (k @ s["q"][i, mine].double().T) / math.sqrt(d)
            lse[i, mine] = torch.logsumexp(score, 0)
            out[i, mine] = torch.softmax(score, 0).T @ v
    return {"out": out, "lse": lse}


def _exact_qk(s):
    c = s["case"]
    n = c["rope_dim"] // 2
    freq = [c["theta"] ** (-2.0 * i / c["rope_dim"]) for i in range(n)]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), s["positions"].double().view(-1, 1) * torch.tensor(freq, dtype=torch.float64, device=DEV))

    def turned(x, weight):
        y = x.double()
        if weight is not None:
            y = weight.double() * y / torch.sqrt(torch.linalg.vector_norm(y, dim=2, keepdim=True) ** 2 / c["head_dim"] + 1e-6)
        z = torch.complex(y[:, :, :n], y[:, :, n:2 * n]) * turn.unsqueeze(1)
        y = y.clone()
        y[:, :, :n], y[:, :, n:2 * n] = z.real, z.imag
        return y

    out = {"q": turned(s["q"], s["q_weight"])}
    for name, rows in (("k_cache", turned(s["k"], s["k_weight"])), ("v_cache", s["v"].double())):
        flat = torch.zeros_like(s[name], dtype=torch.float64).view(-1, c["kv_heads"], c["head_dim"])
        out[name] = flat.index_copy_(0, s["slots"], rows).view_as(s[name])
    return out


def _exact_logits(s):
    c = s["case"]
    v = c["vocab"]
    rows, tops = [], []
    for i in range(c["batch"]):
        x = s["logits"][i].double()
        if c["penalties"]:
            p, n = int(s["prompt_lens"][i]), int(s["total_lens"][i])
            said = s["history"][i, :n].long()
            seen, count = torch.bincount(said, minlength=v), torch.bincount(said[p:], minlength=v)
            r = s["repetition"][i].double()
            x = x * torch.where(seen == 0, 1.0, torch.where(x > 0, 1 / r, r))
            x = x - s["frequency"][i].double() * count - s["presence"][i].double() * (count > 0)
        if c["biases"]:
            table = dict(zip(s["bias_ids"][i].tolist(), s["bias_values"][i].tolist()))
            x[list(table)] += torch.tensor(list(table.values()), device=DEV, dtype=torch.float64)
        if c["mask"]:
            words = s["mask"][i].long() & 0xFFFFFFFF
            token = torch.arange(v, device=DEV)
            x[(words[token // 32] // 2 ** (token % 32)) % 2 == 0] = -math.inf
        rows.append(x)
        tops.append(int(torch.nonzero(x == x.max())[0]) if float(x.max()) > -math.inf else -1)
    return {"logits": torch.stack(rows), "argmax": torch.tensor(tops, dtype=torch.int32)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "qk": _exact_qk, "logits": _exact_logits}[case["op"]](s)
