"""Cases for measuring the readings operators: token sampling and attention over a shared window.

``run`` computes an operator in its plain form (elementary torch operations)
where ``own`` is false, and through ``sheetsage2_refined_b200.ops`` where it is
true.  ``exact`` gives the same outputs from the definition in 64 bits.

sample: x = float32(logits) + bias over the allowed tokens, w = exp((x - max) / T);
tokens ordered by value, then index; top-k keeps the first k, top-p the
shortest prefix holding a share p of what is left, min-p those of at least
min_p of the largest; the token is the lowest index whose running sum of kept
weights exceeds u times their total; logprob is the token's log-probability
under the allowed distribution at temperature 1.

attention: every row attends over one shared K/V and then over its own paged
K/V (64-token pages); out and the log-sum-exp of the scaled scores.
"""

import math

import torch

own = False

PAGE = 64
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _sample(name, rows, vocab, dtype, temperature, top_k, top_p, min_p, per_row, masked, bias):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p, "per_row": per_row, "masked": masked, "bias": bias}


def _attention(name, rows, heads, kv_heads, dim, shared, own_max, dtype, layout):
    return {"name": name, "op": "attention", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "shared": shared, "own_max": own_max, "dtype": dtype, "layout": layout}


def listed():
    return [
        # one reading of the product vocabulary: latency of a single song's step, every filter on
        _sample("sample_1", 1, 32576, "f32", 0.8, 50, 0.95, 0.02, False, True, True),
        # 64 readings (a full batched engine) of the product vocabulary, per-reading parameters
        _sample("sample_64", 64, 32576, "f32", 0.9, 0, 0.9, 0.0, True, True, True),
        # the small synthetic vocabulary, plain temperature, no filter to find
        _sample("sample_small", 16, 2048, "f32", 1.0, 0, 1.0, 0.0, False, True, False),
        # an odd, large vocabulary in bfloat16 (many equal values), top-k then top-p
        _sample("sample_ties", 7, 131071, "bf16", 1.1, 1000, 0.9, 0.0, False, False, False),
        # a box of readings: as many rows as the allocation-free selection takes
        _sample("sample_1024", 1024, 32576, "f32", 1.0, 200, 0.98, 0.01, True, True, True),
        # one reading against one window of the 12-layer decoder: the smallest call
        _attention("attn_1", 1, 16, 16, 64, 1500, 0, "bf16", "head"),
        # 16 readings of a window, its frames not a multiple of a tile
        _attention("attn_16", 16, 16, 16, 64, 1499, 0, "bf16", "head"),
        # 64 readings of the product decoder's window: 7,500 frames, 8 heads
        _attention("attn_64", 64, 8, 8, 64, 7500, 0, "bf16", "head"),
        # 64 readings behind one prompt, each with its own generated tokens in pages
        _attention("attn_prefix", 64, 16, 16, 64, 2048, 1500, "bf16", "token"),
        # grouped heads of width 128 in half precision, short shared part, long own parts
        _attention("attn_grouped", 100, 32, 8, 128, 1111, 2500, "f16", "token"),
        # many rows over a long shared part: bound by the matrix products and exponentials
        _attention("attn_long", 1024, 16, 16, 64, 16384, 200, "bf16", "head"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    top = {"sample": max(work(c)["bytes"] for c in listed() if c["op"] == "sample"),
           "attention": max(work(c)["flops"] for c in listed() if c["op"] == "attention")}
    while True:
        if rng.random() < 0.45:
            vocab = _log_int(rng, 2, 200000)
            c = _sample("", _log_int(rng, 1, 1024), vocab, rng.choice(["f32", "bf16", "f16"]),
                        rng.choice([0.0, 0.25, 0.7, 1.0, 1.6]), rng.choice([0, 1, _log_int(rng, 1, vocab)]),
                        rng.choice([1.0, round(rng.uniform(0.05, 0.999), 3)]),
                        rng.choice([0.0, round(rng.uniform(0.001, 0.5), 3)]), rng.random() < 0.5, rng.random() < 0.7,
                        rng.random() < 0.5)
            cost = work(c)["bytes"]
        else:
            kv_heads = rng.choice([1, 2, 5, 8, 12, 16])
            dim = rng.choice([64, 128])
            c = _attention("", _log_int(rng, 1, 1024), kv_heads * rng.choice([1, 1, 2, 3, 4, 8]), kv_heads, dim,
                           _log_int(rng, 1, 16384) if rng.random() < 0.9 else 0,
                           _log_int(rng, 1, 4000) if rng.random() < 0.6 else 0,
                           rng.choice(["bf16", "f16"]), rng.choice(["head", "token"]))
            cost = work(c)["flops"]
            # the largest listed case holds 0.2 GB of own K/V; a drawn one at most 2 GB
            if 4 * c["rows"] * c["own_max"] * kv_heads * dim > 2e9 or not c["shared"] + c["own_max"]:
                continue
        if cost <= top[c["op"]]:
            del c["name"]
            return c


def _own_mean(case):
    return case["own_max"] * 0.55  # lengths are spread over 0 .. own_max, a tenth of them full


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        byte = n * (SIZE[case["dtype"]] + (1 if case["masked"] else 0)) + (4 * case["vocab"] if case["bias"] else 0)
        return {"bytes": byte + case["rows"] * (4 + 8 + 4 + (16 if case["per_row"] else 0)), "flops": 4 * n}
    r, h, g, d, s = case["rows"], case["heads"], case["kv_heads"], case["dim"], case["shared"]
    keys = s + _own_mean(case)
    return {"bytes": int(2 * 2 * g * d * (s + r * _own_mean(case)) + 2 * 2 * r * h * d + 4 * r * h),
            "flops": int(4 * r * h * d * keys)}


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    if case["op"] == "sample":
        rows, vocab, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
        # a decoder's logits: bfloat16 values, a broad bulk and a few tokens that stand out
        x = normal(rows, vocab) * 2.0
        x += 9.0 * (uniform(rows, vocab) < 12.0 / vocab)
        s = {"case": case, "logits": x.bfloat16().to(dtype), "uniforms": uniform(rows), "bias": None, "allowed": None}
        if case["bias"]:
            s["bias"] = (normal(vocab) * (uniform(vocab) < 0.01)).contiguous()
        if case["masked"]:
            # grammar classes are spans of the vocabulary, each allowed or not; now and then a row has none
            span = torch.div(torch.arange(vocab, device="cuda") * 13, vocab, rounding_mode="floor")
            allowed = (uniform(rows, 13) < 0.5)[:, span]
            s["allowed"] = (allowed & (uniform(rows, 1) > 0.02)).to(torch.uint8)
        for key, kind in (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32),
                          ("min_p", torch.float32)):
            s[key] = case[key]
            if case["per_row"]:  # each reading with its own strength of the filter
                s[key] = (case[key] * (1.0 - 0.2 * uniform(rows))).to(kind)
                if key == "top_k" and case[key] > 0:
                    s[key] = s[key].clamp(min=1)
        return s

    rows, heads, kvh, dim, dtype = case["rows"], case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]

    def projected(*shape):  # a projection's output: each channel of each head with a mean of its own
        return (normal(*shape) + normal(*shape[-2:])).to(dtype)

    s = {"case": case, "q": projected(rows, heads, dim), "own_k": None, "own_v": None, "table": None, "own_len": None}
    kv = [projected(case["shared"], kvh, dim) for _ in range(2)]
    if case["layout"] == "head":  # [heads, tokens, dim] in memory, as a window's cross K/V
        kv = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in kv]
    s["shared_k"], s["shared_v"] = kv
    if case["own_max"]:
        pages = -(-case["own_max"] // PAGE)
        n = (uniform(rows) * (case["own_max"] + 1)).int().clamp(max=case["own_max"])
        n = torch.where(uniform(rows) < 0.1, torch.full_like(n, case["own_max"]), n)
        table = torch.randperm(rows * pages, generator=gen, device="cuda").int().view(rows, pages)
        for name in ("own_k", "own_v"):
            pool = normal(rows * pages, kvh, PAGE, dim)
            s[name] = (pool + normal(kvh, 1, dim)).to(dtype)
        s["table"], s["own_len"] = table, n
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    if state["case"]["op"] == "sample":
        if own:
            from sheetsage2_refined_b200 import ops

            tokens, logprobs = ops.sample(
                state["logits"], state["uniforms"], temperature=state["temperature"], top_k=state["top_k"],
                top_p=state["top_p"], min_p=state["min_p"], bias=state["bias"], allowed=state["allowed"])
            return {"tokens": tokens, "logprobs": logprobs}
        return _plain_sample(state)
    if own:
        from sheetsage2_refined_b200 import ops

        out, lse = ops.shared_attention(
            state["q"], state["shared_k"], state["shared_v"], own_k=state["own_k"], own_v=state["own_v"],
            page_table=state["table"], own_len=state["own_len"])
        return {"out": out, "lse": lse}
    return _plain_attention(state)


def _column(value, rows, kind):
    if isinstance(value, torch.Tensor):
        return value.to(kind)[:, None]
    return torch.full((rows, 1), value, dtype=kind, device="cuda")


def _plain_sample(s):
    rows, vocab = s["logits"].shape
    x = s["logits"].float()
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["allowed"] is not None:
        x = x.masked_fill(s["allowed"] == 0, -math.inf)
    t, p, m = (_column(s[k], rows, torch.float32).double() for k in ("temperature", "top_p", "min_p"))
    k = _column(s["top_k"], rows, torch.int64)
    best = x.amax(-1, keepdim=True)
    empty = best == -math.inf
    d = torch.where(x == -math.inf, -math.inf, x - torch.where(empty, 0.0, best))
    # weights and their running sums in 64 bits: a token is chosen by which side of a border they fall on
    gap = x.double() - torch.where(empty, 0.0, best).double()
    w = torch.where(t > 0, (gap / torch.where(t > 0, t, 1.0)).exp(), (gap == 0).double())
    order = x.sort(dim=-1, descending=True, stable=True)[1]
    sorted_w = w.gather(-1, order)
    rank = torch.arange(vocab, device=x.device)[None]
    sorted_w = torch.where((k > 0) & (rank >= k), 0.0, sorted_w)
    before = sorted_w.cumsum(-1)
    keep = (p >= 1) | (rank == 0) | (before - sorted_w < p * before[:, -1:])
    keep &= sorted_w >= m
    kept = torch.zeros_like(w).scatter(-1, order, torch.where(keep, sorted_w, 0.0))
    running = kept.cumsum(-1)
    token = (running > s["uniforms"].double()[:, None] * running[:, -1:]).to(torch.uint8).argmax(-1)
    token = torch.where((t == 0) | empty, x.argmax(-1, keepdim=True), token[:, None])
    logprob = d.gather(-1, token) - d.exp().sum(-1, keepdim=True).log()
    return {"tokens": token[:, 0], "logprobs": torch.where(empty, -math.inf, logprob)[:, 0]}


def _plain_attention(s):
    case, q = s["case"], s["q"]
    rows, kvh, dim = case["rows"], case["kv_heads"], case["dim"]
    qg = q.float().view(rows, kvh, -1, dim) / math.sqrt(dim)
    k, v = s["shared_k"].float(), s["shared_v"].float()
    score = torch.einsum("rhgd,shd->rhgs", qg, k)
    if s["table"] is not None:
        # the rows' pages side by side: [rows, heads, tokens, dim]
        ok, ov = (t[s["table"].long()].float().transpose(1, 2).reshape(rows, kvh, -1, dim) for t in
                  (s["own_k"], s["own_v"]))
        mine = torch.matmul(qg, ok.transpose(-1, -2))
        gone = torch.arange(mine.shape[-1], device=q.device)[None] >= s["own_len"][:, None]
        score = torch.cat([score, mine.masked_fill(gone[:, None, None], -math.inf)], -1)
    if score.shape[-1] == 0:
        score = torch.full_like(score[..., :1].sum(-1, keepdim=True), -math.inf)
    best = score.amax(-1, keepdim=True)
    none = best == -math.inf
    weight = (score - torch.where(none, 0.0, best)).exp()
    total = weight.sum(-1, keepdim=True)
    out = torch.einsum("rhgs,shd->rhgd", weight[..., : case["shared"]], v)
    if s["table"] is not None:
        out = out + torch.matmul(weight[..., case["shared"]:], ov)
    out = torch.where(none, 0.0, out / torch.where(none, 1.0, total))
    lse = torch.where(none, -math.inf, best + total.log())
    return {"out": out.reshape(q.shape).to(q.dtype), "lse": lse.reshape(rows, -1)}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return _exact_sample(s) if case["op"] == "sample" else _exact_attention(s)


def _exact_sample(s):
    rows, vocab = s["logits"].shape
    tokens, logprobs = [], []
    for r in range(rows):
        x = s["logits"][r].float()
        if s["bias"] is not None:
            x = x + s["bias"]
        x = x.double()
        index = torch.arange(vocab, device=x.device)
        if s["allowed"] is not None:
            index = index[s["allowed"][r] != 0]
            x = x[index]
        t, k, p, m = (float(v[r]) if isinstance(v, torch.Tensor) else float(torch.tensor(v, dtype=torch.float32))
                      for v in (s["temperature"], s["top_k"], s["top_p"], s["min_p"]))
        if not x.numel():
            tokens.append(torch.zeros((), dtype=torch.int64, device="cuda"))
            logprobs.append(torch.full((), -math.inf, dtype=torch.float64, device="cuda"))
            continue
        value, at = torch.sort(x, descending=True, stable=True)
        rank = torch.arange(len(value), device=x.device)
        w = torch.exp((value - value[0]) / t) if t > 0 else (rank == 0).double()
        if k > 0:
            w = w * (rank < k)
        run_sum = torch.cumsum(w, 0)
        if p < 1:
            w = w * ((run_sum - w < p * run_sum[-1]) | (rank == 0))
        w = w * (w >= m)
        by_index = torch.zeros_like(w)
        by_index[at] = w
        total = torch.cumsum(by_index, 0)
        pick = torch.searchsorted(total, (s["uniforms"][r].double() * total[-1]).reshape(1), right=True)[0]
        pick = pick.clamp(max=len(value) - 1)
        tokens.append(index[pick])
        logprobs.append(x[pick] - torch.logsumexp(x, 0))
    return {"tokens": torch.stack(tokens), "logprobs": torch.stack(logprobs)}


def _exact_attention(s):
    case = s["case"]
    rows, heads, kvh, dim = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(rows, heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64, device="cuda")
    for h in range(heads):
        g = h // (heads // kvh)
        q = s["q"][:, h].double() * dim ** -0.5
        parts = [(q @ s["shared_k"][:, g].double().t(), None)]
        if s["table"] is not None:
            pages = s["table"].long()
            k = s["own_k"][:, g][pages].double().flatten(1, 2)
            v = s["own_v"][:, g][pages].double().flatten(1, 2)
            score = (k @ q[:, :, None])[..., 0]
            seen = torch.arange(k.shape[1], device="cuda") < s["own_len"][:, None]
            parts.append((torch.where(seen, score, -math.inf), v))
        total = torch.logsumexp(torch.cat([p for p, _ in parts], -1), -1)
        live = total > -math.inf
        shift = torch.where(live, total, 0.0)[:, None]
        o = torch.exp(parts[0][0] - shift) @ s["shared_v"][:, g].double()
        if s["table"] is not None:
            o = o + (torch.exp(parts[1][0] - shift)[:, None] @ parts[1][1])[:, 0]
        out[:, h] = o
        lse[:, h] = total
    return {"out": out, "lse": lse}
