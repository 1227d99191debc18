"""What the language-model operators are measured on: norm, 8-bit products and sampling.

Plain forms in elementary torch operations (32 bits, rounded once at the end), the
calls of pdefa_b200 that replace them (`own` true), and 64-bit definitions.
"""
import math

import torch

own = False

BLOCK = 128          # values that share a scale
E4M3_MAX = 448.0
TINY = 1e-10         # least row maximum that a scale is derived from
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ----------------------------------------------------------------------------
# Cases
# ----------------------------------------------------------------------------
def listed():
    return [
        # one new token before a projection: latency
        {"name": "norm_token", "op": "norm", "rows": 1, "cols": 4096, "dtype": "bf16", "residual": True, "fp8": True},
        # a batch of odd size and width, no residual (a first or last norm), 16-bit output
        {"name": "norm_odd", "op": "norm", "rows": 509, "cols": 2050, "dtype": "f16", "residual": False, "fp8": False},
        # a long prompt
        {"name": "norm_prompt", "op": "norm", "rows": 16384, "cols": 8192, "dtype": "bf16", "residual": True,
         "fp8": True},
        # a projection for a few new tokens: reading the weights
        {"name": "matmul_tokens", "op": "matmul", "m": 8, "n": 4096, "k": 4096, "out": "bf16"},
        # nothing a multiple of the tiles; the last blocks of n and k are partial
        {"name": "matmul_odd", "op": "matmul", "m": 333, "n": 1201, "k": 2000, "out": "f32"},
        # a projection for a long prompt
        {"name": "matmul_prompt", "op": "matmul", "m": 8192, "n": 8192, "k": 4096, "out": "bf16"},
        # 8 tokens with 8 experts each: about 40 of the 64 experts get rows, most of them one or two
        {"name": "grouped_tokens", "op": "grouped", "rows": 64, "experts": 64, "n": 2048, "k": 2048, "skew": 0.0,
         "out": "bf16"},
        # odd sizes, uneven experts, some of them empty
        {"name": "grouped_odd", "op": "grouped", "rows": 1003, "experts": 17, "n": 1041, "k": 912, "skew": 1.0,
         "out": "f32"},
        # a long prompt's rows over all experts, unevenly
        {"name": "grouped_prompt", "op": "grouped", "rows": 16384, "experts": 32, "n": 4096, "k": 2048, "skew": 0.5,
         "out": "bf16"},
        # one request: latency
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": 32000, "dtype": "bf16", "filters": "all",
         "masked": 0.0},
        # requests with different settings in one batch, a third of the vocabulary ruled out by a grammar
        {"name": "sample_mixed", "op": "sample", "rows": 33, "vocab": 50257, "dtype": "f32", "filters": "mixed",
         "masked": 0.3},
        # a full server
        {"name": "sample_batch", "op": "sample", "rows": 256, "vocab": 131072, "dtype": "bf16", "filters": "all",
         "masked": 0.0},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "matmul", "grouped", "sample"))
    if op == "norm":
        cols = _log_uniform(rng, 256, 16384)
        return {"op": op, "rows": _log_uniform(rng, 1, min(16384, (16384 * 8192) // cols)), "cols": cols,
                "dtype": rng.choice(("bf16", "bf16", "f16", "f32")) if cols <= 4096 else "bf16",
                "residual": rng.random() < 0.7, "fp8": rng.random() < 0.6}
    if op == "matmul":
        n, k = _log_uniform(rng, 256, 8192), 16 * _log_uniform(rng, 16, 512)
        return {"op": op, "m": _log_uniform(rng, 1, min(8192, (8192 * 8192 * 4096) // (n * k))), "n": n, "k": k,
                "out": rng.choice(("bf16", "bf16", "f16", "f32")) if n <= 4096 else "bf16"}
    if op == "grouped":
        e = _log_uniform(rng, 4, 64)
        n, k = _log_uniform(rng, 256, 4096), 16 * _log_uniform(rng, 16, 128)
        return {"op": op, "rows": _log_uniform(rng, 1, 8192), "experts": e, "n": n, "k": k,
                "skew": rng.choice((0.0, 0.5, 1.0)), "out": rng.choice(("bf16", "f16"))}
    vocab = _log_uniform(rng, 1000, 131072)
    return {"op": op, "rows": _log_uniform(rng, 1, 128), "vocab": vocab, "dtype": rng.choice(("bf16", "f16", "f32")),
            "filters": rng.choice(("all", "mixed", "none")), "masked": rng.choice((0.0, 0.3))}


# ----------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def _e4m3(g, *shape):
    """8-bit values as quantisation by the block's largest value leaves them."""
    return (_randn(g, *shape) * 120.0).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _blocks(n):
    return -(-n // BLOCK)


def _shares(case):
    """Each expert's share of the rows: even, or falling with the expert's rank."""
    w = [1.0 / (i + 1) ** case["skew"] for i in range(case["experts"])]
    return [x / sum(w) for x in w]


def _filters(case):
    """Per-row settings (temperature, top_k, top_p, min_p); 0, 1 and 0 turn the last three off."""
    every = {"all": [(0.8, 50, 0.9, 0.02)], "none": [(1.0, 0, 1.0, 0.0)],
             "mixed": [(0.7, 40, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 0.95, 0.0), (1.2, 0, 1.0, 0.05),
                       (1.0, 0, 1.0, 0.0), (0.6, 200, 0.8, 0.0)]}[case["filters"]]
    return [every[i % len(every)] for i in range(case["rows"])]


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    s = {"case": case, "op": op}
    if op == "norm":
        dt, t, c = DT[case["dtype"]], case["rows"], case["cols"]
        # a stream of hidden states whose rows differ in size, as they do along a model's depth
        size = torch.exp2(_rand(g, t, 1) * 6 - 2)
        s["x"] = (_randn(g, t, c) * size).to(dt)
        s["residual"] = (_randn(g, t, c) * size).to(dt) if case["residual"] else None
        s["weight"] = (1.0 + 0.2 * _randn(g, c)).to(dt)
    elif op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["b"] = _e4m3(g, m, k), _e4m3(g, n, k)
        s["a_scales"] = 0.002 + 0.01 * _rand(g, m, _blocks(k))
        s["b_scales"] = 0.0001 + 0.0003 * _rand(g, _blocks(n), _blocks(k))
    elif op == "grouped":
        t, e, n, k = case["rows"], case["experts"], case["n"], case["k"]
        s["a"], s["b"] = _e4m3(g, t, k), torch.empty(e, n, k, dtype=torch.float8_e4m3fn, device="cuda")
        for i in range(e):
            s["b"][i] = _e4m3(g, n, k)
        s["a_scales"] = 0.002 + 0.01 * _rand(g, t, _blocks(k))
        s["b_scales"] = 0.0001 + 0.0003 * _rand(g, e, _blocks(n), _blocks(k))
        share = torch.tensor(_shares(case), device="cuda")[torch.randperm(e, generator=g, device="cuda")]
        expert = torch.multinomial(share, t, replacement=True, generator=g)
        counts = torch.bincount(expert, minlength=e)
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    else:
        b, v = case["rows"], case["vocab"]
        x = _randn(g, b, v) * 2.5
        x += 6.0 * (_rand(g, b, v) < 20.0 / v)      # the few tokens that fit the context
        if case["masked"]:
            x.masked_fill_(_rand(g, b, v) < case["masked"], -math.inf)
        s["logits"] = x.to(DT[case["dtype"]])
        s["noise"] = torch.empty(b, v, device="cuda").exponential_(generator=g)
        t, k, p, m = zip(*_filters(case))
        s["temperature"] = torch.tensor(t, device="cuda", dtype=torch.float32)
        s["top_k"] = torch.tensor(k, device="cuda", dtype=torch.int32)
        s["top_p"] = torch.tensor(p, device="cuda", dtype=torch.float32)
        s["min_p"] = torch.tensor(m, device="cuda", dtype=torch.float32)
    return s


# ----------------------------------------------------------------------------
# Plain forms
# ----------------------------------------------------------------------------
EPS = 1e-6


def _plain_norm(s):
    case = s["case"]
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    r = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    y = h * r * s["weight"].float()
    out = {}
    if s["residual"] is not None:
        out["h"] = h.to(s["x"].dtype)
    if case["fp8"]:
        t, c = y.shape
        nb = _blocks(c)
        pad = torch.nn.functional.pad(y, (0, nb * BLOCK - c)).view(t, nb, BLOCK)
        scales = pad.abs().amax(-1).clamp(min=TINY) / E4M3_MAX
        q = (pad / scales[..., None]).clamp(-E4M3_MAX, E4M3_MAX).view(t, nb * BLOCK)[:, :c]
        out["q"], out["scales"] = q.to(torch.float8_e4m3fn), scales
    else:
        out["y"] = y.to(s["x"].dtype)
    return out


def _values(q, scales):
    """8-bit values times the scale of their 128 columns."""
    k = q.shape[-1]
    return q.float() * scales.repeat_interleave(BLOCK, -1)[..., :k]


def _weights(q, scales):
    """8-bit weights times the scale of their 128 x 128 block."""
    n = q.shape[-2]
    return _values(q, scales.repeat_interleave(BLOCK, -2)[..., :n, :])


def _plain_matmul(s):
    out = _values(s["a"], s["a_scales"]) @ _weights(s["b"], s["b_scales"]).transpose(-1, -2)
    return {"out": out.to(DT[s["case"]["out"]])}


def _plain_grouped(s):
    # each expert's rows padded to the longest group, one batched product, rows put back
    off = s["offsets"].long()
    counts = off[1:] - off[:-1]
    t = s["a"].shape[0]
    at = torch.arange(t, device="cuda")
    expert = torch.searchsorted(off[1:], at, right=True)
    slot = at - off[expert]
    most = int(counts.max())
    a = _values(s["a"], s["a_scales"])
    rows = a.new_zeros(counts.numel(), most, a.shape[1])
    rows[expert, slot] = a
    out = rows @ _weights(s["b"], s["b_scales"]).transpose(-1, -2)
    return {"out": out[expert, slot].to(DT[s["case"]["out"]])}


def _plain_sample(s):
    x = s["logits"].float()
    v = x.shape[1]
    greedy = s["temperature"] == 0
    t = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"])[:, None]
    k = torch.where(greedy, torch.ones_like(s["top_k"]), s["top_k"])[:, None]
    w = torch.exp((x - x.amax(-1, keepdim=True)) / t)
    total = w.sum(-1, keepdim=True)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    sw = w.gather(-1, order)
    before = sw.cumsum(-1) - sw
    rank = torch.arange(v, device=x.device)[None]
    p, m = s["top_p"][:, None], s["min_p"][:, None]
    keep = ((k <= 0) | (rank < k)) & ((p >= 1) | (before < p * total)) & (sw >= m) & (sw > 0)
    race = torch.where(keep, sw / s["noise"].gather(-1, order), torch.full_like(sw, -1.0))
    best = race.amax(-1, keepdim=True)
    token = torch.where(race == best, order, torch.full_like(order, v)).amin(-1, keepdim=True)
    prob = w.gather(-1, token) / total
    return {"token": token[:, 0].to(torch.int32), "prob": prob[:, 0]}


# ----------------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------------
def run(s):
    op = s["op"]
    if not own:
        return {"norm": _plain_norm, "matmul": _plain_matmul, "grouped": _plain_grouped, "sample": _plain_sample}[op](s)
    import pdefa_b200 as pb
    if op == "norm":
        if s["case"]["fp8"]:
            got = pb.ops_rms_norm_fp8(s["x"], s["weight"], residual=s["residual"], eps=EPS)
            return dict(zip(("q", "scales", "h"), got))
        got = pb.ops_rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        return {"y": got} if s["residual"] is None else dict(zip(("y", "h"), got))
    if op == "matmul":
        return {"out": pb.ops_matmul_fp8(s["a"], s["a_scales"], s["b"], s["b_scales"],
                                         out_dtype=DT[s["case"]["out"]])}
    if op == "grouped":
        return {"out": pb.ops_matmul_grouped_fp8(s["a"], s["a_scales"], s["b"], s["b_scales"], s["offsets"],
                                                 out_dtype=DT[s["case"]["out"]])}
    return dict(zip(("token", "prob"),
                    pb.ops_sample(s["logits"], s["noise"], temperature=s["temperature"], top_k=s["top_k"],
                                  top_p=s["top_p"], min_p=s["min_p"])))


# ----------------------------------------------------------------------------
# What a pass cannot do without
# ----------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "norm":
        t, c, e = case["rows"], case["cols"], SIZE[case["dtype"]]
        read = t * c * e * (2 if case["residual"] else 1) + c * e
        write = (t * c * e if case["residual"] else 0) + (t * (c + 4 * _blocks(c)) if case["fp8"] else t * c * e)
        return {"bytes": read + write, "flops": 6 * t * c}
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + _blocks(n)) * _blocks(k) + m * n * SIZE[case["out"]],
                "flops": 2 * m * n * k}
    if op == "grouped":
        t, n, k = case["rows"], case["n"], case["k"]
        active = sum(1 - (1 - p) ** t for p in _shares(case))      # experts that get a row
        return {"bytes": t * k + active * (n * k + 4 * _blocks(n) * _blocks(k)) + 4 * t * _blocks(k)
                + 4 * (case["experts"] + 1) + t * n * SIZE[case["out"]], "flops": 2 * t * n * k}
    b, v = case["rows"], case["vocab"]
    free = sum(t > 0 and k <= 0 and p >= 1 and m <= 0 for t, k, p, m in _filters(case))   # every token's variate counts
    return {"bytes": b * v * SIZE[case["dtype"]] + free * v * 4 + b * 24, "flops": 4 * b * v}


# ----------------------------------------------------------------------------
# The definitions in 64 bits (floating outputs unrounded)
# ----------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        rows = []
        for lo in range(0, case["rows"], 2048):
            h = s["x"][lo:lo + 2048].double()
            if s["residual"] is not None:
                h += s["residual"][lo:lo + 2048].double()
            y = s["weight"].double() * h / ((h * h).sum(1, keepdim=True) / case["cols"] + EPS).sqrt()
            got = {} if s["residual"] is None else {"h": h}
            if case["fp8"]:
                parts = torch.split(y, BLOCK, dim=1)
                sc = torch.stack([torch.maximum(q.abs().max(1).values, torch.tensor(TINY, device="cuda").double())
                                  for q in parts], 1) / E4M3_MAX
                got["scales"] = sc
                got["q"] = torch.cat([q / sc[:, i:i + 1] for i, q in enumerate(parts)], 1)
            else:
                got["y"] = y
            rows.append(got)
        return {key: torch.cat([r[key] for r in rows]) for key in rows[0]}
    if op in ("matmul", "grouped"):
        k, n = case["k"], case["n"]
        kb = torch.arange(k, device="cuda") // BLOCK
        nb = torch.arange(n, device="cuda") // BLOCK
        a = s["a"].double() * s["a_scales"].double()[:, kb]
        if op == "matmul":
            return {"out": a @ (s["b"].double() * s["b_scales"].double()[nb][:, kb]).t()}
        out = torch.zeros(case["rows"], n, dtype=torch.float64, device="cuda")
        off = s["offsets"].tolist()
        for i in range(case["experts"]):
            if off[i + 1] > off[i]:
                w = s["b"][i].double() * s["b_scales"][i].double()[nb][:, kb]
                out[off[i]:off[i + 1]] = a[off[i]:off[i + 1]] @ w.t()
        return {"out": out}
    # one row at a time: walk the sorted row until a filter ends it, then the race among those kept
    tokens, probs = [], []
    for i, (t, k, p, m) in enumerate(_filters(case)):
        x = s["logits"][i].double()
        t, k = (1.0, 1) if t == 0 else (float(torch.tensor(t)), k)
        p, m = float(torch.tensor(p)), float(torch.tensor(m))
        w = ((x - x.max()) / t).exp()
        z = w.sum()
        sw, order = torch.sort(w, descending=True, stable=True)      # w rises with x, so the order is x's
        n = int((sw > 0).sum()) if m <= 0 else int((sw >= m).sum())
        if k > 0:
            n = min(n, k)
        if p < 1:
            n = min(n, 1 + int((sw.cumsum(0) < p * z).sum()))
        kept = order[:n]
        token = kept[int(torch.argmax(sw[:n] / s["noise"][i][kept].double()))]
        tokens.append(token)
        probs.append(w[token] / z)
    return {"token": torch.stack(tokens).to(torch.int32), "prob": torch.stack(probs)}
