"""Operators of served language models, as cases that can be timed and compared with their plain forms.

Three kinds, products of tokens whose weights each token names:

* ``route``: the choice of experts from router logits (``ops.moe.route``), whose answer the dispatch and the experts take.
* ``experts``: a whole mixture-of-experts layer for a few tokens, bf16 or block-scaled e4m3 weights (``ops.moe.MoeExperts``).
* ``lora``: the low-rank adapters of many requests at once, added to what a shared projection gave (``ops.lora.LoraAdapters``).
"""
import math

import torch

own = False

DEVICE = "cuda"
BLOCK = 128  # rows and columns of a weight that share a scale


def listed():
    return [
        # one token of a single conversation
        {"name": "route_1_token", "kind": "route", "tokens": 1, "experts": 256, "topk": 8, "scoring": "softmax", "bias": False,
         "groups": 1, "topk_groups": 1, "dtype": "f32"},
        # a prefill batch, experts chosen within the best groups by scores with a balancing bias
        {"name": "route_4096_tokens_in_groups", "kind": "route", "tokens": 4096, "experts": 256, "topk": 8, "scoring": "sigmoid", "bias": True,
         "groups": 8, "topk_groups": 4, "dtype": "f32"},
        # one token through a small layer: latency
        {"name": "experts_1_token_small", "kind": "experts", "tokens": 1, "hidden": 2048, "inner": 768, "experts": 64, "total": 64, "topk": 8,
         "dtype": "bf16", "absent": 0.0},
        # one token through a large layer
        {"name": "experts_1_token", "kind": "experts", "tokens": 1, "hidden": 7168, "inner": 2048, "experts": 32, "total": 32, "topk": 8,
         "dtype": "bf16", "absent": 0.0},
        # sizes that divide nothing, and slots without an expert
        {"name": "experts_37_tokens_ragged", "kind": "experts", "tokens": 37, "hidden": 1928, "inner": 1000, "experts": 40, "total": 40, "topk": 6,
         "dtype": "bf16", "absent": 0.1},
        # few and wide experts, many tokens for each
        {"name": "experts_64_tokens_wide", "kind": "experts", "tokens": 64, "hidden": 4096, "inner": 8192, "experts": 8, "total": 8, "topk": 2,
         "dtype": "bf16", "absent": 0.0},
        # one GPU's 32 of 256 experts in a decode batch
        {"name": "experts_128_tokens_share", "kind": "experts", "tokens": 128, "hidden": 7168, "inner": 2048, "experts": 32, "total": 256, "topk": 8,
         "dtype": "bf16", "absent": 0.0},
        # the same with e4m3 weights
        {"name": "experts_128_tokens_share_e4m3", "kind": "experts", "tokens": 128, "hidden": 7168, "inner": 2048, "experts": 32, "total": 256,
         "topk": 8, "dtype": "e4m3", "absent": 0.0},
        # one request's token
        {"name": "lora_1_token", "kind": "lora", "tokens": 1, "k": 4096, "n": 4096, "rank": 16, "adapters": 32, "run": 1, "absent": 0.0},
        # a decode batch: every token another request's, some without an adapter
        {"name": "lora_64_tokens", "kind": "lora", "tokens": 64, "k": 8192, "n": 8192, "rank": 16, "adapters": 64, "run": 1, "absent": 0.1},
        # short prompts of several requests, odd sizes, larger ranks
        {"name": "lora_777_tokens_ragged", "kind": "lora", "tokens": 777, "k": 7168, "n": 2056, "rank": 40, "adapters": 24, "run": 61, "absent": 0.1},
        # a prefill batch of a few long prompts
        {"name": "lora_8192_tokens", "kind": "lora", "tokens": 8192, "k": 8192, "n": 8192, "rank": 16, "adapters": 16, "run": 1500, "absent": 0.0},
    ]


def _spread(rng, low, high, step=1):
    """A multiple of `step` from low to high, spread over its logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["route", "experts", "experts", "experts", "lora", "lora"])
    if kind == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * _spread(rng, 8, 512 // groups)
        scoring = rng.choice(["softmax", "sigmoid"])
        return {"kind": kind, "tokens": _spread(rng, 1, 4096), "experts": experts, "topk": rng.randint(1, 8), "scoring": scoring,
                "bias": rng.random() < 0.5, "groups": groups, "topk_groups": max(1, groups // 2), "dtype": rng.choice(["f32", "bf16"])}
    if kind == "experts":
        topk = rng.randint(1, 8)
        experts = _spread(rng, 8, 64)
        total = experts * rng.choice([1, 1, 8])
        hidden, inner, dtype = _spread(rng, 1024, 7168, 16), _spread(rng, 512, 4096, 16), rng.choice(["bf16", "bf16", "e4m3"])
        while experts * hidden * inner > 32 * 7168 * 2048:
            inner = max(256, inner // 32 * 16)
            experts, total = max(8, experts // 2), max(8, total // 2)
        return {"kind": kind, "tokens": _spread(rng, 1, 128), "hidden": hidden, "inner": inner, "experts": experts, "total": total, "topk": topk,
                "dtype": dtype, "absent": rng.choice([0.0, 0.1])}
    tokens = _spread(rng, 1, 8192)
    run = 1 if tokens <= 256 else _spread(rng, 32, 2048)
    return {"kind": kind, "tokens": tokens, "k": _spread(rng, 1024, 8192, 8), "n": _spread(rng, 1024, 8192, 8), "rank": rng.choice([8, 16, 16, 32, 40, 64]),
            "adapters": _spread(rng, 2, 64 if tokens <= 256 else 16), "run": run, "absent": rng.choice([0.0, 0.1])}


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"route": _prepare_route, "experts": _prepare_experts, "lora": _prepare_lora}[case["kind"]](case, g)


def run(state):
    return {"route": _run_route, "experts": _run_experts, "lora": _run_lora}[state["kind"]](state)


def work(case):
    return {"route": _work_route, "experts": _work_experts, "lora": _work_lora}[case["kind"]](case)


def exact(case, seed):
    return {"route": _exact_route, "experts": _exact_experts, "lora": _exact_lora}[case["kind"]](prepare(case, seed))


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=dtype)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEVICE)


# ---- route ----

def _prepare_route(case, g):
    t, e = case["tokens"], case["experts"]
    logits = _randn(g, t, e) * 1.5 + 0.5 * _randn(g, e)  # some experts are more popular than others
    return {"kind": "route", "logits": logits.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32), "topk": case["topk"],
            "scoring": case["scoring"], "bias": 0.05 * _randn(g, e) if case["bias"] else None, "groups": case["groups"],
            "topk_groups": case["topk_groups"], "scale": 2.5}


def _run_route(s):
    if own:
        from execution_ucx_b200.ops import moe
        idx, w = moe.route(s["logits"], s["topk"], scoring=s["scoring"], bias=s["bias"], groups=s["groups"], topk_groups=s["topk_groups"],
                           renormalize=True, scale=s["scale"])
        return {"idx": idx, "w": w}
    # in 64 bits: experts whose scores are next to each other
    logits = s["logits"].double()
    t, e = logits.shape
    if s["scoring"] == "softmax":
        scores = torch.exp(logits - logits.amax(-1, keepdim=True))
        scores = scores / scores.sum(-1, keepdim=True)
    else:
        scores = 1 / (1 + torch.exp(-logits))
    choice = scores if s["bias"] is None else scores + s["bias"].double()
    if s["bias"] is None and s["groups"] == 1:
        choice = logits
    if s["groups"] > 1:
        best = choice.view(t, s["groups"], -1).sort(dim=-1, descending=True, stable=True).values[..., :2].sum(-1)
        kept = best.sort(dim=-1, descending=True, stable=True).indices[:, :s["topk_groups"]]
        open_ = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        choice = choice.masked_fill(~open_.repeat_interleave(e // s["groups"], dim=1), -math.inf)
    idx = choice.sort(dim=-1, descending=True, stable=True).indices[:, :s["topk"]]
    w = scores.gather(1, idx)
    w = w / w.sum(-1, keepdim=True) * s["scale"]
    return {"idx": idx.to(torch.int32), "w": w.float()}


def _exact_route(s):
    logits = s["logits"].cpu().double()
    bias = None if s["bias"] is None else s["bias"].cpu().double()
    t, e = logits.shape
    size = e // s["groups"]
    p = torch.softmax(logits, -1) if s["scoring"] == "softmax" else torch.sigmoid(logits)
    c = p if bias is None else p + bias
    if bias is None and s["groups"] == 1:
        c = logits
    if s["groups"] > 1:
        parts = c.reshape(t * s["groups"], size).topk(min(2, size), -1).values.sum(-1).reshape(t, s["groups"])
        # the place of each group: how many are ahead of it
        ahead = (parts[:, None, :] > parts[:, :, None]).sum(-1)
        c = torch.where((ahead < s["topk_groups"]).repeat_interleave(size, 1), c, torch.tensor(-math.inf, dtype=torch.float64))
    idx = torch.argsort(-c, dim=-1, stable=True)[:, :s["topk"]]
    w = torch.take_along_dim(p, idx, 1)
    return {"idx": idx.to(torch.int32), "w": s["scale"] * w / w.sum(-1, keepdim=True)}


def _work_route(case):
    t, e = case["tokens"], case["experts"]
    return {"bytes": t * e * (2 if case["dtype"] == "bf16" else 4) + t * case["topk"] * 8 + (4 * e if case["bias"] else 0), "flops": 4 * t * e}


# ---- experts ----

def _weight(g, e, rows, cols, dtype):
    """Weights of e experts, and the scales of their blocks (None for bf16)."""
    if dtype == "bf16":
        return _randn(g, e, rows, cols, dtype=torch.bfloat16) * cols ** -0.5, None
    q = torch.empty(e, rows, cols, dtype=torch.float8_e4m3fn, device=DEVICE)
    for i in range(e):
        q[i] = (_randn(g, rows, cols) * 96).clamp_(-448, 448).to(torch.float8_e4m3fn)
    scale = (0.5 + _rand(g, e, -(-rows // BLOCK), -(-cols // BLOCK))) * (cols ** -0.5 / 96)
    return q, scale


def _prepare_experts(case, g):
    t, h, i, e, k = case["tokens"], case["hidden"], case["inner"], case["experts"], case["topk"]
    gate_up, gate_up_scale = _weight(g, e, 2 * i, h, case["dtype"])
    down, down_scale = _weight(g, e, h, i, case["dtype"])
    logits = _randn(g, t, case["total"]) + 0.5 * _randn(g, case["total"])
    top = logits.topk(k, -1)
    idx = top.indices - (case["total"] - e) // 2  # this GPU's experts lie in the middle of them all
    idx = torch.where(_rand(g, t, k) < case["absent"], -1, idx).to(torch.int32)
    s = {"kind": "experts", "x": _randn(g, t, h).to(torch.bfloat16), "idx": idx, "w": torch.softmax(top.values, -1), "gate_up": gate_up,
         "gate_up_scale": gate_up_scale, "down": down, "down_scale": down_scale, "layer": None}
    if own:
        from execution_ucx_b200.ops import moe
        s["layer"] = moe.MoeExperts(gate_up, down, gate_up_scale=gate_up_scale, down_scale=down_scale)
    return s


def _dequantized(q, scale):
    if scale is None:
        return q.float()
    rows, cols = q.shape[1:]
    full = scale.repeat_interleave(BLOCK, 1)[:, :rows].repeat_interleave(BLOCK, 2)[:, :, :cols]
    return q.float() * full


def _picked(s, name, idx):
    scale = s[name + "_scale"]
    return _dequantized(s[name][idx], None if scale is None else scale[idx])


def _run_experts(s):
    if own:
        return s["layer"](s["x"], s["idx"], s["w"])
    x, w = s["x"].float(), s["w"]
    t, k = w.shape
    e, h, inner = s["down"].shape
    here = (s["idx"] >= 0) & (s["idx"] < e)
    idx, w = s["idx"].clamp(0, e - 1).long(), torch.where(here, w, 0.0)
    if t * k <= e:  # each entry's own weights
        gu = torch.bmm(_picked(s, "gate_up", idx.view(-1)), x.repeat_interleave(k, 0).unsqueeze(-1)).squeeze(-1)
        gate, up = gu[:, :inner], gu[:, inner:]
        y = torch.bmm(_picked(s, "down", idx.view(-1)), (gate / (1 + torch.exp(-gate)) * up).unsqueeze(-1)).squeeze(-1)
        y = (y.view(t, k, h) * w.unsqueeze(-1)).sum(1)
    else:  # every token through every expert
        per_expert = torch.zeros(t, e, device=x.device).scatter_add_(1, idx, w)
        gu = torch.matmul(x, _dequantized(s["gate_up"], s["gate_up_scale"]).transpose(1, 2))  # [e, t, 2 * inner]
        gate, up = gu[..., :inner], gu[..., inner:]
        y = torch.bmm(gate / (1 + torch.exp(-gate)) * up, _dequantized(s["down"], s["down_scale"]).transpose(1, 2))
        y = (y * per_expert.t().unsqueeze(-1)).sum(0)
    return y.to(torch.bfloat16)


def _exact_experts(s):
    x, idx, w = s["x"].double(), s["idx"], s["w"].double()
    e, h, inner = s["down"].shape
    y = torch.zeros(x.shape[0], h, dtype=torch.float64, device=x.device)

    def full(name, j):
        m = s[name][j].double()
        if s[name + "_scale"] is not None:
            m = m * torch.kron(s[name + "_scale"][j].double(), torch.ones(BLOCK, BLOCK, dtype=torch.float64, device=x.device))[:m.shape[0], :m.shape[1]]
        return m

    for j in range(e):
        rows, slots = (idx == j).nonzero(as_tuple=True)
        if len(rows):
            up = full("gate_up", j) @ x[rows].t()
            hidden = torch.nn.functional.silu(up[:inner]) * up[inner:]
            y.index_add_(0, rows, (full("down", j) @ hidden).t() * w[rows, slots].unsqueeze(1))
    return y


def _named(count, share, draws):
    """How many of `count` things `draws` independent draws name, each naming one with the probability `share`."""
    return count * (1 - (1 - share) ** draws)


def _work_experts(case):
    t, h, i, e, k = case["tokens"], case["hidden"], case["inner"], case["experts"], case["topk"]
    used = _named(e, k * (1 - case["absent"]) / case["total"], t)
    entries = t * k * (1 - case["absent"]) * e / case["total"]
    per_weight = 2 if case["dtype"] == "bf16" else 1 + 4 / BLOCK ** 2
    return {"bytes": used * 3 * h * i * per_weight + 4 * t * h + 8 * t * k, "flops": 6 * h * i * entries}


# ---- lora ----

def _prepare_lora(case, g):
    m, k, n, r, count = case["tokens"], case["k"], case["n"], case["rank"], case["adapters"]
    a = _randn(g, count, r, k, dtype=torch.bfloat16) * k ** -0.5
    b = _randn(g, count, n, r, dtype=torch.bfloat16) * r ** -0.5
    runs = -(-m // case["run"])  # consecutive tokens belong to one request
    ids = torch.randint(0, count, (runs,), generator=g, device=DEVICE)
    ids = torch.where(_rand(g, runs) < case["absent"], -1, ids).repeat_interleave(case["run"])[:m].to(torch.int32)
    scale = 0.5 + _rand(g, count)
    s = {"kind": "lora", "x": _randn(g, m, k).to(torch.bfloat16), "y": _randn(g, m, n).to(torch.bfloat16), "ids": ids, "a": a, "b": b, "scale": scale,
         "adapters": None}
    if own:
        from execution_ucx_b200.ops import lora
        s["adapters"] = lora.LoraAdapters(a, b, scale)
    return s


def _run_lora(s):
    if own:
        return s["adapters"](s["x"], s["ids"], s["y"])
    count, r, k = s["a"].shape
    m, n = s["y"].shape
    here = s["ids"] >= 0
    down = torch.matmul(s["x"].float(), s["a"].float().view(count * r, k).t()).view(m, count, r)
    mine = torch.arange(count, device=down.device) == s["ids"].unsqueeze(1)
    down = torch.where(mine.unsqueeze(-1), down, 0.0) * (s["scale"][s["ids"].clamp(min=0).long()] * here).view(m, 1, 1)
    delta = torch.matmul(down.view(m, count * r), s["b"].float().transpose(1, 2).reshape(count * r, n))
    return (s["y"].float() + delta).to(torch.bfloat16)


def _exact_lora(s):
    out = s["y"].double()
    for j in range(s["a"].shape[0]):
        rows = (s["ids"] == j).nonzero().squeeze(1)
        if len(rows):
            v = s["x"][rows].double() @ s["a"][j].double().t()
            out[rows] += s["scale"][j].double() * (v @ s["b"][j].double().t())
    return out


def _work_lora(case):
    m, k, n, r = case["tokens"], case["k"], case["n"], case["rank"]
    with_one = m * (1 - case["absent"])
    used = _named(case["adapters"], (1 - case["absent"]) / case["adapters"], -(-m // case["run"]))
    return {"bytes": 2 * (with_one * k + 2 * m * n + used * r * (k + n)) + 4 * m, "flops": 2 * with_one * r * (k + n)}
