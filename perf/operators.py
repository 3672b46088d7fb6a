"""The operators that stand beside the routed-MoE layer, as cases to time and compare.

Kinds:

  route    logits of `tokens` tokens to picks and weights (osm_route_experts):
           softmax or sigmoid scores, a bias for balance, groups, top-k,
           renormalised and scaled weights
  group    rows grouped by a small key, in their order (osm_group_rows): the
           (token, expert) pairs of a routed batch, or a batch's tokens by
           their adapter
  project  a q4 projection of `tokens` tokens with a low-rank adapter of each
           token's own beside it (osm_q4_project)

`own` says which side run() computes: the plain forms in elementary torch
operations, or the framework's calls. Inputs come from the seed alone.
"""

import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

own = False

FLOATS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # One token of a model with grouped sigmoid routing: latency alone counts.
        dict(name="route_1_groups", kind="route", tokens=1, experts=256, top_k=8, score="sigmoid", bias=True, groups=8,
             top_groups=4, group_score=2, scale=2.5, dtype="f32"),
        # A ragged decode batch of the softmax model this repository benchmarks, logits in bf16 (ties are common).
        dict(name="route_157_softmax", kind="route", tokens=157, experts=512, top_k=10, score="softmax", bias=False,
             groups=1, top_groups=1, group_score=1, scale=1.0, dtype="bf16"),
        # A prompt through grouped sigmoid routing.
        dict(name="route_4096_groups", kind="route", tokens=4096, experts=256, top_k=8, score="sigmoid", bias=True,
             groups=8, top_groups=4, group_score=2, scale=2.5, dtype="f32"),
        # Several prompts at once, softmax scores of 512 experts with a bias, no groups.
        dict(name="route_16383_bias", kind="route", tokens=16383, experts=512, top_k=10, score="softmax", bias=True,
             groups=1, top_groups=1, group_score=1, scale=1.0, dtype="f32"),
        # A decode batch's tokens by their request's adapter, some without one.
        dict(name="group_64_tokens", kind="group", rows=64, buckets=16, outside=0.1),
        # The pairs of 8,192 tokens with ten picks each, by expert.
        dict(name="group_81920_pairs", kind="group", rows=81920, buckets=512, outside=0.0),
        # One request generating through its adapter, fp32 activations as the layer's.
        dict(name="project_1", kind="project", tokens=1, rows=4096, cols=2048, group=64, meta="bf16", x="f32",
             adapters=8, rank=16, adapter="bf16", ragged=False, order="mixed"),
        # A ragged batch of requests, an adapter of its own rank for nearly each.
        dict(name="project_37_ragged", kind="project", tokens=37, rows=2048, cols=4096, group=64, meta="f32", x="f32",
             adapters=32, rank=24, adapter="f16", ragged=True, order="mixed"),
        # A full decode batch in bf16, 64 adapters of rank 16, over a wide output of odd size.
        dict(name="project_64_wide", kind="project", tokens=64, rows=12289, cols=2048, group=64, meta="bf16", x="bf16",
             adapters=64, rank=16, adapter="bf16", ragged=False, order="mixed"),
        # A prompt chunk in fp32 of a few requests, one after another.
        dict(name="project_500_f32", kind="project", tokens=500, rows=2048, cols=2048, group=32, meta="f32", x="f32",
             adapters=4, rank=8, adapter="f32", ragged=False, order="runs"),
        # The benchmark's prompt chunk in bf16.
        dict(name="project_512", kind="project", tokens=512, rows=4096, cols=2048, group=64, meta="bf16", x="bf16",
             adapters=4, rank=16, adapter="bf16", ragged=False, order="runs"),
        # Several long prompts with wide adapters, the largest call.
        dict(name="project_4096", kind="project", tokens=4096, rows=8192, cols=4096, group=64, meta="bf16", x="bf16",
             adapters=8, rank=64, adapter="bf16", ragged=False, order="mixed"),
    ]


LARGEST = 4096 * 8192 * 4096  # products of the largest listed projection


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["route", "route", "group", "project", "project", "project"])
    if kind == "route":
        experts = rng.choice([8, 60, 64, 128, 160, 256, 384, 512])
        groups = rng.choice([1, 1, 4, 8]) if experts % 8 == 0 and experts >= 64 else 1
        per = experts // groups
        top_groups = rng.randint(1, groups)
        return {"kind": kind, "tokens": log(1, 16383), "experts": experts,
                "top_k": rng.randint(1, min(12, top_groups * per)), "score": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.6, "groups": groups, "top_groups": top_groups,
                "group_score": rng.choice([1, 2]) if groups > 1 else 1, "scale": rng.choice([1.0, 2.5]),
                "dtype": rng.choice(["f32", "f32", "bf16", "f16"])}
    if kind == "group":
        return {"kind": kind, "rows": log(1, 81920), "buckets": log(1, 1024), "outside": rng.choice([0.0, 0.1, 0.5])}
    c = {"kind": kind, "cols": 128 * log(4, 40), "rows": log(512, 16384), "group": rng.choice([32, 64, 64, 128]),
         "meta": rng.choice(["f32", "f16", "bf16"]), "x": rng.choice(["f32", "f16", "bf16"]), "adapters": log(1, 64),
         "rank": rng.choice([4, 8, 16, 16, 21, 32, 64]), "adapter": rng.choice(["f32", "f16", "bf16", "bf16"]),
         "ragged": rng.random() < 0.3, "order": rng.choice(["mixed", "runs"])}
    c["tokens"] = min(log(1, 4096), LARGEST // (c["rows"] * c["cols"]))
    if c["tokens"] > 256:  # the plain form multiplies by every adapter's matrices
        c["adapters"] = min(c["adapters"], 16)
    return c


def work(case):
    c = case
    if c["kind"] == "route":
        T, E = c["tokens"], c["experts"]
        return {"bytes": T * E * BYTES[c["dtype"]] + (4 * E if c["bias"] else 0) + 8 * T * c["top_k"], "flops": 4.0 * T * E}
    if c["kind"] == "group":
        return {"bytes": 8 * c["rows"] + 4 * (c["buckets"] + 1), "flops": 2.0 * c["rows"]}
    T, N, K = c["tokens"], c["rows"], c["cols"]
    weights = N * K // 2 + 2 * (N * K // c["group"]) * BYTES[c["meta"]]
    # The adapters that T tokens reach, expected over uniform ones.
    reached = c["adapters"] * (1.0 - (1.0 - 1.0 / c["adapters"]) ** T) if c["order"] == "mixed" else min(T, c["adapters"])
    rank = c["rank"] * (0.5 if c["ragged"] else 1.0)
    return {"bytes": weights + reached * rank * (N + K) * BYTES[c["adapter"]] + T * (N + K) * BYTES[c["x"]],
            "flops": 2.0 * T * N * K + 2.0 * T * rank * (N + K)}


# ---- inputs ---------------------------------------------------------------------------
def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def route_inputs(c, seed):
    g = generator(seed * 131 + 1)
    logits = (2.0 * torch.randn(c["tokens"], c["experts"], device="cuda", generator=g)).to(FLOATS[c["dtype"]])
    bias = 0.1 * torch.randn(c["experts"], device="cuda", generator=g) if c["bias"] else None
    return logits, bias


def group_inputs(c, seed):
    g = generator(seed * 131 + 2)
    keys = torch.randint(0, c["buckets"], (c["rows"],), device="cuda", generator=g, dtype=torch.int32)
    none = torch.rand(c["rows"], device="cuda", generator=g) < c["outside"]
    return torch.where(none, -1, keys)


def project_inputs(c, seed):
    g = generator(seed * 131 + 3)
    T, N, K, n, r = c["tokens"], c["rows"], c["cols"], c["adapters"], c["rank"]
    words = torch.randint(-(2**31), 2**31, (N, K // 8), device="cuda", generator=g, dtype=torch.int64).to(torch.int32)
    scales = torch.randn(N, K // c["group"], device="cuda", generator=g).abs() * 0.02
    biases = -8.0 * scales + 0.002 * torch.randn(N, K // c["group"], device="cuda", generator=g)
    x = torch.randn(T, K, device="cuda", generator=g).to(FLOATS[c["x"]])
    a = (torch.randn(n, r, K, device="cuda", generator=g) / math.sqrt(K)).to(FLOATS[c["adapter"]])
    b = (0.5 * torch.randn(n, N, r, device="cuda", generator=g)).to(FLOATS[c["adapter"]])
    factors = 0.5 + 1.5 * torch.rand(n, device="cuda", generator=g)
    # A request without an adapter now and then; requests one after another, or interleaved.
    ids = torch.randint(-1 if n > 2 else 0, n, (T,), device="cuda", generator=g, dtype=torch.int32)
    if c["order"] == "runs":
        ids = ids.sort().values
    ranks = torch.randint(1, r + 1, (n,), device="cuda", generator=g, dtype=torch.int32) if c["ragged"] else None
    meta = FLOATS[c["meta"]]
    return words, scales.to(meta), biases.to(meta), x, a, b, factors, ids, ranks


_framework = None


def framework():
    """The program's binding and its one context, kept for its life."""
    global _framework
    if _framework is None:
        sys.path.insert(0, os.path.join(ROOT, "orbi-streammoe_amd"))
        import osm_hip

        _framework = osm_hip, osm_hip.Context(0)
    return _framework


def prepare(case, seed):
    c = dict(case)
    if c["kind"] == "route":
        logits, bias = route_inputs(c, seed)
        s = {"case": c, "logits": logits, "bias": bias,
             "ids": torch.empty(c["tokens"], c["top_k"], dtype=torch.int32, device="cuda"),
             "weights": torch.empty(c["tokens"], c["top_k"], dtype=torch.float32, device="cuda")}
        if own:
            osm_hip, _ = framework()
            s["rule"] = osm_hip.RouteRule(c["experts"], c["top_k"], getattr(osm_hip, "SCORE_" + c["score"].upper()),
                                          groups=c["groups"], top_groups=c["top_groups"], group_score=c["group_score"],
                                          renormalize=True, scale=c["scale"])
        return s
    if c["kind"] == "group":
        return {"case": c, "keys": group_inputs(c, seed),
                "offsets": torch.empty(c["buckets"] + 1, dtype=torch.int32, device="cuda"),
                "order": torch.empty(c["rows"], dtype=torch.int32, device="cuda")}
    words, scales, biases, x, a, b, factors, ids, ranks = project_inputs(c, seed)
    s = {"case": c, "words": words, "scales": scales, "biases": biases, "x": x, "a": a, "b": b, "factors": factors,
         "ids": ids, "ranks": ranks, "y": torch.empty(c["tokens"], c["rows"], dtype=x.dtype, device="cuda")}
    if own:
        osm_hip, ctx = framework()
        code = {"f32": osm_hip.F32, "f16": osm_hip.F16, "bf16": osm_hip.BF16}
        s["projection"] = osm_hip.Q4ProjectionWeights.on_device(ctx, words.data_ptr(), c["rows"], c["cols"] // 8,
                                                               scales.data_ptr(), biases.data_ptr(), c["group"], code[c["meta"]])
        s["adapters"] = osm_hip.Adapters(a.data_ptr(), b.data_ptr(), c["adapters"], c["rank"], code[c["adapter"]],
                                         scales=factors.data_ptr(), ranks=ranks.data_ptr() if ranks is not None else None)
        s["dtype"] = code[c["x"]]
    return s


# ---- one pass -------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"route": own_route, "group": own_group, "project": own_project}[kind](state)
    return {"route": plain_route, "group": plain_group, "project": plain_project}[kind](state)


def own_route(s):
    osm_hip, ctx = framework()
    c, bias = s["case"], s["bias"]
    osm_hip.route_experts(ctx, s["rule"], s["logits"].data_ptr(), getattr(osm_hip, c["dtype"].upper()), c["tokens"],
                          s["ids"].data_ptr(), s["weights"].data_ptr(), bias_ptr=bias.data_ptr() if bias is not None else None)
    return {"ids": s["ids"], "weights": s["weights"]}


def own_group(s):
    osm_hip, ctx = framework()
    osm_hip.group_rows(ctx, s["keys"].data_ptr(), s["case"]["rows"], s["case"]["buckets"], s["offsets"].data_ptr(),
                       s["order"].data_ptr())
    return {"offsets": s["offsets"], "order": s["order"]}


def own_project(s):
    osm_hip, ctx = framework()
    osm_hip.q4_project(ctx, s["projection"], s["x"].data_ptr(), s["y"].data_ptr(), s["case"]["tokens"], x_dtype=s["dtype"],
                       y_dtype=s["dtype"], adapters=s["adapters"], adapter_ids_ptr=s["ids"].data_ptr())
    return s["y"]


def plain_route(s):
    c = s["case"]
    l = s["logits"].double()  # scores next to one another decide the picks
    if c["score"] == "softmax":
        p = torch.exp(l - l.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-l))
    choice = p if s["bias"] is None else p + s["bias"].double()
    if c["groups"] > 1:
        g = choice.view(c["tokens"], c["groups"], -1)
        best = g.sort(dim=-1, descending=True).values[..., :c["group_score"]].sum(-1)
        kept = best.sort(dim=-1, descending=True, stable=True).indices[:, :c["top_groups"]]
        keep = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        choice = torch.where(keep[..., None], g, -math.inf).view_as(choice)
    ids = choice.sort(dim=-1, descending=True, stable=True).indices[:, :c["top_k"]]
    w = p.gather(1, ids)
    w = c["scale"] * w / w.sum(-1, keepdim=True)
    return {"ids": ids.to(torch.int32), "weights": w.to(torch.float32)}


def plain_group(s):
    buckets = s["case"]["buckets"]
    key = torch.where(s["keys"] < 0, buckets, s["keys"]).long()
    counts = torch.bincount(key, minlength=buckets + 1)
    offsets = torch.cumsum(counts, 0) - counts
    return {"offsets": offsets.to(torch.int32), "order": key.sort(dim=0, stable=True).indices.to(torch.int32)}


def plain_project(s):
    c, x = s["case"], s["x"].float()
    n, r = c["adapters"], c["rank"]
    shifts = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    q = ((s["words"][..., None] >> shifts) & 15).view(c["rows"], -1, c["group"]).float()
    w = (q * s["scales"].float()[..., None] + s["biases"].float()[..., None]).view(c["rows"], c["cols"])
    y = x @ w.t()
    # Every adapter's first product, kept where the adapter is the token's own (and the rank the adapter's).
    v = x @ s["a"].float().view(n * r, c["cols"]).t() * s["factors"].repeat_interleave(r)
    column = torch.arange(n * r, device="cuda")
    mine = column // r == s["ids"][:, None]
    if s["ranks"] is not None:
        mine &= column % r < s["ranks"].repeat_interleave(r)
    y += torch.where(mine, v, 0.0) @ s["b"].float().permute(0, 2, 1).reshape(n * r, c["rows"])
    return y.to(s["x"].dtype)


# ---- the same in 64 bits ----------------------------------------------------------------
def exact(case, seed):
    c = case
    if c["kind"] == "group":
        return None
    if c["kind"] == "route":
        logits, bias = route_inputs(c, seed)
        l = logits.double()
        score = torch.softmax(l, -1) if c["score"] == "softmax" else torch.sigmoid(l)
        left = score if bias is None else score + bias
        if c["groups"] > 1:
            rest = left.reshape(c["tokens"], c["groups"], -1).clone()
            total = 0.0
            for _ in range(c["group_score"]):
                top = rest.max(-1, keepdim=True)
                total = total + top.values[..., 0]
                rest.scatter_(-1, top.indices, -math.inf)
            # The groups above a group, and the equal ones before it, are counted.
            before = torch.ones(c["groups"], c["groups"], device="cuda").tril(-1).bool()
            above = (total[:, None, :] > total[:, :, None]) | ((total[:, None, :] == total[:, :, None]) & before)
            left = left.reshape(c["tokens"], c["groups"], -1).masked_fill((above.sum(-1) >= c["top_groups"])[..., None], -math.inf)
            left = left.reshape(c["tokens"], -1)
        left, picked = left.clone(), []
        for _ in range(c["top_k"]):
            top = left.amax(-1, keepdim=True)
            first = (left == top).to(torch.uint8).argmax(-1, keepdim=True)
            picked.append(score.gather(1, first))
            left.scatter_(1, first, -math.inf)
        w = torch.cat(picked, 1)
        return {"ids": None, "weights": c["scale"] * w / w.sum(-1, keepdim=True)}
    words, scales, biases, x, a, b, factors, ids, ranks = project_inputs(c, seed)
    q = torch.stack([(words.long() >> (4 * j)) & 15 for j in range(8)], -1).reshape(c["rows"], c["cols"]).double()
    w = q * scales.double().repeat_interleave(c["group"], 1) + biases.double().repeat_interleave(c["group"], 1)
    x = x.double()
    y = x @ w.t()
    for i in range(c["adapters"]):
        t = (ids == i).nonzero()[:, 0]
        k = c["rank"] if ranks is None else int(ranks[i])
        y[t] += float(factors[i]) * (x[t] @ a[i, :k].double().t()) @ b[i, :, :k].double().t()
    return y
