"""Performance cases of what a decoder layer calls beside its quantised products, from one decode token to a large prefill.

* lora:   low-rank adapters of many requests added to a shared projection's output (`lora_add`);
* router: the router's product, 16-bit hidden states and weights to float32 logits (`router_logits`);
* route:  experts and weights from the logits: scores, bias, groups, top-k (`route_topk`).
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
WEIGHT_STD = 0.02


def listed():
    return [
        # one decoded token of one adapter beside a narrow projection: launches and latency
        {"name": "lora_1", "kind": "lora", "t": 1, "seqs": 1, "k": 7168, "slices": "2112", "rank": 16, "mixed": False, "adapters": 4,
         "dtype": "bf16"},
        # a decode batch whose requests name sixteen adapters of two ranks, beside the widest merged layer
        {"name": "lora_64_gate_up", "kind": "lora", "t": 64, "seqs": 64, "k": 7168, "slices": "18432 18432", "rank": 32, "mixed": True,
         "adapters": 16, "dtype": "bf16"},
        # a ragged chunk of five requests beside query, key and value projections, float16
        {"name": "lora_257_qkv", "kind": "lora", "t": 257, "seqs": 5, "k": 8192, "slices": "8192 1024 1024", "rank": 64, "mixed": False,
         "adapters": 3, "dtype": "fp16"},
        # a prefill of a few requests beside the widest merged layer: the largest
        {"name": "lora_4096_gate_up", "kind": "lora", "t": 4096, "seqs": 4, "k": 7168, "slices": "18432 18432", "rank": 64, "mixed": False,
         "adapters": 8, "dtype": "bf16"},
        # one decoded token's router: latency
        {"name": "router_1", "kind": "router", "t": 1, "e": 256, "k": 7168, "dtype": "bf16"},
        # a decode batch, a smaller layer, float16
        {"name": "router_64_small", "kind": "router", "t": 64, "e": 128, "k": 2048, "dtype": "fp16"},
        # a ragged chunk of tokens
        {"name": "router_511", "kind": "router", "t": 511, "e": 160, "k": 5120, "dtype": "bf16"},
        # a long prefill
        {"name": "router_8192", "kind": "router", "t": 8192, "e": 256, "k": 7168, "dtype": "bf16"},
        # one decoded token, groups by their best two biased scores: latency
        {"name": "route_1", "kind": "route", "t": 1, "e": 256, "topk": 8, "groups": 8, "kept": 4, "top": 2, "scoring": "sigmoid", "bias": True,
         "renorm": True, "factor": 2.5, "masked": 0.0, "dtype": "fp32"},
        # a ragged chunk, groups by their best probability, weights as they are
        {"name": "route_1999_max", "kind": "route", "t": 1999, "e": 160, "topk": 6, "groups": 8, "kept": 3, "top": 1, "scoring": "softmax",
         "bias": False, "renorm": False, "factor": 16.0, "masked": 0.0, "dtype": "bf16"},
        # a long prefill without groups, a few experts out of service
        {"name": "route_8192_masked", "kind": "route", "t": 8192, "e": 128, "topk": 8, "groups": 1, "kept": 1, "top": 1, "scoring": "softmax",
         "bias": True, "renorm": True, "factor": 1.0, "masked": 0.05, "dtype": "bf16"},
        # the longest prefill, grouped and biased
        {"name": "route_16384", "kind": "route", "t": 16384, "e": 256, "topk": 8, "groups": 8, "kept": 4, "top": 2, "scoring": "sigmoid",
         "bias": True, "renorm": True, "factor": 2.5, "masked": 0.0, "dtype": "fp32"},
    ]


def _log_int(rng, lo, hi, step=1):
    """An integer in [lo, hi], spread over the logarithm, rounded to a multiple of `step`."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // step * step, max((lo + step - 1) // step * step, int(round(v / step)) * step))


def _draw_once(rng):
    kind = rng.choices(["lora", "router", "route"], [4, 3, 3])[0]
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "lora":
        t = _log_int(rng, 1, 8192)
        n = rng.choice([1, 1, 2, 3])
        return {"kind": kind, "t": t, "seqs": t if t <= 256 and rng.random() < 0.6 else _log_int(rng, 1, min(t, 64)),
                "k": _log_int(rng, 256, 18432, rng.choice([8, 64, 128])),
                "slices": " ".join(str(_log_int(rng, 64, 18432, rng.choice([1, 8, 64]))) for _ in range(n)),
                "rank": rng.choice([8, 16, 16, 32, 64, 128]), "mixed": rng.random() < 0.4, "adapters": _log_int(rng, 1, 32), "dtype": dtype}
    if kind == "router":
        return {"kind": kind, "t": _log_int(rng, 1, 16384), "e": _log_int(rng, 8, 512, rng.choice([1, 8, 32])),
                "k": _log_int(rng, 256, 8192, rng.choice([8, 64, 128])), "dtype": dtype}
    groups = rng.choice([1, 1, 2, 4, 8, 16])
    e = groups * _log_int(rng, max(2, 8 // groups), 512 // groups)
    kept = rng.randint(1, groups)
    bias = rng.random() < 0.5
    return {"kind": kind, "t": _log_int(rng, 1, 32768), "e": e, "topk": rng.randint(1, min(10, kept * e // groups)), "groups": groups,
            "kept": kept, "top": 2 if groups > 1 and bias else 1, "scoring": rng.choice(["softmax", "sigmoid"]), "bias": bias,
            "renorm": rng.random() < 0.7, "factor": rng.choice([1.0, 2.5, 16.0]), "masked": rng.choice([0.0, 0.0, 0.05]),
            "dtype": rng.choice(["bf16", "fp16", "fp32"])}


def _slices(case):
    """How many columns of the output each merged projection has."""
    return [int(n) for n in case["slices"].split()]


def _cost(case):
    """What a case costs, and what the plain form of a `lora` case multiplies (every token with every adapter)."""
    w, plain = work(case), 0
    if case["kind"] == "lora":
        plain = 2 * case["t"] * case["adapters"] * case["rank"] * (len(_slices(case)) * case["k"] + sum(_slices(case)))
    return {**w, "plain": plain}


def draw(rng):
    most = {}
    for c in listed():
        most = {k: max(most.get(k, 0), v) for k, v in _cost(c).items()}
    while True:
        case = _draw_once(rng)
        if all(v <= most[k] for k, v in _cost(case).items()):
            return case


# ---- inputs -----------------------------------------------------------------------------------------------------------


def _activations(gen, m, k, dtype, outliers=0.001):
    """N(0, 1) rows, a value in a thousand ten times as large."""
    x = torch.randn(m, k, generator=gen, device=DEV, dtype=torch.float32)
    x = torch.where(torch.rand(m, k, generator=gen, device=DEV) < outliers, x * 10, x)
    return x.to(DTYPES[dtype])


def _ranks(case):
    """The adapters' ranks: every other one's is half the largest where they are mixed."""
    return [case["rank"] // 2 if case["mixed"] and l % 2 else case["rank"] for l in range(case["adapters"])]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, t, dtype = case["kind"], case["t"], DTYPES[case["dtype"]]
    if kind == "router":
        w = torch.randn(case["e"], case["k"], generator=gen, device=DEV) * WEIGHT_STD
        return {"kind": kind, "x": _activations(gen, t, case["k"], case["dtype"]), "w": w.to(dtype)}
    if kind == "route":
        logits = torch.randn(t, case["e"], generator=gen, device=DEV) * 1.5
        if case["masked"]:  # experts out of service, the same for every token
            off = torch.rand(case["e"], generator=gen, device=DEV) < case["masked"]
            logits = logits.masked_fill(off, -math.inf)
        scale = 0.1 if case["scoring"] == "sigmoid" else 0.2 / case["e"]
        bias = torch.randn(case["e"], generator=gen, device=DEV) * scale if case["bias"] else None
        return {"kind": kind, "x": logits.to(dtype), "bias": bias, **{k: case[k] for k in ("topk", "groups", "kept", "top", "scoring", "renorm",
                                                                                      "factor")}}
    k, n, rank, adapters, slices = case["k"], sum(_slices(case)), case["rank"], case["adapters"], len(_slices(case))
    # requests of uneven lengths one after the other, each with an adapter of its own choice or with none
    cuts = torch.randperm(t - 1, generator=gen, device=DEV)[: case["seqs"] - 1] + 1 if t > 1 else torch.zeros(0, device=DEV, dtype=torch.int64)
    seq = torch.zeros(t, dtype=torch.int64, device=DEV)
    seq[cuts] = 1
    ids = torch.randint(-1, adapters, (case["seqs"],), generator=gen, device=DEV, dtype=torch.int32)
    if case["seqs"] <= 4:  # (a few requests: all of them have one)
        ids = ids.clamp(min=0)
    a = torch.randn(adapters, slices * rank, k, generator=gen, device=DEV) * (1.0 / math.sqrt(k))
    b = torch.randn(adapters, n, rank, generator=gen, device=DEV) * WEIGHT_STD
    return {"kind": kind, "x": _activations(gen, t, k, case["dtype"]), "base": torch.randn(t, n, generator=gen, device=DEV).to(dtype),
            "a": a.to(dtype), "b": b.to(dtype), "ids": ids[seq.cumsum(0)], "slices": tuple(_slices(case)),
            "ranks": torch.tensor(_ranks(case), dtype=torch.int32, device=DEV),
            "scalings": torch.rand(adapters, generator=gen, device=DEV) + 0.5}


# ---- one pass ---------------------------------------------------------------------------------------------------------


def _plain_lora(st):
    x, a, b, slices = st["x"], st["a"], st["b"], st["slices"]
    adapters, n, rank = b.shape
    in_rank = torch.arange(rank, device=DEV) < st["ranks"][:, None]  # [adapters, rank]
    rows = torch.where(in_rank[:, None, :, None], a.float().view(adapters, len(slices), rank, -1), 0.0)
    h = (x.float() @ rows.flatten(0, 2).t()).view(-1, adapters, len(slices), rank)
    mine = st["ids"][:, None] == torch.arange(adapters, device=DEV)
    h = torch.where(mine[:, :, None, None], h * st["scalings"][None, :, None, None], 0.0)
    cols = torch.where(in_rank[:, None, :], b.float(), 0.0).transpose(0, 1)  # [n, adapters, rank]
    out, at = st["base"].float(), 0
    for s, width in enumerate(slices):
        out[:, at : at + width] += h[:, :, s].flatten(1) @ cols[at : at + width].flatten(1).t()
        at += width
    return out.to(x.dtype)


def _plain_route(st):
    # in 64 bits: in 32 two scores may change their order
    x = st["x"].double()
    t, e = x.shape
    x = torch.where(torch.isnan(x), -math.inf, x).clamp(max=torch.finfo(torch.float32).max)
    live = x > -math.inf
    if st["scoring"] == "softmax":
        low = x
        top = x.amax(-1, keepdim=True)
        p = torch.where(live, torch.exp(x - torch.where(top > -math.inf, top, 0.0)), 0.0)
        s = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    else:
        low = torch.where(live, x.clamp(max=0.0) - torch.log1p(torch.exp(-x.abs())), -math.inf)  # log of the score
        s = torch.where(live, 1.0 / (1.0 + torch.exp(-x)), 0.0)
    c = s if st["bias"] is None else s + st["bias"].double()
    c = torch.where(live, c, -math.inf)
    # (a score grows with its logit: without a bias the logits decide the order)
    key = x if st["bias"] is None else c
    if st["groups"] > 1:
        of = (x if st["bias"] is None and st["top"] == 1 else c).view(t, st["groups"], -1)
        best = torch.sort(of, dim=-1, descending=True)[0][..., : st["top"]]
        value = torch.where(best > -math.inf, best, 0.0).sum(-1)
        value = torch.where(best[..., 0] > -math.inf, value, -math.inf)
        order = torch.sort(value, dim=-1, descending=True, stable=True)[1][:, : st["kept"]]
        keep = torch.zeros(t, st["groups"], dtype=torch.bool, device=DEV).scatter_(1, order, True)
        key = torch.where(keep[:, :, None], key.view(t, st["groups"], -1), -math.inf).view(t, e)
    value, ids = torch.sort(key, dim=-1, descending=True, stable=True)
    value, ids = value[:, : st["topk"]], ids[:, : st["topk"]]
    there = value > -math.inf
    if st["renorm"]:
        w = torch.where(there, low.gather(1, ids), -math.inf)
        w = torch.exp(w - torch.where(there[:, :1], w.amax(-1, keepdim=True), 0.0))
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
    else:
        w = torch.where(there, s.gather(1, ids), 0.0)
    return (w * st["factor"]).float(), torch.where(there, ids, -1).to(torch.int32)


def run(state):
    kind = state["kind"]
    if not own:
        if kind == "lora":
            return _plain_lora(state)
        return _plain_route(state) if kind == "route" else state["x"].float() @ state["w"].float().t()
    from sglang_b200 import ops

    if kind == "lora":
        return ops.lora_add(state["base"], state["x"], state["a"], state["b"], state["ids"], state["scalings"], ranks=state["ranks"],
                            slices=state["slices"])
    if kind == "router":
        return ops.router_logits(state["x"], state["w"])
    return ops.route_topk(state["x"], state["topk"], scoring_func=state["scoring"], correction_bias=state["bias"],
                          num_expert_group=state["groups"], topk_group=state["kept"], group_top=state["top"], renormalize=state["renorm"],
                          routed_scaling_factor=state["factor"])


def work(case):
    kind, t = case["kind"], case["t"]
    if kind == "route":
        return {"bytes": t * case["e"] * DTYPES[case["dtype"]].itemsize + 8 * t * case["topk"], "flops": 8 * t * case["e"]}
    if kind == "router":
        return {"bytes": 2 * case["k"] * (t + case["e"]) + 4 * t * case["e"], "flops": 2 * t * case["e"] * case["k"]}
    # adapters that are expected to be named at all, when every request names any of them or none
    n, slices, adapters = sum(_slices(case)), len(_slices(case)), case["adapters"]
    few = case["seqs"] <= 4
    live = adapters * (1.0 - (1.0 - 1.0 / (adapters + (not few))) ** case["seqs"])
    rank = sum(_ranks(case)) / adapters
    share = 1.0 if few else adapters / (adapters + 1)
    return {"bytes": 2 * (t * case["k"] + 2 * t * n + live * rank * (slices * case["k"] + n)),
            "flops": 2 * t * share * rank * (slices * case["k"] + n)}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------


def _exact_lora(st):
    out = st["base"].double()
    rank_max = st["b"].shape[2]
    for l, rank in enumerate(st["ranks"].tolist()):
        rows = (st["ids"] == l).nonzero()[:, 0]
        if not len(rows):
            continue
        x, lo = st["x"][rows].double(), 0
        for s, width in enumerate(st["slices"]):
            a = st["a"][l, s * rank_max : s * rank_max + rank].double()
            b = st["b"][l, lo : lo + width, :rank].double()
            out[rows, lo : lo + width] += (x @ a.t()) @ b.t() * float(st["scalings"][l])
            lo += width
    return out


def _exact_route(st):
    """The weights of the experts that the order names; the order is taken pick by pick."""
    x = st["x"].double()
    t, e = x.shape
    x = torch.where(x.isnan(), -math.inf, x).clamp(max=torch.finfo(torch.float32).max)
    off = x == -math.inf
    if st["scoring"] == "softmax":
        logs = x - torch.logsumexp(x, -1, keepdim=True)
    else:
        logs = torch.nn.functional.logsigmoid(x)
    s = torch.exp(logs).masked_fill(off, 0.0)
    b = torch.zeros(e, device=DEV, dtype=torch.float64) if st["bias"] is None else st["bias"].double()
    c = (s + b).masked_fill(off, -math.inf)
    if st["bias"] is None:
        c = x.clone()
    gs = e // st["groups"]
    if st["groups"] > 1:
        left = (c if st["top"] == 1 else (s + b).masked_fill(off, -math.inf)).clone().view(t, st["groups"], gs)
        value = torch.zeros(t, st["groups"], device=DEV, dtype=torch.float64)
        for i in range(st["top"]):
            best, at = left.max(-1)
            value += best if i == 0 else best.clamp(min=-1e300).masked_fill(best == -math.inf, 0.0)
            left.scatter_(2, at[..., None], -math.inf)
        # a group stays when fewer than `kept` are better, or as good and before it
        better = (value[:, None, :] > value[:, :, None]).sum(-1)
        index = torch.arange(st["groups"], device=DEV)
        better += ((value[:, None, :] == value[:, :, None]) & (index[None, None, :] < index[None, :, None])).sum(-1)
        c = c.masked_fill((better >= st["kept"]).repeat_interleave(gs, 1), -math.inf)
    ids, index = [], torch.arange(e, device=DEV)
    for _ in range(st["topk"]):
        best = c.amax(-1, keepdim=True)
        at = torch.where(c == best, index, e).amin(-1)
        ids.append(torch.where(best[:, 0] > -math.inf, at, -1))
        c = c.scatter(1, at[:, None], -math.inf)
    ids = torch.stack(ids, -1)
    picked = torch.where(ids >= 0, logs.gather(1, ids.clamp(min=0)), -math.inf)
    w = torch.exp(picked)
    if st["renorm"]:
        w = torch.exp(picked - torch.logsumexp(picked, -1, keepdim=True)).masked_fill(ids < 0, 0.0)
    return w * st["factor"], ids.to(torch.int32)


def exact(case, seed):
    st = prepare(case, seed)
    if st["kind"] == "lora":
        return _exact_lora(st)
    if st["kind"] == "route":
        return _exact_route(st)
    w = st["w"].double().t().contiguous()
    return torch.cat([part.double() @ w for part in st["x"].split(1024)])
