"""Performance cases of the 4-bit floating-point operators, from one decode token to a large prefill.

Values are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a byte, the even column in the low half.  They share
a scale per group of a row's columns: 16 columns an e4m3 scale, beside one float32 scale of the whole tensor, or 32 columns a
power of two (e8m0).

* quant: rows are quantised and read back (`per_token_group_quant_fp4`, `per_token_group_dequant_fp4`);
* silu:  silu(gate) * up of a gated MLP's rows, quantised in the same pass, and read back (`silu_and_mul_quant_fp4`);
* mm:    the product of quantised activations with a quantised weight (`w4a4_group_fp4_matmul`);
* moe:   the routed experts of a few tokens on 4-bit weights and 16-bit activations (`fused_experts_fp4`).
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
        # one decoded token's hidden state: launches and latency
        {"name": "quant_1", "kind": "quant", "m": 1, "k": 7168, "group": 16, "dtype": "bf16"},
        # a ragged chunk of tokens with power-of-two scales
        {"name": "quant_1999_mx", "kind": "quant", "m": 1999, "k": 8192, "group": 32, "dtype": "fp16"},
        # a long prefill at a dense layer's intermediate width
        {"name": "quant_8192", "kind": "quant", "m": 8192, "k": 18432, "group": 16, "dtype": "bf16"},
        # a decode batch between the two products of an MLP
        {"name": "silu_64", "kind": "silu", "m": 64, "k": 2048, "group": 16, "dtype": "bf16"},
        # a prefill between the two products of a wide MLP
        {"name": "silu_4096", "kind": "silu", "m": 4096, "k": 18432, "group": 16, "dtype": "bf16"},
        # one decoded token through a narrow projection: latency
        {"name": "mm_1", "kind": "mm", "m": 1, "n": 2112, "k": 7168, "group": 16, "dtype": "bf16", "bias": False},
        # a decode batch through a wide layer: weight streaming
        {"name": "mm_64_gate_up", "kind": "mm", "m": 64, "n": 36864, "k": 7168, "group": 16, "dtype": "bf16", "bias": False},
        # a ragged chunk of tokens, power-of-two scales, a bias, float16
        {"name": "mm_257_qkv_mx", "kind": "mm", "m": 257, "n": 10240, "k": 8192, "group": 32, "dtype": "fp16", "bias": True},
        # a prefill through the widest layer: the largest product
        {"name": "mm_4096_gate_up", "kind": "mm", "m": 4096, "n": 36864, "k": 7168, "group": 16, "dtype": "bf16", "bias": False},
        # one decoded token through one GPU's eighth of every expert: latency
        {"name": "moe_1_shard", "kind": "moe", "m": 1, "e": 256, "topk": 8, "h": 7168, "i": 256, "dtype": "bf16"},
        # a decode batch through many small experts
        {"name": "moe_32_small", "kind": "moe", "m": 32, "e": 128, "topk": 8, "h": 2048, "i": 768, "dtype": "bf16"},
        # a few tokens through whole large experts: most of the weights they touch are read for one token each
        {"name": "moe_16_large", "kind": "moe", "m": 16, "e": 256, "topk": 8, "h": 7168, "i": 2048, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi, step=1):
    """An integer in [lo, hi], spread over the logarithm, rounded to a multiple of `step`."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // step * step, max((lo + step - 1) // step * step, int(round(v / step)) * step))


def _draw_once(rng):
    kind = rng.choices(["quant", "silu", "mm", "moe"], [2, 2, 4, 3])[0]
    group = rng.choice([16, 16, 32])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "quant":
        return {"kind": kind, "m": _log_int(rng, 1, 16384), "k": _log_int(rng, 64, 18432, group), "group": group,
                "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if kind == "silu":
        return {"kind": kind, "m": _log_int(rng, 1, 16384), "k": _log_int(rng, 64, 18432, group), "group": group, "dtype": dtype}
    if kind == "mm":
        return {"kind": kind, "m": _log_int(rng, 1, 8192), "n": _log_int(rng, 256, 36864, rng.choice([8, 64, 128])),
                "k": _log_int(rng, 256, 18432, 32), "group": group, "dtype": dtype, "bias": rng.random() < 0.25}
    e = rng.choice([8, 16, 32, 64, 128, 256])
    return {"kind": kind, "m": _log_int(rng, 1, 64), "e": e, "topk": rng.randint(1, min(8, e // 2)),
            "h": _log_int(rng, 512, 7168, 32), "i": _log_int(rng, 128, 2048, 32), "dtype": dtype}


def _slots(case):
    """How many weight values the plain form of a `moe` case lays out."""
    return case["m"] * case["topk"] * case["h"] * case["i"] if case["kind"] == "moe" else 0


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        most = {k: max(most.get(k, 0), v) for k, v in {**w, "slots": _slots(c)}.items()}
    while True:
        case = _draw_once(rng)
        if all(v <= most[k] for k, v in {**work(case), "slots": _slots(case)}.items()):
            return case


# ---- the format, in elementary operations -----------------------------------------------------------------------------

VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _e2m1(q):
    """`q` to the nearest e2m1 value, ties to the even mantissa, saturating."""
    a = q.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign(torch.clamp(torch.round(a / step) * step, max=6.0), q)


def _e4m3(s):
    """`s` >= 0 to the nearest e4m3 value, ties to the even mantissa, saturating."""
    step = torch.ldexp(torch.ones_like(s), torch.clamp(torch.frexp(s)[1] - 4, min=-9))
    return torch.clamp(torch.round(s / step) * step, max=448.0)


def _quantize(x, global_scale, group):
    """x [m, k] -> (values [m, k / group, group], scales [m, k / group, 1]), both float64: a value or a scale next to a border
    falls to the wrong side of it in 32 bits."""
    groups = x.double().unflatten(-1, (-1, group)) * global_scale.double()
    amax = groups.abs().amax(-1, keepdim=True)
    if group == 32:
        e = torch.where(amax == 0, -127, torch.frexp(amax)[1] - 3).clamp(-127, 127)
        s = torch.ldexp(torch.ones_like(amax), e)
    else:
        s = _e4m3(amax / 6.0)
    return torch.where(s > 0, _e2m1(groups / s), 0.0), s


def _round_trip(x, global_scale, group):
    v, s = _quantize(x, global_scale, group)
    return (v * s / global_scale.double()).flatten(-2)


def _pack(v):
    """e2m1 values [.., k] -> two codes to a byte [.., k / 2], the even column in the low half."""
    a = v.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code += torch.signbit(v).to(torch.uint8) * 8
    return code[..., 0::2] + code[..., 1::2] * 16


def _scale_bytes(s, group):
    """Scales as the format holds them, one byte each."""
    if group == 32:
        return (torch.frexp(s)[1] + 126).to(torch.uint8).view(torch.float8_e8m0fnu)
    return s.to(torch.float8_e4m3fn)


def _blocked(s):
    """Scales [m, g] in the order of the products' operands: blocks of 128 rows x 4 groups, a block's rows r, r + 32, r + 64
    and r + 96 side by side, the tensor padded with zeros to whole blocks."""
    m, g = s.shape
    mb, gb = -(-m // 128), -(-g // 4)
    p = torch.zeros(mb * 128, gb * 4, dtype=torch.uint8, device=s.device)
    p[:m, :g] = s.view(torch.uint8)
    return p.view(mb, 4, 32, gb, 4).permute(0, 3, 2, 1, 4).contiguous().view(mb * 128, gb * 4).view(s.dtype)


def _unblocked(p, m, g):
    mb, gb = p.shape[0] // 128, p.shape[1] // 4
    rows = p.view(torch.uint8).view(mb, gb, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(mb * 128, gb * 4)[:m, :g]
    return rows.contiguous().view(p.dtype)


def _scale_values(s):
    """Scales [.., g] as float32."""
    if s.dtype == torch.float8_e8m0fnu:
        e = s.view(torch.uint8).to(torch.int32) - 127
        return torch.ldexp(torch.ones(e.shape, device=e.device), e)
    return s.float()


def _table(dtype=torch.float32):
    v = torch.tensor(VALUES, dtype=dtype, device=DEV)
    return torch.stack((v.repeat(16), v.repeat_interleave(16)), -1)  # of every byte: the low half's value, the high half's


def _decode(codes, scales):
    """codes [.., k / 2], scales [.., g] in rows' order -> values [.., k] float32."""
    v = _table().index_select(0, codes.flatten().to(torch.int32)).view(*scales.shape, -1)
    return v.mul_(_scale_values(scales)[..., None]).flatten(-2)


# ---- inputs -----------------------------------------------------------------------------------------------------------


def _global_scale(x):
    """The scale that brings the largest value to the largest code under the largest group scale."""
    return (448.0 * 6.0 / x.abs().amax().float()).reshape(1)


def _activations(gen, m, k, dtype, outliers=0.001):
    """N(0, 1) rows, a value in a thousand ten times as large."""
    x = torch.randn(m, k, generator=gen, device=DEV, dtype=torch.float32)
    x = torch.where(torch.rand(m, k, generator=gen, device=DEV) < outliers, x * 10, x)
    return x.to(DTYPES[dtype])


def _operand(x, group):
    """What a program holds of a quantised operand: codes, scales in blocked order, the tensor's scale."""
    g = _global_scale(x) if group == 16 else torch.ones(1, device=DEV)
    v, s = _quantize(x, g, group)
    return _pack(v.flatten(-2)), _blocked(_scale_bytes(s[..., 0], group)), g


def _experts(gen, e, n, k):
    """Experts' weights [e, n, k]: codes, scales in rows' order, each expert's factor."""
    codes = torch.empty(e, n, k // 2, dtype=torch.uint8, device=DEV)
    scales = torch.empty(e, n, k // 16, dtype=torch.float8_e4m3fn, device=DEV)
    alpha = torch.empty(e, device=DEV)
    for b in range(e):
        w = torch.randn(n, k, generator=gen, device=DEV) * WEIGHT_STD
        g = _global_scale(w)
        v, s = _quantize(w, g, 16)
        codes[b], scales[b], alpha[b : b + 1] = _pack(v.flatten(-2)), _scale_bytes(s[..., 0], 16), 1.0 / g
    return codes, scales, alpha


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, m, dtype = case["kind"], case["m"], case["dtype"]
    if kind in ("quant", "silu"):
        x = _activations(gen, m, case["k"] * (2 if kind == "silu" else 1), dtype)
        scale = None
        if case["group"] == 16:  # a calibrated scale, not the tensor's own: a program has it before the rows
            scale = torch.full((1,), 448.0 * 6.0 / (60.0 if kind == "quant" else 400.0), device=DEV)
        return {"kind": kind, "x": x, "scale": scale, "group": case["group"]}
    if kind == "mm":
        group = case["group"]
        a, sa, ga = _operand(_activations(gen, m, case["k"], dtype), group)
        b, sb, gb = _operand(torch.randn(case["n"], case["k"], generator=gen, device=DEV) * WEIGHT_STD, group)
        bias = torch.randn(case["n"], generator=gen, device=DEV).to(DTYPES[dtype]) if case["bias"] else None
        return {"kind": kind, "a": a, "sa": sa, "b": b, "sb": sb, "alpha": 1.0 / (ga * gb) if group == 16 else None,
                "bias": bias, "dtype": DTYPES[dtype], "group": group}
    e, h, i = case["e"], case["h"], case["i"]
    w13, s13, a13 = _experts(gen, e, 2 * i, h)
    w2, s2, a2 = _experts(gen, e, h, i)
    x = _activations(gen, m, h, dtype)
    logits = torch.randn(m, e, generator=gen, device=DEV)
    weights, ids = torch.softmax(logits, -1).topk(case["topk"], -1)
    weights = weights / weights.sum(-1, keepdim=True)
    return {"kind": kind, "x": x, "w13": w13, "s13": s13, "a13": a13, "w2": w2, "s2": s2, "a2": a2, "weights": weights,
            "ids": ids.to(torch.int32)}


# ---- one pass ---------------------------------------------------------------------------------------------------------


def _silu_mul(x):
    gate, up = x.chunk(2, -1)
    return gate / (1.0 + torch.exp(-gate)) * up


def _plain(state):
    kind = state["kind"]
    if kind in ("quant", "silu"):
        x = _silu_mul(state["x"].double()) if kind == "silu" else state["x"]
        one = torch.ones(1, device=DEV)
        return _round_trip(x, one if state["scale"] is None else state["scale"], state["group"]).to(torch.bfloat16)
    if kind == "mm":
        (m, k), n, g = state["a"].shape, state["b"].shape[0], state["group"]
        a = _decode(state["a"], _unblocked(state["sa"], m, 2 * k // g))
        b = _decode(state["b"], _unblocked(state["sb"], n, 2 * k // g))
        out = a @ b.t()
        if state["alpha"] is not None:
            out = out * state["alpha"]
        if state["bias"] is not None:
            out = out + state["bias"].float()
        return out.to(state["dtype"])
    x, ids = state["x"], state["ids"].flatten()
    topk = state["ids"].shape[1]
    rows = x.float().repeat_interleave(topk, 0)[:, :, None]
    h = torch.bmm(_decode(state["w13"][ids], state["s13"][ids]), rows)[..., 0] * state["a13"][ids][:, None]
    h = _silu_mul(h)[:, :, None]
    y = torch.bmm(_decode(state["w2"][ids], state["s2"][ids]), h)[..., 0] * state["a2"][ids][:, None]
    return (y.view(*state["ids"].shape, -1) * state["weights"][..., None]).sum(1).to(x.dtype)


def run(state):
    if not own:
        return _plain(state)
    from sglang_b200 import ops

    kind = state["kind"]
    if kind == "mm":
        return ops.w4a4_group_fp4_matmul(state["a"], state["b"], state["sa"], state["sb"], state["alpha"],
                                         output_dtype=state["dtype"], bias=state["bias"])
    if kind == "moe":
        return ops.fused_experts_fp4(state["x"], state["w13"], state["w2"], state["s13"], state["s2"], state["weights"],
                                     state["ids"], w13_alpha=state["a13"], w2_alpha=state["a2"])
    quantizer = ops.silu_and_mul_quant_fp4 if kind == "silu" else ops.per_token_group_quant_fp4
    codes, scales = quantizer(state["x"], state["scale"], state["group"])
    return ops.per_token_group_dequant_fp4(codes, scales, state["scale"])


def work(case):
    kind, m = case["kind"], case["m"]
    if kind in ("quant", "silu"):
        values, two = m * case["k"], 2 if kind == "silu" else 1
        held = values // 2 + values // case["group"]  # codes and scales
        return {"bytes": values * two * DTYPES[case["dtype"]].itemsize + held + 2 * values, "flops": values * (4 + 6 * (two - 1))}
    if kind == "mm":
        n, k = case["n"], case["k"]
        held = (m + n) * (k // 2 + k // case["group"])
        return {"bytes": held + 2 * m * n, "flops": 2 * m * n * k}
    # experts that are expected to be named at all, when every token names `topk` different ones
    e, h, i = case["e"], case["h"], case["i"]
    live = e * (1.0 - (1.0 - case["topk"] / e) ** m)
    return {"bytes": live * 3 * h * i * 9 / 16 + 4 * m * h, "flops": 6 * m * case["topk"] * h * i}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------


def _near(q, table, even_first):
    """The nearest of the sorted `table` for q >= 0 (float64), ties to the entry whose index is even; beyond the end: the end."""
    t = torch.tensor(table, dtype=torch.float64, device=q.device)
    hi = torch.searchsorted(t, q).clamp(1, len(table) - 1)
    lo = hi - 1
    down, up = q - t[lo], t[hi] - q
    take = (down < up) | ((down == up) & (lo % 2 == (0 if even_first else 1)))
    return torch.where(take, t[lo], t[hi])


def _exact_round_trip(x, scale, group):
    grid4 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    grid8 = [m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0**e for e in range(-6, 9) for m in range(8)][:-1]
    m, k = x.shape
    out = torch.empty(m, k, dtype=torch.float64, device=x.device)
    for b in range(0, m, 1024):
        part = x[b : b + 1024].unflatten(-1, (-1, group))
        amax = part.abs().amax(-1, keepdim=True)
        if group == 32:
            s = torch.where(amax > 0, torch.exp2(torch.floor(torch.log2(amax)) - 2), 2.0**-127)
        else:
            s = _near(amax * scale / 6.0, grid8, True)
        v = _near((part * scale / torch.where(s > 0, s, 1.0)).abs(), grid4, True)
        v = torch.where(s > 0, torch.copysign(v, part), 0.0)
        out[b : b + 1024] = (v * s / scale).flatten(-2)
    return out


def _exact_weight(codes, scales):
    low, high = codes & 15, codes >> 4
    both = torch.stack((low, high), -1).flatten(-2).to(torch.int64)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=codes.device)
    v = torch.where(both >= 8, -grid[both % 8], grid[both % 8])
    byte = scales.view(torch.uint8).to(torch.float64)
    if scales.dtype == torch.float8_e8m0fnu:
        s = torch.exp2(byte - 127)
    else:
        e, f = torch.floor(byte / 8), byte % 8
        s = torch.where(e > 0, (1 + f / 8) * torch.exp2(e - 7), f / 8 * 2.0**-6)
    return v * s.repeat_interleave(v.shape[-1] // s.shape[-1], -1)


def _exact_rows_order(p, m, g):
    r = torch.arange(m, device=p.device)[:, None]
    c = torch.arange(g, device=p.device)[None, :]
    at = ((r // 128) * (p.shape[1] // 4) + c // 4) * 512 + (r % 32) * 16 + r % 128 // 32 * 4 + c % 4
    return p.view(torch.uint8).flatten()[at].view(p.dtype)


def exact(case, seed):
    st = prepare(case, seed)
    kind = st["kind"]
    if kind in ("quant", "silu"):
        x = st["x"].double()
        if kind == "silu":
            gate, up = x[:, : case["k"]], x[:, case["k"] :]
            x = gate * up / (1.0 + torch.exp(-gate))
        return _exact_round_trip(x, 1.0 if st["scale"] is None else float(st["scale"]), st["group"])
    if kind == "mm":
        m, n, g = case["m"], case["n"], case["k"] // case["group"]
        a = _exact_weight(st["a"], _exact_rows_order(st["sa"], m, g)).t().contiguous()
        scale = 1.0 if st["alpha"] is None else float(st["alpha"])
        out = torch.empty(m, n, dtype=torch.float64, device=DEV)
        sb = _exact_rows_order(st["sb"], n, g)
        for b in range(0, n, 4096):
            out[:, b : b + 4096] = (_exact_weight(st["b"][b : b + 4096], sb[b : b + 4096]) @ a).t() * scale
        return out if st["bias"] is None else out + st["bias"].double()
    x, ids = st["x"].double(), st["ids"].tolist()
    out = torch.zeros_like(x)
    for t, row in enumerate(ids):
        for j, e in enumerate(row):
            h = _exact_weight(st["w13"][e], st["s13"][e]) @ x[t] * st["a13"][e].double()
            gate, up = h[: case["i"]], h[case["i"] :]
            y = _exact_weight(st["w2"][e], st["s2"][e]) @ (gate * up / (1.0 + torch.exp(-gate)))
            out[t] += y * st["a2"][e].double() * st["weights"][t, j].double()
    return out
