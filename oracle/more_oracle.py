"""Low-rank adapters, the router's product and routing from their definitions, in float64 on the CPU (numpy)."""
from __future__ import annotations

import numpy as np

F32_MAX = float(np.finfo(np.float32).max)


def lora_add(base, x, a, b, ids, scalings, ranks, slices):
    """(out unrounded, what the adapter's sums add up in magnitude) as float64 [T, N]."""
    out, mass = base.astype(np.float64).copy(), np.zeros(base.shape)
    R = b.shape[2]
    for t, l in enumerate(ids):
        if not 0 <= l < a.shape[0]:
            continue
        r, lo = int(min(max(ranks[l], 0), R)), 0
        for s, width in enumerate(slices):
            rows = a[l, s * R : s * R + r]
            h, hm = rows @ x[t], np.abs(rows) @ np.abs(x[t])
            cols = b[l, lo : lo + width, :r]
            out[t, lo : lo + width] += scalings[l] * (cols @ h)
            mass[t, lo : lo + width] += abs(scalings[l]) * (np.abs(cols) @ hm)
            lo += width
    return out, mass


def route(x, topk, scoring, bias=None, groups=1, kept=1, top=1, renorm=True, factor=1.0):
    """(weights float64, ids) of the logits x [T, E] (float64 values).  c that float64 holds as equal go by their logits (which is the order of
    the real numbers where their biases are equal), then by index; groups likewise where one c is their value."""
    T, E = x.shape
    w, ids = np.zeros((T, topk)), np.full((T, topk), -1, dtype=np.int32)
    for t in range(T):
        v = np.where(np.isnan(x[t]), -np.inf, np.minimum(x[t], F32_MAX))
        live = v > -np.inf
        if not live.any():
            continue
        with np.errstate(over="ignore"):
            if scoring == "softmax":
                mx = v[live].max()
                logs = v - mx - np.log(np.exp(v[live] - mx).sum())
            else:
                logs = np.minimum(v, 0.0) - np.log1p(np.exp(-np.abs(v)))
        s = np.where(live, np.exp(logs), 0.0)
        c = s if bias is None else s + bias
        c = np.where(live & (c > -np.inf), c, -np.inf)  # (a NaN is not greater)
        key = c if bias is not None else v
        allowed = np.ones(E, bool)
        if groups > 1:
            value, second = np.full(groups, -np.inf), np.zeros(groups)
            for g in range(groups):
                of = (v if bias is None and top == 1 else c)[g * (E // groups) : (g + 1) * (E // groups)]
                best = sorted((z for z in of if z > -np.inf), reverse=True)[:top]
                if best:
                    value[g] = sum(best)
                    if top == 1:
                        second[g] = max(z for z, cz in zip(v[g * (E // groups) : (g + 1) * (E // groups)], of) if cz == best[0])
            order = sorted(range(groups), key=lambda g: (-value[g], -second[g], g))[:kept]
            allowed = np.repeat([g in order for g in range(groups)], E // groups)
        order = sorted((e for e in range(E) if allowed[e] and c[e] > -np.inf), key=lambda e: (-key[e], -v[e], e))[:topk]
        ids[t, : len(order)] = order
        if order:
            if renorm:
                part = np.exp(logs[order] - logs[order].max())
                w[t, : len(order)] = part / part.sum() * factor
            else:
                w[t, : len(order)] = s[order] * factor
    return w, ids
