"""Plain 64-bit evaluations of routing, rotary positions and log probabilities, row by row from their definitions."""
import numpy as np


def route(logits, bias, k, score, groups, keep, group_score, renorm, scale):
    """(idx [T][k], w fp64 [T][k]) from logits [T][E] of any float type, as include/berth_b200.h words it."""
    T, E = logits.shape
    gs = E // groups
    idx, w = np.empty((T, k), np.int64), np.empty((T, k))
    for t in range(T):
        l = logits[t].astype(np.float64)
        l = np.where(l == np.inf, float(np.finfo(np.float32).max), l)
        nan, masked = np.isnan(l), l == -np.inf
        live = ~nan & ~masked
        s = np.zeros(E)
        with np.errstate(over="ignore"):
            if score == "sigmoid":
                s[live] = 1.0 / (1.0 + np.exp(-l[live]))
            elif live.any():
                s[live] = np.exp(l[live] - l[live].max())
                s /= s.sum()
        sums = group_score == "top2" and keep < groups
        c = l if bias is None and not sums else (s if bias is None else s + bias.astype(np.float64))
        c = np.where(live, c, -np.inf)
        cand = np.arange(E)
        if keep < groups:
            worth = []
            for g in range(groups):
                best = np.sort(c[g * gs:(g + 1) * gs])[::-1]
                v = best[0]
                if sums and gs > 1 and best[1] > -np.inf:
                    v = best[0] + best[1]
                worth.append(v)
            kept = sorted(range(groups), key=lambda g: (-worth[g], g))[:keep]
            cand = np.concatenate([np.arange(g * gs, (g + 1) * gs) for g in sorted(kept)])
        order = sorted(cand, key=lambda e: (nan[e], -c[e] if not nan[e] else 0.0, e))[:k]
        idx[t] = order
        sel = s[order]
        if renorm:
            if score == "softmax":     # relative to the chosen, so that nothing underflows
                m = l[order][live[order]].max() if live[order].any() else 0.0
                sel = np.where(live[order], np.exp(np.where(live[order], l[order] - m, 0.0)), 0.0)
            else:                      # ln sigmoid = min(l, 0) - ln(1 + exp(-|l|)), relative to the largest
                ls = np.where(live[order], np.minimum(l[order], 0) - np.log1p(np.exp(-np.abs(l[order]))), -np.inf)
                m = ls.max()
                sel = np.exp(ls - m) if m > -np.inf else np.zeros(k)
            total = sel.sum()
            sel = sel / total if total > 0 else sel
        w[t] = np.nan if nan.any() else sel * scale
    return idx, w


def rope(x, positions, inv_freq, interleaved, factor, norm, eps, bias):
    """[T][heads][dim] fp64 from any float type; norm fp64 [dim] or None."""
    y = x.astype(np.float64)
    if norm is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * (norm + bias)
    half = len(inv_freq)
    turns = positions.astype(np.int64)[:, None].astype(np.float64) * inv_freq[None, :]
    cos, sin = factor * np.cos(turns)[:, None, :], factor * np.sin(turns)[:, None, :]
    out = y.copy()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    out[..., a] = y[..., a] * cos - y[..., b] * sin
    out[..., b] = y[..., b] * cos + y[..., a] * sin
    size = np.abs(y)                       # what an output's rounding errors scale with
    pair = np.abs(y[..., a]) + np.abs(y[..., b])
    size[..., a] = size[..., b] = abs(factor) * pair
    return out, size


def logprobs(logits, tokens, top, inv_temp):
    """dict of fp64 / int arrays; logits [rows][vocab]."""
    R, V = logits.shape
    out = {"logprob": np.zeros(R), "rank": np.full(R, -1, np.int64), "entropy": np.zeros(R), "top": np.zeros((R, top), np.int64),
           "top_logprob": np.zeros((R, top))}
    for r in range(R):
        x = logits[r].astype(np.float64)
        nan = np.isnan(x)
        order = np.lexsort((np.arange(V), np.where(nan, 0.0, -x), nan))      # NaN last, then larger first, then lower token
        place = np.empty(V, np.int64)
        place[order] = np.arange(V)
        z = x * inv_temp
        if nan.any() or (x == np.inf).any():
            lp, h = np.full(V, np.nan), np.nan
        elif (x == -np.inf).all():
            lp, h = np.full(V, -np.inf), 0.0
        else:
            d = z - z.max()
            e = np.exp(d)
            lp = d - np.log(e.sum())
            h = -(np.exp(lp) * np.where(np.isinf(lp), 0.0, lp)).sum()
        if tokens is not None and 0 <= tokens[r] < V:
            out["logprob"][r] = lp[tokens[r]]
            out["rank"][r] = -1 if nan[tokens[r]] else place[tokens[r]]
        out["entropy"][r] = h
        out["top"][r] = order[:top]
        out["top_logprob"][r] = lp[order[:top]]
    return out
