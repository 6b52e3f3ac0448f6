"""What each request brings of its own, in 64 bits from the definitions, with bounds of
what the kernels' roundings may change.  numpy, on the host."""
import math

import numpy as np
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half a subnormal step


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def adapters(a, b, scales, ranks, sections, ids, x, base):
    """(output float64 [tokens][rows], bound of its error)."""
    dt = x.dtype
    a, b, scales, x, out = f64(a), f64(b), f64(scales), f64(x), f64(base)
    rank = b.shape[2]
    err = np.zeros_like(out)
    # the inner product is held as a sum of two numbers of the type, in float32, or better
    held = HALF_STEP[dt] ** 2
    for t, i in enumerate(ids.tolist()):
        if not 0 <= i < a.shape[0]:
            continue
        r = rank if ranks is None else min(max(int(ranks[i]), 0), rank)
        row = 0
        for s, many in enumerate(sections):
            down = a[i, s * rank:s * rank + r]
            up = b[i, row:row + many, :r]
            h = down @ x[t]
            # float32 sums of cols products, in any order; then of rank products
            off = held * np.abs(h) + x.shape[1] * 2.0 ** -24 * (np.abs(down) @ np.abs(x[t]))
            out[t, row:row + many] += scales[i] * (up @ h)
            err[t, row:row + many] += abs(scales[i]) * (
                np.abs(up) @ off + (2 * r + 4) * 2.0 ** -24 * (np.abs(up) @ np.abs(h)))
            row += many
    # float32 of base + delta, then the type's rounding
    err += 2.0 ** -23 * (np.abs(out) + np.abs(f64(base)))
    return out, err * (1 + HALF_STEP[dt]) + HALF_STEP[dt] * np.abs(out) + SMALLEST[dt]


def _row(logits):
    l = np.array(logits, dtype=np.float64)
    l[np.isnan(l)] = -math.inf
    return l


def _weights(l, temperature):
    """Weights of logits in the order's sequence, l[0] the largest (not minus infinity)."""
    with np.errstate(invalid="ignore", over="ignore"):
        d = (l - l[0]) / temperature
    d[l == l[0]] = 0.0
    d[np.isneginf(l)] = -math.inf
    return np.exp(d)


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log-probability, number of kept tokens) of one row."""
    l = _row(logits)
    order = np.lexsort((np.arange(len(l)), -l))
    l = l[order]
    if np.isneginf(l[0]):
        return -1, -math.inf, 0
    l = l[~np.isneginf(l)]
    if not temperature > 0 or top_p <= 0:
        return int(order[0]), 0.0, 1
    # 64 bits of mantissa: sums of thousands of weights beside which one of 1e-14 counts
    w = _weights(l, temperature).astype(np.longdouble)
    n = len(w) if top_k <= 0 else min(top_k, len(w))
    first = n
    if top_p < 1:
        total = w[:n].cumsum()
        before = np.concatenate(([0.0], total[:-1]))
        n = min(n, int((before < top_p * total[-1]).sum()))
    if min_p > 0:
        n = min(n, int((w[:first] >= min(min_p, 1.0)).sum()))
    total = w[:n].cumsum()
    u = min(max(u, 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    at = int(np.argmax(total > u * total[-1]))
    return int(order[at]), math.log(float(w[at] / total[-1])), n


def logprobs(logits, top):
    """(log-probabilities [vocab], their bounds, ids of the top ones) of one row."""
    l = _row(logits)
    order = np.lexsort((np.arange(len(l)), -l))
    best = l[order[0]]
    if np.isneginf(best):
        return np.full(len(l), -math.inf), np.zeros(len(l)), order[:top]
    w = np.zeros(len(l))
    w[order] = _weights(l[order], 1.0)
    rest = w[order[1:]].sum()
    if math.isinf(best):
        far, out = np.zeros(len(l)), np.where(w > 0, 0.0, -math.inf) - math.log1p(rest)
    else:
        far = np.where(np.isneginf(l), 0.0, best - np.where(np.isneginf(l), best, l))
        out = np.where(np.isneginf(l), -math.inf, l - best - math.log1p(rest))
    # the others' weights: float32 differences (2^-24 of them) and exponentials (2 steps),
    # and those that float32 has no normal number for (2^-126) may count as nothing, each
    lost = float((np.where(w < 1, w, 0.0) * (far + 4) * 2.0 ** -23).sum()) + 2.0 ** -126
    lost += float(np.where(w < 2.0 ** -125, w, 0.0).sum())
    err = lost / (1 + rest) + 2.0 ** -24 * np.where(np.isfinite(out), np.abs(out), 0.0) + 2.0 ** -149
    return out, err * 1.001, order[:top]
