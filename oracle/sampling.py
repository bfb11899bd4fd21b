"""Oracle of the sampler: one row at a time, sorted, in float64 on the CPU (the reference samples by temperature alone,
``inference/layers/sampler.py:5-10``)."""

import math


def kept(x, t, k=0, p=1.0, m=0.0):
    """{index: weight} of the tokens that the filters keep; t > 0, no NaN among x."""
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    top = x[order[0]]

    def weight(v):
        return 1.0 if v == top else math.exp((v - top) / t) if v != -math.inf else 0.0

    order = order[:k] if 0 < k < len(x) else order
    w = [weight(x[i]) for i in order]
    total, before, out = math.fsum(w), 0.0, {}
    for n, (i, v) in enumerate(zip(order, w)):
        if p < 1 and n and not before < p * total:
            break
        if m > 0 and v < min(m, 1.0):
            break
        out[i] = v
        before += v
    return out


def draw(x, u, t, k=0, p=1.0, m=0.0):
    """The answer of one row, a list of floats."""
    for i, v in enumerate(x):
        if v != v:
            return i
    if not t > 0:
        return max(range(len(x)), key=lambda i: (x[i], -i))
    w = kept(x, t, k, p, m)
    u = min(max(u, 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    aim, c = u * math.fsum(w.values()), 0.0
    for i in sorted(w):
        c += w[i]
        if c > aim:
            return i
    return max(w)
