"""Plain restatements of the operators on drafted tokens, for the tests: in 64 bits, step by step on Python lists."""
import math

import torch

F64 = torch.float64


def dequantized(pool, bits):
    """The values of a pool's rows, fp64 [pages, heads, page, D]."""
    if bits == 16:
        return pool[0].to(F64)
    w, s, b = pool
    q = ((w[..., None].to(torch.int64) >> (torch.arange(32 // bits, device=w.device) * bits)) & (2 ** bits - 1)).reshape(*w.shape[:-1], -1)
    return q.to(F64) * s.to(F64).repeat_interleave(64, -1) + b.to(F64).repeat_interleave(64, -1)


def line_of(parents, t):
    """Node t and the nodes before it, itself first."""
    line = [t]
    while 0 <= parents[line[-1]] < line[-1]:
        line.append(parents[line[-1]])
    return line


def visible(parents, t, n, length, window, sinks):
    """(place, position) of every token that node t sees."""
    base = length - n
    depth = [len(line_of(parents, i)) - 1 for i in range(n)]
    me = base + depth[t]
    tokens = [(j, j) for j in range(base)] + [(base + i, base + depth[i]) for i in sorted(line_of(parents, t))]
    return [(j, at) for j, at in tokens if window <= 0 or at > me - window or at < sinks]


def attention(q, k, v, scale):
    """q [R, D], k, v [T, D] fp64: result, sum p |v|, largest scale * sum |q| |k| of a row."""
    if k.shape[0] == 0:
        return torch.zeros_like(q), torch.zeros_like(q), torch.zeros(q.shape[0], 1, dtype=F64, device=q.device)
    p = torch.softmax(q @ k.T * scale, -1)
    return p @ v, p @ v.abs(), (abs(scale) * q.abs() @ k.abs().T).amax(-1, keepdim=True)


def tolerance(o, A, S, bits, v):
    """Of one output o = sum p v of the tree attention over the values v: half a bf16 step of the result, 2^-8 |o|, and against A = sum p |v|:
    half a step of every probability (bf16 beside bf16 values, 2^-8; else fp16, 2^-11), half an fp16 step of the values at 4 and 8 bits
    (2^-11), the approximate exponential (a cubic of 7.5e-5 may stand for it: 2^-12 for sum and normaliser), and twice the scores' error: at 4
    and 8 bits half an fp16 step of every key, 2^-11 of S = scale * sum |q| |k|, and fp32 sums whose roundings, truncating ones too, are off
    by 2^-23 of S each step of 16 products and for the reference, 20 in all.

    Probabilities under fp16's normal range are off by 2^-25 each, whatever the sum A at that dim: a token's P' = p 2^(e - r) meets
    v 2^-e < 2^15, so n of them move the sum by at most n 2^-25 2^15.  The reference was placed where the largest P' was 2^8, of a token with a
    value of M >= 2^14 2^e: its p alone makes the normaliser at least 2^8 2^-e >= 2^22 / M.  So the result moves by at most
    n 2^-10 M 2^-22 = n 2^-32 M, M at most the largest |v|."""
    quantised = bits != 16
    part = 2.0 ** -8 if not quantised else 2.0 ** -11 + 2.0 ** -11
    small = v.shape[0] * 2.0 ** -32 * float(v.abs().max()) if quantised and v.numel() else 0.0
    return 2.0 ** -8 * o.abs() + A * (part + 2.0 ** -12 + S * (40 * 2.0 ** -23 + (2.0 ** -10 if quantised else 0.0))) * 1.01 + small + 1e-30


def sample(x, u, t, k, p, least):
    """One row: (token, margin): the token, and how far (relative to the sum) the nearest border that decided it lies."""
    l = [-math.inf if math.isnan(v) else v for v in x]
    top = max(l)
    if top == -math.inf:
        return -1, 1.0
    order = sorted(range(len(l)), key=lambda i: (-l[i], i))
    if not t > 0:
        return order[0], 1.0
    w = {i: 1.0 if l[i] == top else (0.0 if l[i] == -math.inf else math.exp((l[i] - top) / t)) for i in order}
    margin = 1.0
    if k > 0:
        order = order[:k]
    if p < 1:
        total = math.fsum(w[i] for i in order)
        run, n = 0.0, 0
        for i in order:
            if n and run >= p * total:
                break
            if n:
                margin = min(margin, (p * total - run) / total)
            run += w[i]
            n += 1
        if n < len(order):
            margin = min(margin, abs(run - p * total) / total)
        order = order[:n]
    first = order[0]
    order = [i for i in order if i == first or not least > 0 or w[i] >= least]
    total = math.fsum(w[i] for i in order)
    run, token = 0.0, None
    for i in sorted(order):
        run += w[i]
        margin = min(margin, abs(run - u * total) / total) if run != total else margin
        if run > u * total:
            token = i
            break
    return max(order) if token is None else token, margin


def walk(parents, tokens, sampled, n):
    """The nodes that the samples confirm."""
    if n == 0:
        return []
    path = [0]
    while True:
        child = [i for i in range(path[-1] + 1, n) if parents[i] == path[-1] and tokens[i] == sampled[path[-1]]]
        if not child:
            return path
        path.append(child[0])
