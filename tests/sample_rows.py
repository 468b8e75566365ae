"""A row's token by the definition in 64 bits, on arrays, for rows too long or too many for the step-by-step restatement in drafted_ref.py.

Margins are in units of the largest weight.  There the kernel's sums are known: every weight is rounded to 2^-45 and its exponential off by 2.3e-15 of itself, so
that two sums that are compared differ by (V + 2) 2^-44 and 2^-48 of the whole sum from those of the definition, borders rounded to whole numbers
and products in fp64 among that (``step``)."""
import math

import numpy as np


def weights(row, t):
    l = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    top = l.max()
    return l, top, np.where(l == top, 1.0, np.exp((l - top) / t))


def draw(row, u, t, k, p, least):
    """(token, margin, step): the token, how near the nearest border that decided it lies, and how near one is decided by the weights' rounding.  For a
    temperature above 0 and a row with something in it."""
    l, top, w = weights(row, t)
    step = (len(l) + 2) * 2.0 ** -44 + float(w.sum()) * 2.0 ** -48
    order = np.argsort(-l, kind="stable")
    margin = math.inf
    if k > 0:
        order = order[:k]
    if p < 1:
        run = np.cumsum(w[order].astype(np.longdouble))
        goal = np.longdouble(p) * run[-1]
        n = max(1, int(np.searchsorted(run, goal, side="left")) + 1)
        near = run[max(0, n - 2):n + 1]
        near = near[1:] if n == 1 else near          # (the first stays whatever it weighs)
        margin = min([margin] + [float(abs(v - goal)) for v in near if v != run[-1]])
        order = order[:n]
    keep = order[(w[order] >= least) | (order == order[0])] if least > 0 else order
    if least > 0:
        if np.min(np.abs(w[order][w[order] < 1] - least), initial=1.0) <= least * 2.0 ** -48:    # (two exponentials in 64 bits)
            margin = 0.0
    keep = np.sort(keep)
    run = np.cumsum(w[keep].astype(np.longdouble))
    goal = np.longdouble(u) * run[-1]
    i = min(int(np.searchsorted(run, goal, side="right")), len(keep) - 1)
    near = [run[j] for j in (i - 1, i) if 0 <= j < len(keep) - 1]
    margin = min([margin] + [float(abs(v - goal)) for v in near])
    return int(keep[i]), margin, step


def logprob(row, token):
    l, top, _ = weights(row, 1.0)
    return (0.0 if l[token] == top else float(l[token] - top)) - math.log(float(np.sum(np.where(l == top, 1.0, np.exp(l - top)).astype(np.longdouble))))
