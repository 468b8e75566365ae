"""GPU tests of sampling where a border decides: nuclei that leave next to nothing out, and places of the random number beside a token's border.

Tokens have to be those of 64-bit sums (sample_rows.py).  A border nearer than the step given there is decided by the weights' rounding: the rows where
that happens are counted, and a test says how many there may be.  Log-probabilities as in test_gpu_sample.py."""
import random

import numpy as np
import pytest
import torch

import qb200
from sample_rows import draw, logprob

pytestmark = pytest.mark.gpu
I32, F32 = torch.int32, torch.float32


def f32(v):
    return float(np.float32(v))


def check(x, u, t, k, p, m, undecided=0, runs=3):
    """x [N, V] on the device, the rest lists of N."""
    N, V = x.shape
    args = [torch.tensor(v, dtype=I32 if v is k else F32, device="cuda") for v in (u, t, k, p, m)]
    tokens, logprobs = qb200.sample(x, *args, want_logprobs=True)
    for _ in range(runs):
        assert torch.equal(qb200.sample(x, *args), tokens)
    rows = x.float().cpu().numpy()
    skipped = 0
    for i, (got, lp) in enumerate(zip(tokens.tolist(), logprobs.tolist())):
        want, margin, step = draw(rows[i], f32(u[i]), f32(t[i]), k[i], f32(p[i]), f32(m[i]))
        if margin <= step:
            skipped += 1
        else:
            assert got == want, f"row {i}: token {got}, expected {want}, margin {margin:.1e}, t {t[i]} k {k[i]} p {p[i]} m {m[i]} u {u[i]}"
        y = logprob(rows[i], got)
        assert abs(lp - y) <= 2.0 ** -22 * abs(y) + V * 2.0 ** -44 + 2.0 ** -21, f"row {i}: {lp} for {y}"
    assert skipped <= undecided, f"{skipped} rows lie on a border"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [2101, 3500, 8193, 20011, 33000, 60000])
def test_nuclei_of_nearly_everything(V, dtype):
    """top-p so near 1 that the steps in which the border is sought reach the end of the order; lists of every length beside what one may hold."""
    rng, N = random.Random(V), 24
    g = torch.Generator(device="cuda").manual_seed(V)
    std = torch.tensor([rng.uniform(0.3, 6.0) for _ in range(N)], device="cuda")[:, None]
    x = torch.randn(N, V, device="cuda", generator=g) * std
    x[::3, : V // 50] += 12.0                            # a few far above the rest
    # (bf16 logits are equal in hundreds, so that a border among them is one of index, and the sum that it meets one of many equal steps)
    check(x.to(dtype), [rng.random() for _ in range(N)], [rng.choice([0.5, 1.0, 1.7]) for _ in range(N)], [rng.choice([0, 0, V - 1, V * 3 // 4]) for _ in range(N)],
          [rng.uniform(0.996, 0.9999) for _ in range(N)], [0.0] * N)


def test_nuclei_whose_last_steps_hold_the_most():
    """Two heaps of logits in the last steps of the order, of sizes around those that a list takes, and top-p where the upper end of the search meets the
    whole sum."""
    rng = random.Random(5)
    torch.manual_seed(5)
    for far, other in ((1447, 1449), (1535, 1537), (2047, 2049), (700, 836)):
        N, V = 16, 6000
        x = torch.full((N, V), -1e30, device="cuda")
        x[:, 0] = 9.0
        for i in range(N):
            d = 1.0 + i * 0.55
            x[i, 1:1 + far] = 9.0 - d - torch.rand(far, device="cuda") * 0.004
            x[i, 1 + far:1 + far + other] = 9.0 - d - 1.0 - torch.rand(other, device="cuda") * 0.004
        x = x[:, torch.randperm(V, device="cuda")]
        check(x, [rng.random() for _ in range(N)], [1.0] * N, [0] * N, [rng.uniform(0.996, 0.9999) for _ in range(N)], [0.0] * N, runs=10)


def beside_borders(row, t, near, count, rng):
    """Random numbers in fp32 whose place lies within `near` (of a token's own weight) of that token's border, on either side."""
    w = np.exp((row.astype(np.float64) - float(row.max())) / t)
    run = np.cumsum(w.astype(np.longdouble))
    found = []
    while len(found) < count:
        u = f32(rng.uniform(0.3, 0.7))
        place = np.longdouble(u) * run[-1]
        i = int(np.searchsorted(run, place, side="right"))
        part = float((run[i] - place) / w[i])
        if w[i] < 1 and min(part, 1 - part) < near:
            found.append(u)
    return found


@pytest.mark.parametrize("top,t", [(16.5, 1.5), (16.5, 1.3), (17.9, 1.6), (9.1, 0.8)])
def test_places_beside_a_border_where_logits_lie_far_below_the_largest(top, t):
    """Half of the row at a logit whose distance from the largest is rounded up in fp32, half at one where it is rounded down, by nearly half a step: sums of
    fp32 weights lie a part of a token beside those of 64 bits, and the token may not be the neighbour for that."""
    V, N = 2 ** 19, 32
    top = f32(top)
    near = [np.float32(0.3)]
    for _ in range(200):
        near.append(np.nextafter(near[-1], np.float32(1)))
    off = [float(np.float32(v - np.float32(top))) - (float(v) - top) for v in near]
    row = np.empty(V, np.float32)
    row[: V // 2], row[V // 2:], row[0] = near[int(np.argmax(off))], near[int(np.argmin(off))], top
    # (the weights' rounding decides up to 2^-25 of the largest weight, the token's own is e^(-16.2 / 1.3) and more: a quarter of the 3 % around a border)
    some = N // 2
    u = beside_borders(row, t, 0.03, N, random.Random(int(top * 10)))
    x = torch.from_numpy(row).cuda()[None].expand(N, V)
    check(x, u, [t] * N, [0] * N, [1.0] * N, [1e-6] * N, undecided=some)
    check(x, u, [t] * N, [0] * N, [1.0] * N, [0.0] * N, undecided=some)
    check(torch.cat([x[:1, :1].expand(1, 1), x[:1, 1:].flip(1)], 1).expand(N, V), u, [t] * N, [0] * N, [1.0] * N, [1e-6] * N, undecided=some)


@pytest.mark.parametrize("size,steps", [(1e10, 1024.0), (-1e10, 1024.0), (3e37, 2.0 ** 101), (100.0, 2.0 ** -17)])
def test_logits_of_any_size(size, steps):
    """Logits a few steps of fp32 beside one another, at temperatures under, around and over a step."""
    N, V = 24, 5000
    torch.manual_seed(8)
    x = (torch.randint(-20, 21, (N, V), device="cuda", dtype=torch.float64) * steps + size).float()
    rng = random.Random(9)
    t = [min(steps * (0.01, 0.7, 5.0)[i % 3], 3e37) for i in range(N)]
    u = [rng.random() for _ in range(N)]
    check(x, u, t, [0] * N, [1.0] * N, [0.0] * N)
    check(x, u, t, [0] * N, [1.0] * N, [(0.0, 1e-4, 0.3)[i // 3 % 3] for i in range(N)])
    check(x, u, t, [0, 200] * (N // 2), [0.9, 0.99, 1.0] * (N // 3), [0.0] * N)
