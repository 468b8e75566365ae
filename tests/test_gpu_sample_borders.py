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
