"""GPU tests of sampling a token from rows of logits, against the definition step by step in 64 bits.

Tokens have to be equal.  Weights are rounded to 2^-45 of the largest (half a step of 2^-44) and their sums hold n of them, so a border nearer
than n * 2^-44 of the sum is decided by that; the inputs' own borders are asserted to lie further away before the tokens are looked at.
Log-probabilities: half a step of the fp32 result, 2^-24 relative, a sum of n whole numbers of 2^-44 off by half of one each and the fp64 functions: 2^-24 |y|
+ n * 2^-44 + 2^-40; sums in fp32 of terms of 2^-22 (an approximate exponential) are allowed for with 2^-21 + 2^-22 |y|."""
import math
import random

import numpy as np
import pytest
import torch

import qb200
from drafted_ref import sample as plain

pytestmark = pytest.mark.gpu
I32, F32 = torch.int32, torch.float32
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def settings(N, seed, kinds=None):
    rng = random.Random(seed)
    kinds = kinds or dict(t=[0.0, 0.3, 0.7, 1.0, 1.7], k=[0, 1, 3, 50, 700, 10 ** 6], p=[1.0, 0.95, 0.5, 0.01, 0.0], m=[0.0, 0.02, 0.3, 1.0])
    return {n: [rng.choice(v) for _ in range(N)] for n, v in kinds.items()}


def check(x, u, s, **kw):
    """x [N, V] on the device, u and the settings as lists."""
    N, V = x.shape
    dev = lambda v, d=F32: torch.tensor(v, dtype=d, device="cuda")
    tokens, logprobs = qb200.sample(x, dev(u), dev(s["t"]), dev(s["k"], I32), dev(s["p"]), dev(s["m"]), want_logprobs=True, **kw)
    again = qb200.sample(x, dev(u), dev(s["t"]), dev(s["k"], I32), dev(s["p"]), dev(s["m"]))
    assert torch.equal(tokens, again)
    rows = x.double().cpu().tolist()
    f = lambda v: float(np.float32(v))
    got, lp = tokens.tolist(), logprobs.tolist()
    for i in range(N):
        want, margin = plain(rows[i], f(u[i]), f(s["t"][i]), s["k"][i], f(s["p"][i]), f(s["m"][i]))
        if margin <= V * 2.0 ** -44:
            continue                                    # (decided below the weights' step; counted by the caller's inputs)
        assert got[i] == want, f"row {i}: token {got[i]}, expected {want}, margin {margin:.1e}, settings {({k: v[i] for k, v in s.items()})}"
        if want < 0:
            assert lp[i] == 0
            continue
        r = [-math.inf if math.isnan(v) else v for v in rows[i]]
        top = max(r)
        y = (0.0 if r[want] == top else r[want] - top) - math.log(math.fsum(1.0 if v == top else math.exp(v - top) for v in r))
        assert abs(lp[i] - y) <= 2.0 ** -22 * abs(y) + V * 2.0 ** -44 + 2.0 ** -21, f"row {i}: {lp[i]} for {y}"


def logits(N, V, dtype, seed, std=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(N, V, device="cuda", generator=g) * std
    x[:, :: max(1, V // 9)] += torch.rand(x[:, :: max(1, V // 9)].shape, device="cuda", generator=g) * 9
    return x.to(dtype)


def uniform(N, seed):
    return [random.Random(seed * 1000 + i).random() for i in range(N)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 32, 255, 1000, 4097, 8192, 16001, 32768, 50001])
def test_sizes_and_settings(V, dtype):
    N = 40 if V < 10000 else 16
    check(logits(N, V, dtype, V), uniform(N, V), settings(N, V))


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_vocabularies(dtype):
    check(logits(6, 151667, dtype, 1), uniform(6, 1), settings(6, 1))
    check(logits(4, 262144, dtype, 2, 1.0), uniform(4, 2), settings(4, 2, dict(t=[1.0, 2.0], k=[0, 100000], p=[0.97, 1.0], m=[0.0, 1e-4])))
    check(logits(2, 2 ** 19, dtype, 3), uniform(2, 3), settings(2, 3, dict(t=[1.0], k=[0], p=[0.9, 1.0], m=[0.0])))


def test_every_setting_by_itself_and_together():
    for i, kinds in enumerate([dict(t=[1.0], k=[0], p=[1.0], m=[0.0]), dict(t=[0.0], k=[0], p=[1.0], m=[0.0]), dict(t=[0.8], k=[40], p=[1.0], m=[0.0]),
                               dict(t=[0.8], k=[0], p=[0.9], m=[0.0]), dict(t=[0.8], k=[0], p=[1.0], m=[0.1]), dict(t=[0.8], k=[40], p=[0.9], m=[0.1]),
                               dict(t=[50.0], k=[2000], p=[0.99], m=[0.0]), dict(t=[0.01], k=[0], p=[0.9], m=[0.0])]):
        check(logits(24, 5000, torch.bfloat16, i), uniform(24, i), settings(24, i, kinds))


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_logits_go_by_index(dtype):
    """All alike, few values, two values: every border lies among equal logits."""
    N, V = 30, 3001
    g = torch.Generator(device="cuda").manual_seed(4)
    for x in (torch.zeros(N, V, device="cuda"), torch.randint(0, 3, (N, V), device="cuda", generator=g).float(), torch.randint(0, 2, (N, V), device="cuda", generator=g) * -30.0,
              torch.randint(-4, 5, (N, V), device="cuda", generator=g) / 4.0):
        check(x.to(dtype), uniform(N, 5), settings(N, 6))
    x = torch.zeros(N, V, device="cuda").to(dtype)
    x[:, ::2] = -0.0                                     # (equal to 0)
    check(x, uniform(N, 6), settings(N, 7))
    check(torch.full((3, 200000), 1.5, device="cuda", dtype=dtype), uniform(3, 7), dict(t=[1.0] * 3, k=[0, 150001, 70000], p=[0.7, 1.0, 0.3], m=[0.0] * 3))


@pytest.mark.parametrize("dtype", DTYPES)
def test_masks_and_what_is_not_finite(dtype):
    N, V = 48, 2500
    x = logits(N, V, dtype, 8)
    g = torch.Generator(device="cuda").manual_seed(9)
    out = torch.rand(N, V, device="cuda", generator=g) < 0.9
    low = torch.finfo(dtype).min
    x[:16] = x[:16].masked_fill(out[:16], -math.inf)
    x[16:32] = x[16:32].masked_fill(out[16:32], low)
    x[32] = -math.inf                                    # nothing to choose from
    x[33] = low                                          # everything at the type's lowest value
    x[34] = math.nan
    x[35, 100:] = math.nan
    x[36, 77] = math.inf
    x[37, 5::7] = math.inf
    x[38] = -math.inf
    x[38, V - 1] = -3.0
    x[39] = -math.inf
    x[39, 3], x[39, 9] = low, low
    x[40, :] = torch.finfo(dtype).max
    x[41, ::3] = torch.finfo(dtype).max
    x[41, 1::3] = low
    check(x, uniform(N, 10), settings(N, 11))
    check(x, uniform(N, 12), settings(N, 13, dict(t=[1.0, 0.0, 0.5], k=[0, 5], p=[1.0, 0.9], m=[0.0])))


def test_settings_at_their_ends():
    nan, inf = math.nan, math.inf
    x = logits(1, 300, torch.float32, 14).expand(14, 300)
    s = dict(t=[nan, -1.0, inf, 1e-30, 1e30, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0], k=[0, 0, 0, 0, 0, -5, 300, 301, 2 ** 31 - 1, 0, 0, 0, 0, 0],
             p=[1.0] * 9 + [nan, -1.0, 2.0, 1.0, 1.0], m=[0.0] * 12 + [nan, 2.0])
    u = uniform(14, 15)
    dev = lambda v, d=F32: torch.tensor(v, dtype=d, device="cuda")
    got = qb200.sample(x, dev(u), dev(s["t"]), dev(s["k"], I32), dev(s["p"]), dev(s["m"])).tolist()
    row = x[0].double().tolist()
    best = max(range(300), key=lambda i: (row[i], -i))
    f = lambda v: float(np.float32(v))
    assert got[0] == best and got[1] == best                     # no temperature above 0: greedy
    assert got[2] == int(f(u[2]) * 300)                          # an infinite one: all alike
    assert got[3] == best
    for i in (4, 5, 6, 7, 8):
        assert got[i] == plain(row, f(u[i]), f(s["t"][i]), max(0, min(s["k"][i], 300)), 1.0, 0.0)[0]
    assert got[9] == plain(row, f(u[9]), 1.0, 0, 1.0, 0.0)[0]    # NaN filters are none
    assert got[10] == best and got[11] == plain(row, f(u[11]), 1.0, 0, 1.0, 0.0)[0]
    assert got[12] == plain(row, f(u[12]), 1.0, 0, 1.0, 0.0)[0] and got[13] == best


def test_random_numbers_at_their_ends():
    x = logits(8, 1000, torch.float32, 16)
    x[:, 0] = -math.inf
    x[:, -1] = -math.inf
    dev = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, math.nan, math.inf, 1e-45], device="cuda")
    assert qb200.sample(x, dev).tolist() == [1, 998, 998, 998, 1, 1, 998, 1]


def test_defaults_strides_and_one_setting_for_all():
    x = logits(20, 1203, torch.bfloat16, 17)
    u = uniform(20, 18)
    dev = torch.tensor(u, device="cuda")
    one = dict(t=[1.0] * 20, k=[0] * 20, p=[1.0] * 20, m=[0.0] * 20)
    check(x, u, one)
    want = qb200.sample(x, dev)
    wide = torch.full((20, 1500), 50.0, dtype=x.dtype, device="cuda")
    wide[:, 7:1210] = x
    assert torch.equal(qb200.sample(wide[:, 7:1210], dev), want)
    every = torch.zeros(20, 3, device="cuda")
    every[:, 1] = dev
    assert torch.equal(qb200.sample(x, every[:, 1]), want)
    t = torch.tensor([0.6], device="cuda")
    a = qb200.sample(x, dev, t.expand(20), torch.tensor([30], dtype=I32, device="cuda").expand(20), want_logprobs=True)
    b = qb200.sample(x, dev, t.repeat(20), torch.full((20,), 30, dtype=I32, device="cuda"), want_logprobs=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    same = qb200.sample(x[3:4].expand(9, 1203), dev[:9])
    assert same.tolist() == [plain(x[3].double().tolist(), float(np.float32(v)), 1.0, 0, 1.0, 0.0)[0] for v in u[:9]]
    assert qb200.sample(x[:0], dev[:0]).shape == (0,)
    # columns of a tensor whose rows are far apart: beyond 2^32 bytes
    far = torch.empty(3, 600_000_000, dtype=torch.float32, device="cuda")[:, :1203]
    far.copy_(x[:3].float())
    assert torch.equal(qb200.sample(far, dev[:3]), want[:3])


def test_frequencies_follow_the_weights():
    """Evenly spaced numbers: every token is drawn as often as its weight says, to one draw."""
    n = 4096
    x = torch.tensor([0.0, 1.0, -math.inf, 2.0, 0.5, 3.0], device="cuda")
    u = (torch.arange(n, device="cuda") + 0.5) / n
    got = torch.bincount(qb200.sample(x.expand(n, 6), u.float()).long(), minlength=6).double().cpu()
    want = torch.softmax(x.double(), 0).cpu() * n
    assert (got - want).abs().max() <= 1.0 + 1e-6


def test_streams_and_graphs():
    x = logits(33, 30011, torch.bfloat16, 19)
    u = torch.tensor(uniform(33, 20), device="cuda")
    t, k, p = torch.full((33,), 0.9, device="cuda"), torch.full((33,), 60, dtype=I32, device="cuda"), torch.full((33,), 0.9, device="cuda")
    want = qb200.sample(x, u, t, k, p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = qb200.sample(x, u, t, k, p)
    side.synchronize()
    assert torch.equal(a, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = qb200.sample(x, u, t, k, p)
    x2, u2 = logits(33, 30011, torch.bfloat16, 21), torch.tensor(uniform(33, 22), device="cuda")
    expect = qb200.sample(x2, u2, t, k, p)
    x.copy_(x2)
    u.copy_(u2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, expect)
    for _ in range(4):
        assert torch.equal(qb200.sample(x, u, t, k, p), expect)


def test_without_clusters(no_clusters):
    check(logits(8, 60000, torch.bfloat16, 23), uniform(8, 24), settings(8, 25))
    check(logits(3, 262143, torch.float32, 26), uniform(3, 27), settings(3, 28))
