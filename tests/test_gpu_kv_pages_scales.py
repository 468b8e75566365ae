"""GPU tests of the attention over pages where the two scale groups of a head, or the tokens of a group, differ by much in size: the error
of every dim stays within the bounds of test_gpu_kv_pages_attention.py, which count that dim's own values."""
import pytest
import torch

import qb200
from test_gpu_kv_pages_attention import BF16, check, ints, make_pool, make_table, run

pytestmark = pytest.mark.gpu
D, H = 128, 2


def sized(pool, group, factor):
    """The pool with a group's values times a power of two, which changes no code."""
    q, s, b = (t.clone() for t in pool)
    s[..., group] = (s[..., group].float() * factor).to(BF16)
    b[..., group] = (b[..., group].float() * factor).to(BF16)
    return q, s, b


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("small", [0, 1])
@pytest.mark.parametrize("steps", [12, 20, 24, 32, 60])
@pytest.mark.parametrize("lens", [[500, 90], [6000, 1]])
def test_one_group_far_below_the_other(bits, small, steps, lens):
    torch.manual_seed(steps + small)
    page = 32
    P = sum(-(-n // page) for n in lens)
    kp, vp = make_pool(P, H, page, D, bits), make_pool(P, H, page, D, bits)
    vp = sized(sized(vp, small, 2.0 ** -(steps // 2)), 1 - small, 2.0 ** (steps - steps // 2))
    table = make_table(lens, page, -(-lens[0] // page), P)
    q, out = run(kp, vp, table, lens, bits, 2, 8, D)
    check(out, q, kp, vp, table, lens, page, bits, D ** -0.5)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("power", [1.0, -1.0, 0.25])
def test_values_that_grow_or_shrink_along_the_sequence(bits, D, power):
    """By a factor of two every 16 or 64 tokens, one group the other way round: the exponents move block by block."""
    torch.manual_seed(int(power * 4) + bits)
    page, n = 16, 700
    P = -(-n // page)
    kp, vp = make_pool(P, H, page, D, bits), make_pool(P, H, page, D, bits)
    table = make_table([n, 333], page, P, 2 * P)
    kp, vp = (tuple(torch.cat([t, t]) for t in p) for p in (kp, vp))
    size = torch.ones(2 * P, device="cuda")
    for row in table:
        for i, e in enumerate(row):
            if e >= 0:
                size[e] = 2.0 ** round(power * (i - P // 2))
    for t in vp[1:]:
        for g in range(D // 64):
            t[..., g] = (t[..., g].float() * (size if g == 0 else 1.0 / size)[:, None, None]).to(BF16)
    q, out = run(kp, vp, table, [n, 333], bits, 2, 8, D)
    check(out, q, kp, vp, table, [n, 333], page, bits, D ** -0.5)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("part", [1, 2])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("group", [0, 1])
def test_a_group_that_is_not_finite_leaves_the_other_alone(bits, part, bad, group):
    """One token's scale or bias of one group: the dims of that group show it, in the heads that see it, and those of the other group do not."""
    torch.manual_seed(bits + group)
    page, lens = 32, [400, 70]
    kp, vp = make_pool(16, H, page, D, bits), make_pool(16, H, page, D, bits)
    table = make_table(lens, page, 13, 16)
    mine = slice(64 * group, 64 * group + 64)
    clean = tuple(t.clone() for t in vp)
    for t in clean[1:]:
        t[..., group] = 0.0                          # for the check: dims that are not looked at are zero
    vp[part][table[0][5], 1, 7, group] = bad
    q, out = run(kp, vp, table, lens, bits, 2, 8, D)
    assert not bool(torch.isfinite(out[0, 4:, :, mine]).any())
    assert bool(torch.isfinite(out[0, :4]).all()) and bool(torch.isfinite(out[1]).all())
    rest = out.clone()
    rest[..., mine] = 0.0
    check(rest, q, kp, clean, table, lens, page, bits, D ** -0.5)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("gqa", [1, 4, 8])
@pytest.mark.parametrize("at", [0, 17, 40])
def test_large_values_that_no_query_looks_at(bits, gqa, at):
    """A block of 64 tokens with values 2^26 times the others', and scores 40 below theirs: what it adds is nothing beside the rest.  So
    many queries of one sequence that a warp meets it among others."""
    torch.manual_seed(at)
    page, M, B = 64, 41, 200
    kp, vp = make_pool(M, H, page, D, bits), make_pool(M, H, page, D, bits)
    table = make_table([M * page], page, M, M)
    e = table[0][at]
    u = torch.randn(D, device="cuda")
    kp[0][e], kp[1][e], kp[2][e] = (x.expand(H, page, -1) for x in qb200.quantize((-40.0 * D ** 0.5 / float(u @ u) * u).to(BF16)[None], 64, bits))
    vp[1][e] *= 2.0 ** 26
    vp[2][e] *= 2.0 ** 26
    q = (u + 0.05 * torch.randn(B, H * gqa, 1, D, device="cuda")).to(BF16)
    out = qb200.kv_pages_decode_attention(q, kp, vp, ints(table), ints([M * page]), bits, 64, D ** -0.5, rows=ints([0] * B))
    some = [0, 1, 77, 130, 199]
    check(out[some], q[some], kp, vp, table, [M * page], page, bits, D ** -0.5, rows=[0] * len(some))
