"""GPU tests of the attention of drafted trees over pages, against fp64 on the values that the codes stand for (tolerance: drafted_ref.py)."""
import random

import pytest
import torch

import qb200
from drafted_ref import F64, attention, dequantized, tolerance, visible

pytestmark = pytest.mark.gpu
I32, BF16 = torch.int32, torch.bfloat16


def ints(x):
    return torch.tensor(x, dtype=I32, device="cuda")


def make_pool(P, H, page, D, bits, std=1.0):
    x = (torch.randn(P, H, page, D, device="cuda") * std).to(BF16)
    return (x, None, None) if bits == 16 else qb200.quantize(x, 64, bits)


def make_table(lens, page, M, P, seed=0):
    perm = list(range(P))
    random.Random(seed).shuffle(perm)
    return [[perm.pop() if p * page < n else -1 for p in range(M)] for n in lens]


def make_tree(n, T, seed, kind="mixed"):
    rng = random.Random(seed)
    t = []
    for i in range(n):
        t.append({"chain": i - 1, "star": 0 if i else -1, "roots": -1}.get(kind, -1 if i == 0 or rng.random() < 0.05 else rng.randrange(max(0, i - 5), i)))
    return t + [rng.choice([-1, 0, 63, 7]) for _ in range(T - n)]           # (what stands behind the count does not matter)


def check(out, q, kp, vp, table, lens, trees, counts, page, bits, scale, window=0, sinks=0, rows=None, poisoned=None):
    B, Hq, T, D = q.shape
    k, v = dequantized(kp, bits), dequantized(vp, bits)
    rep = Hq // k.shape[1]
    worst = 0.0
    for b in range(B):
        r = b if rows is None else rows[b]
        length = max(0, min(lens[r], len(table[r]) * page)) if 0 <= r < len(table) else 0
        n = max(0, min(counts[b], T, length))
        assert (out[b, :, n:] == 0).all(), f"b {b}: rows behind the nodes"
        for t in range(n):
            places = [j for j, _ in visible(trees[b], t, n, length, window, sinks) if 0 <= table[r][j // page] < k.shape[0]]
            at = torch.tensor(places, device="cuda", dtype=torch.long)
            pid = torch.tensor([table[r][j // page] for j in places], device="cuda", dtype=torch.long)
            for h in range(k.shape[1]):
                got = out[b, h * rep:(h + 1) * rep, t].to(F64)
                if poisoned is not None and poisoned(b, t, places):
                    assert not torch.isfinite(got).all(-1).any(), f"b {b} node {t}: sees what is not finite"
                    continue
                o, A, S = attention(q[b, h * rep:(h + 1) * rep, t].to(F64), k[pid, h, at % page], v[pid, h, at % page], scale)
                tol = tolerance(o, A, S, bits, v[pid, h, at % page])
                err = (got - o).abs()
                assert not torch.isnan(got).any(), f"b {b} node {t} head {h}: NaN"
                worst = max(worst, float((err / tol).max()))
                assert (err <= tol).all(), f"b {b} node {t} head {h}: {float((err / tol).max()):.2f} of the tolerance"
    return worst


def case(bits, D, H, gqa, page, lens, counts, T, kind="mixed", window=0, sinks=0, seed=0, **kw):
    torch.manual_seed(seed + 1)
    M = max(1, max(-(-n // page) for n in lens)) + 1
    P = sum(-(-n // page) for n in lens) + 3
    kp, vp = make_pool(P, H, page, D, bits), make_pool(P, H, page, D, bits)
    table = make_table(lens, page, M, P, seed)
    q = torch.randn(len(lens), H * gqa, T, D, device="cuda").to(BF16)
    trees = [make_tree(max(0, min(c, T)), T, seed + i, kind) for i, c in enumerate(counts)]
    out = qb200.kv_pages_tree_attention(q, kp, vp, ints(table), ints(lens), ints(trees), bits, 64, D ** -0.5, window=window, sinks=sinks, counts=ints(counts), **kw)
    check(out, q, kp, vp, table, lens, trees, counts, page, bits, D ** -0.5, window, sinks)
    return out


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("D,H,gqa,page,lens,counts,T", [
    (128, 2, 4, 64, [9, 70, 200], [4, 8, 7], 8), (64, 1, 1, 16, [17, 1, 130], [1, 1, 1], 1), (128, 4, 7, 32, [300, 40], [16, 11], 16),
    (64, 8, 8, 128, [129, 64], [64, 64], 64), (128, 1, 11, 16, [77], [27], 27), (64, 2, 16, 256, [700, 3], [3, 3], 3), (128, 8, 4, 64, [640], [32], 33)])
def test_lengths_heads_and_trees(bits, D, H, gqa, page, lens, counts, T):
    case(bits, D, H, gqa, page, lens, counts, T, seed=bits)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("kind", ["chain", "star", "roots", "mixed"])
@pytest.mark.parametrize("D", [64, 128])
def test_shapes_of_trees(bits, kind, D):
    case(bits, D, 2, 4, 32, [250, 64, 128, 129], [40, 64, 33, 1], 64, kind, seed=3)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 1), (64, 0), (128, 4), (130, 40), (200, 300), (1000, 0)])
def test_windows_and_sinks(bits, window, sinks):
    case(bits, 128, 2, 3, 16, [513, 130, 20, 300], [20, 12, 20, 1], 20, window=window, sinks=sinks, seed=5)
    case(bits, 64, 1, 8, 64, [700], [24], 24, "chain", window=window, sinks=sinks, seed=6)


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_counts_and_lengths_at_their_ends(bits):
    # no tokens, fewer tokens than nodes, no nodes, more nodes than there is room for, a length beyond the table
    case(bits, 128, 1, 4, 16, [0, 3, 50, 20, 16], [4, 8, 0, 99, -3], 8, seed=7)
    case(bits, 64, 2, 2, 16, [8, 8], [8, 8], 8, "chain", seed=8)


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_long_contexts_share_their_sums(bits):
    case(bits, 128, 2, 4, 64, [9000, 4097, 129], [12, 9, 12], 12, seed=9)
    case(bits, 64, 1, 4, 128, [20000], [6], 6, seed=10)


def test_many_sequences():
    lens = [(7 * i) % 150 + 1 for i in range(200)]
    case(4, 128, 1, 2, 16, lens, [min(n, 1 + i % 6) for i, n in enumerate(lens)], 6, seed=11)


def test_every_size_of_query_tiles():
    for T in (1, 2, 4, 5, 8, 9, 16, 17, 32, 33, 48, 64):
        case(16, 64, 1, 5, 32, [150, 90], [T, min(T, 40)], T, seed=T)


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_rows_missing_pages_and_wrong_page_numbers(bits):
    torch.manual_seed(2)
    page, D, lens = 16, 128, [100, 260, 40]
    kp, vp = make_pool(40, 2, page, D, bits), make_pool(40, 2, page, D, bits)
    table = make_table(lens, page, 18, 40)
    table[0][2], table[1][4], table[1][0] = -1, 10 ** 6, -77
    rows, counts = [2, -1, 1, 0, 5], [5, 5, 9, 9, 9]
    q = torch.randn(5, 4, 9, D, device="cuda").to(BF16)
    trees = [make_tree(c, 9, i) for i, c in enumerate(counts)]
    out = qb200.kv_pages_tree_attention(q, kp, vp, ints(table), ints(lens), ints(trees), bits, 64, 0.1, rows=ints(rows), counts=ints(counts))
    check(out, q, kp, vp, table, lens, trees, counts, page, bits, 0.1, rows=rows)


def test_default_counts_and_parents_that_do_not_come_before():
    torch.manual_seed(3)
    kp, vp = make_pool(8, 1, 32, 64, 16), make_pool(8, 1, 32, 64, 16)
    table, lens = make_table([70], 32, 3, 8), [70]
    trees = [[5, 0, 2, 1, -9, 100, 3, 2 ** 31 - 1]]
    q = torch.randn(1, 2, 8, 64, device="cuda").to(BF16)
    out = qb200.kv_pages_tree_attention(q, kp, vp, ints(table), ints(lens), ints(trees), 16, 64, 0.125)
    check(out, q, kp, vp, table, lens, trees, [8], 32, 16, 0.125)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_scales(bits, scale):
    torch.manual_seed(4)
    lens, page = [300, 77], 32
    kp, vp = make_pool(20, 2, page, 128, bits), make_pool(20, 2, page, 128, bits)
    table = make_table(lens, page, 10, 20)
    q = torch.randn(2, 6, 10, 128, device="cuda").to(BF16)
    trees = [make_tree(10, 10, i) for i in range(2)]
    out = qb200.kv_pages_tree_attention(q, kp, vp, ints(table), ints(lens), ints(trees), bits, 64, scale)
    check(out, q, kp, vp, table, lens, trees, [10, 10], page, bits, scale)


@pytest.mark.parametrize("bits", [4, 16])
def test_scores_that_rise_and_fall(bits):
    """Rows whose largest score comes last, first, or far above all others: the running reference has to move."""
    torch.manual_seed(5)
    page, T, D = 64, 6, 128
    n = 2000
    x = torch.randn(n + 64, 1, D, device="cuda")
    ramp = torch.linspace(0, 40, n + 64, device="cuda")
    q = torch.randn(3, 2, T, D, device="cuda")
    d = torch.nn.functional.normalize(torch.randn(D, device="cuda"), dim=0)
    q = (q + 4 * d).to(BF16)
    outs = []
    for b, r in enumerate([ramp, ramp.flip(0), torch.where(torch.arange(n + 64, device="cuda") == 777, 60.0, 0.0)]):
        rows = (x[:, 0] * 0.3 + r[:, None] * d * 2.0).to(BF16)
        P = (n + 63) // page
        pool = rows[: P * page].reshape(P, 1, page, D).contiguous()
        kp = (pool, None, None) if bits == 16 else qb200.quantize(pool, 64, bits)
        vp = make_pool(P, 1, page, D, bits)
        table, trees = [list(range(P))], [make_tree(T, T, b)]
        out = qb200.kv_pages_tree_attention(q[b:b + 1], kp, vp, ints(table), ints([n]), ints(trees), bits, 64, D ** -0.5)
        check(out, q[b:b + 1], kp, vp, table, [n], trees, [T], page, bits, D ** -0.5)
        outs.append(out)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_finite_in_masked_places(bits, what):
    """Rows behind the end, behind the window and of nodes on other lines may hold anything; who sees them gives what is not finite."""
    torch.manual_seed(6)
    page, D, n, T = 16, 128, 300, 8
    lens, counts = [n], [T]
    kp, vp = make_pool(25, 1, page, D, bits), make_pool(25, 1, page, D, bits)
    table = make_table(lens, page, 21, 25)
    trees = [[-1, 0, 0, 1, 2, 3, 4, 6]]           # two lines: 1 3 5 and 2 4 6 7
    window = 100
    bad = [n - T + 2, 50]                          # node 2; a cached token that no query sees
    for pool in (kp, vp):
        for j in bad:
            (pool[0] if bits == 16 else pool[1])[table[0][j // page], :, j % page] = what
        last = table[0][(n - 1) // page]
        (pool[0] if bits == 16 else pool[2])[last, :, n % page:] = what
    q = torch.randn(1, 4, T, D, device="cuda").to(BF16)
    out = qb200.kv_pages_tree_attention(q, kp, vp, ints(table), ints(lens), ints(trees), bits, 64, 0.1, window=window, sinks=2)
    check(out, q, kp, vp, table, lens, trees, counts, page, bits, 0.1, window, 2, poisoned=lambda b, t, places: bad[0] in places)


def test_only_values_not_finite_at_the_edge_of_a_window():
    """A cached token that some nodes see and deeper ones no longer do, with values that are not finite."""
    torch.manual_seed(7)
    page, D, n, T, bits = 32, 64, 200, 6, 16
    lens, trees, window = [n], [[-1, 0, 1, 2, 3, 4]], 64
    kp, vp = make_pool(9, 1, page, D, bits), make_pool(9, 1, page, D, bits)
    table = make_table(lens, page, 8, 9)
    edge = n - T - window + 3                      # seen from depth 2 down, not from 3 on
    vp[0][table[0][edge // page], :, edge % page, 5] = float("nan")
    q = torch.randn(1, 4, T, D, device="cuda").to(BF16)
    out = qb200.kv_pages_tree_attention(q, kp, vp, ints(table), ints(lens), ints(trees), bits, 64, 0.125, window=window)
    check(out, q, kp, vp, table, lens, trees, [T], page, bits, 0.125, window, poisoned=lambda b, t, places: edge in places)


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_one_scale_group_far_above_the_other(bits):
    torch.manual_seed(8)
    page, D, lens, T = 32, 128, [400], 6
    x = torch.randn(14, 2, page, D, device="cuda")
    x[..., 64:] *= 1e6
    pool = x.to(BF16)
    vp = (pool, None, None) if bits == 16 else qb200.quantize(pool, 64, bits)
    kp = make_pool(14, 2, page, D, bits)
    table, trees = make_table(lens, page, 13, 14), [make_tree(T, T, 0)]
    q = torch.randn(1, 8, T, D, device="cuda").to(BF16)
    out = qb200.kv_pages_tree_attention(q, kp, vp, ints(table), ints(lens), ints(trees), bits, 64, D ** -0.5)
    check(out, q, kp, vp, table, lens, trees, [T], page, bits, D ** -0.5)


def test_strided_queries_results_lists_and_pools():
    torch.manual_seed(9)
    page, D, H, B, T, bits = 16, 128, 2, 2, 7, 8
    lens = [120, 65]
    whole = qb200.quantize(torch.randn(2, 15, H, page, D, device="cuda").to(BF16), 64, bits)
    kp, vp = tuple(t[0] for t in whole), tuple(t[1] for t in whole)
    table = make_table(lens, page, 9, 15)
    trees = [make_tree(T, T, i) for i in range(B)]
    wide = torch.randn(B, T, H * 3, D + 3, device="cuda").to(BF16)
    q = wide.transpose(1, 2)[..., 3:]                                          # rows off 16 bytes, nodes before heads
    par = torch.full((B, T + 4), 9, dtype=I32, device="cuda")
    par[:, 2:-2] = ints(trees)
    tab = torch.full((B, 12), -5, dtype=I32, device="cuda")
    tab[:, 1:10] = ints(table)
    res = torch.full((B, T, H * 3, D + 8), 7.0, dtype=BF16, device="cuda")
    out = res[..., 1:D + 1].transpose(1, 2)
    qb200.kv_pages_tree_attention(q, kp, vp, tab[:, 1:10], ints(lens), par[:, 2:-2], bits, 64, 0.09, out=out)
    check(out, q, kp, vp, table, lens, trees, [T, T], page, bits, 0.09)
    assert (res[..., 0] == 7).all() and (res[..., D + 1:] == 7).all()
    # heads in front of pages, scales on rows of their own
    order = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in kp]
    pad = torch.zeros(*kp[1].shape[:-1], 5, dtype=BF16, device="cuda")
    for i in (1, 2):
        p = pad.clone()
        p[..., 1:3] = order[i]
        order[i] = p[..., 1:3]
    qc = q.contiguous()
    a = qb200.kv_pages_tree_attention(qc, tuple(order), vp, ints(table), ints(lens), ints(trees), bits, 64, 0.09)
    check(a, qc, kp, vp, table, lens, trees, [T, T], page, bits, 0.09)


def test_a_tree_of_one_is_the_next_token():
    """Within both tolerances: the decode attention of the same cache."""
    torch.manual_seed(10)
    page, D, lens = 64, 128, [500, 90, 64]
    for bits in (4, 8, 16):
        kp, vp = make_pool(14, 2, page, D, bits), make_pool(14, 2, page, D, bits)
        table = make_table(lens, page, 9, 14)
        q = torch.randn(3, 8, 1, D, device="cuda").to(BF16)
        a = qb200.kv_pages_tree_attention(q, kp, vp, ints(table), ints(lens), ints([[-1]] * 3), bits, 64, D ** -0.5)
        b = qb200.kv_pages_decode_attention(q, kp, vp, ints(table), ints(lens), bits, 64, D ** -0.5)
        rel = float((a.double() - b.double()).norm() / b.double().norm())
        assert rel < 1e-2, rel


def test_no_allocation_other_streams_graphs_and_one_workspace():
    torch.manual_seed(11)
    page, D, bits, T = 32, 128, 4, 9
    lens = [3000, 700]
    kp, vp = make_pool(120, 4, page, D, bits), make_pool(120, 4, page, D, bits)
    table, trees = make_table(lens, page, 96, 120), [make_tree(T, T, i) for i in range(2)]
    dt, dl, dp = ints(table), ints(lens), ints(trees)
    q = torch.randn(2, 16, T, D, device="cuda").to(BF16)
    want = qb200.kv_pages_tree_attention(q, kp, vp, dt, dl, dp, bits, 64, 0.09)
    check(want, q, kp, vp, table, lens, trees, [T, T], page, bits, 0.09)
    n = qb200.kv_pages_tree_attention_workspace_size(2, 16, 4, T, D)
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        qb200.kv_pages_tree_attention(q, kp, vp, dt, dl, dp, bits, 64, 0.09, workspace=ws, out=out)
    side.synchronize()
    assert torch.equal(out, want)
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    qb200.kv_pages_tree_attention(q, kp, vp, dt, dl, dp, bits, 64, 0.09, workspace=ws, out=out)
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qb200.kv_pages_tree_attention(q, kp, vp, dt, dl, dp, bits, 64, 0.09, workspace=ws, out=out)
        qb200.kv_pages_tree_attention(q, kp, vp, dt, dl, dp, bits, 64, 0.09, workspace=ws, out=out)
    # other lengths, trees and queries at replay
    q2 = torch.randn_like(q)
    lens2, trees2 = [1500, 33], [make_tree(T, T, 7 + i, "chain") for i in range(2)]
    for dst, src in ((q, q2), (dl, ints(lens2)), (dp, ints(trees2))):
        dst.copy_(src)
    ws.fill_(255)
    out.fill_(3)
    graph.replay()
    torch.cuda.synchronize()
    check(out, q2, kp, vp, table, lens2, trees2, [T, T], page, bits, 0.09)


def test_positions_beyond_32_bit_offsets():
    """Pages far into a pool of more than 2^32 bytes, and heads far apart in it."""
    torch.manual_seed(12)
    P, H, page, D = 34000, 2, 256, 128           # 4.4 GB of bf16 rows each
    lens, T = [600], 5
    kp, vp = (torch.zeros(P, H, page, D, dtype=BF16, device="cuda"), None, None), (torch.zeros(P, H, page, D, dtype=BF16, device="cuda"), None, None)
    pages = [P - 1, P - 7, 3, 0]
    for pool in (kp, vp):
        for p in pages:
            pool[0][p] = torch.randn(H, page, D, device="cuda").to(BF16)
    q = torch.randn(1, 4, T, D, device="cuda").to(BF16)
    trees = [make_tree(T, T, 0)]
    out = qb200.kv_pages_tree_attention(q, kp, vp, ints([pages]), ints(lens), ints(trees), 16, 64, 0.09)
    small_k, small_v = [(p[0][pages].contiguous(), None, None) for p in (kp, vp)]
    check(out, q, small_k, small_v, [[0, 1, 2, 3]], lens, trees, [T], page, 16, 0.09)


def test_results_do_not_depend_on_the_run():
    torch.manual_seed(13)
    page, D, bits, T, lens = 64, 128, 8, 16, [5000, 64, 900]
    kp, vp = make_pool(100, 2, page, D, bits), make_pool(100, 2, page, D, bits)
    table, trees = make_table(lens, page, 80, 100), [make_tree(T, T, i) for i in range(3)]
    q = torch.randn(3, 8, T, D, device="cuda").to(BF16)
    args = (q, kp, vp, ints(table), ints(lens), ints(trees), bits, 64, 0.09)
    first = qb200.kv_pages_tree_attention(*args)
    for _ in range(5):
        assert torch.equal(qb200.kv_pages_tree_attention(*args), first)
