"""GPU tests of the attention of drafted trees where the tables are wide, so that a tile has up to 128 query rows, against fp64."""
import pytest
import torch

import qb200
from test_gpu_tree_attention import BF16, check, ints, make_pool, make_table, make_tree

pytestmark = pytest.mark.gpu


def wide(bits, D, H, gqa, page, lens, counts, T, window=0, sinks=0, seed=0):
    torch.manual_seed(seed + 11)
    M = 160 * 1024 // page                       # (room for many more tokens than there are)
    P = sum(-(-n // page) for n in lens) + 3
    kp, vp = make_pool(P, H, page, D, bits), make_pool(P, H, page, D, bits)
    table = make_table(lens, page, M, P, seed)
    trees = [make_tree(n, T, seed + b) for b, n in enumerate(counts)]
    q = (torch.randn(len(lens), H * gqa, T, D, device="cuda")).to(BF16)
    scale = D ** -0.5
    out = qb200.kv_pages_tree_attention(q, kp, vp, ints(table), ints(lens), ints(trees), bits, 64, scale, window=window, sinks=sinks, counts=ints(counts))
    check(out, q, kp, vp, table, lens, trees, counts, page, bits, scale, window, sinks)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("D,H,gqa,page,lens,counts,T", [
    (128, 2, 4, 32, [200, 1, 130, 0, 700], [20, 1, 17, 0, 20], 20),          # one tile, 80 rows
    (64, 3, 5, 16, [513, 128, 129, 40], [27, 27, 13, 26], 27),              # 135 rows: a tile and a few rows
    (128, 1, 8, 64, [1500, 64, 63], [64, 64, 33], 64),                      # four tiles
    (64, 1, 3, 128, [64, 640], [64, 43], 64),                               # 192 rows
    (128, 1, 2, 256, [2300, 5, 257], [40, 4, 64], 64),                      # exactly 128
])
def test_wide_tables(bits, D, H, gqa, page, lens, counts, T):
    wide(bits, D, H, gqa, page, lens, counts, T)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (64, 5), (130, 130), (1000, 0)])
def test_wide_tables_with_windows(bits, window, sinks):
    wide(bits, 128, 2, 4, 32, [900, 300, 33], [24, 32, 24], 32, window, sinks, seed=3)


@pytest.mark.parametrize("bits", [4, 16])
def test_one_call_by_both_widths(bits):
    """The same call by a narrow and a wide table: each within the bounds of the 64-bit result."""
    torch.manual_seed(5)
    lens, counts, T, page, D = [1000, 260], [32, 20], 32, 32, 128
    P = sum(-(-n // page) for n in lens) + 2
    kp, vp = make_pool(P, 2, page, D, bits), make_pool(P, 2, page, D, bits)
    q = torch.randn(2, 8, T, D, device="cuda").to(BF16)
    trees = [make_tree(n, T, b) for b, n in enumerate(counts)]
    for M in (32, 8000):
        table = make_table(lens, page, M, P)
        o = qb200.kv_pages_tree_attention(q, kp, vp, ints(table), ints(lens), ints(trees), bits, 64, 0.1, counts=ints(counts))
        check(o, q, kp, vp, table, lens, trees, counts, page, bits, 0.1)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("T,gqa", [(16, 7), (8, 7), (4, 7), (4, 4)])
def test_units_and_pages_of_long_ragged_batches_do_not_mix(bits, page, T, gqa):
    """Tokens of very different sizes over many blocks, pages missing here and there: every run gives the same, and the right rows."""
    torch.manual_seed(9)
    H, D, B = 2, 128, 9
    lens = [2500 - 217 * b for b in range(B)]
    counts = [max(1, T - b) for b in range(B)]
    P = sum(-(-n // page) for n in lens) + 3
    pools = []
    for _ in range(2):
        x = torch.randn(P, H, page, D, device="cuda") * torch.exp2(torch.randint(-3, 4, (P, H, page, 1), device="cuda").float())
        pools.append((x.to(BF16), None, None) if bits == 16 else qb200.quantize(x.to(BF16), 64, bits))
    M = 160 * 1024 // page
    table = make_table(lens, page, M, P)
    for b in range(B):
        table[b][3 * b + 1] = -1
    trees = [make_tree(n, T, b) for b, n in enumerate(counts)]
    q = torch.randn(B, H * gqa, T, D, device="cuda").to(BF16)
    args = (q, *pools, ints(table), ints(lens), ints(trees), bits, 64, 0.02)
    out = qb200.kv_pages_tree_attention(*args, counts=ints(counts))
    check(out, q, *pools, table, lens, trees, counts, page, bits, 0.02)
    for _ in range(20):
        assert torch.equal(out, qb200.kv_pages_tree_attention(*args, counts=ints(counts)))
