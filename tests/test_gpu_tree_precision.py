"""GPU tests of how near the attention of drafted trees comes to 64 bits: its errors stay under the result's own rounding, over pages of every kind."""
import math

import pytest
import torch

import qb200
from drafted_ref import F64, attention, dequantized, visible
from test_gpu_tree_attention import BF16, ints, make_pool, make_table, make_tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("D,gqa,T,wide", [(64, 1, 1, False), (64, 2, 16, False), (64, 4, 16, False), (64, 4, 32, True), (128, 1, 9, False), (128, 2, 13, False), (128, 5, 13, False),
                                          (128, 4, 32, True)])
@pytest.mark.parametrize("half", [2.0 ** -8, 2.0 ** -11])
def test_probabilities_that_round_one_way(bits, D, gqa, T, wide, half):
    """All tokens but every 128th have one score, whose probability, beside the others' power of two, lies just under the middle of two numbers of 8 (or 11)
    bits: rounded to those, all of them lose up to 2^-8 (2^-11) of themselves and the normaliser nothing.  Values of 1 show that: the result is 1, rounded to
    bf16 from within 2^-10 of it (the next numbers are 1 - 2^-8 and 1 + 2^-7, so half-way is 2^-9)."""
    page, n = 32, 1000 + T
    P = -(-n // page)
    M = 160 * 1024 // page if wide else P
    k = torch.zeros(P, 1, page, D, device="cuda")
    table = make_table([n], page, M, P)
    for i in range(0, n, 128):                                 # (one in front of every part that the kernel may make of the sequence)
        k[table[0][i // page], 0, i % page, 0] = 1.0
    v = torch.ones(P, 1, page, D, device="cuda")
    kp, vp = [(x.to(BF16), None, None) if bits == 16 else qb200.quantize(x.to(BF16), 64, bits) for x in (k, v)]
    q = torch.zeros(1, gqa, T, D, device="cuda", dtype=BF16)
    q[..., 0] = 1.0
    key = dequantized(kp, bits)[table[0][0], 0, :2, 0]
    gap = float(key[0] - key[1])                               # (the codes' own difference)
    scale = (3.0 - math.log2(1.0 + half - 2.0 ** -14)) * math.log(2.0) / gap
    trees = [[t - 1 for t in range(T)]]
    out = qb200.kv_pages_tree_attention(q, kp, vp, ints(table), ints([n]), ints(trees), bits, 64, scale)
    assert torch.equal(out, torch.ones_like(out) * dequantized(vp, bits)[0, 0, 0, 0].to(BF16)), float((out.float() - 1).abs().max())


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("D,gqa,T,wide", [(64, 2, 8, False), (64, 8, 8, False), (64, 8, 16, True), (128, 4, 4, False), (128, 4, 8, False), (128, 4, 16, False), (128, 4, 32, True)])
def test_errors_beside_the_rounding_of_the_result(bits, D, gqa, T, wide):
    """Root mean square over a call, against that of rounding the 64-bit results to bf16.  At 16 bits probabilities keep 16 bits, 2^-17: nothing beside it.  At 4 and 8
    bits three roundings to fp16 come on top, of keys, values and probabilities: evenly spread within 2^-11 of a number, of mean square 2^-22 / 3 and less; a
    value's or probability's weighs p v of a sum of such terms, a key's moves its score by scale sqrt(sum q^2 k^2), 1 here, times that: each adds at most
    2^-22 / 3 of the result's square.  2 % for the sample and the sums."""
    torch.manual_seed(D + T + bits)
    page, lens, H = 64, [900, 333, 80], 2
    P = sum(-(-n // page) for n in lens) + 1
    kp, vp = make_pool(P, H, page, D, bits), make_pool(P, H, page, D, bits)
    table = make_table(lens, page, 160 * 1024 // page if wide else 15, P)
    trees = [make_tree(T, T, b) for b in range(len(lens))]
    q = torch.randn(len(lens), H * gqa, T, D, device="cuda").to(BF16)
    out = qb200.kv_pages_tree_attention(q, kp, vp, ints(table), ints(lens), ints(trees), bits, 64, D ** -0.5).to(F64)
    k, v = dequantized(kp, bits), dequantized(vp, bits)
    want = torch.zeros_like(out)
    for b, n in enumerate(lens):
        for t in range(T):
            at = torch.tensor([j for j, _ in visible(trees[b], t, T, n, 0, 0)], device="cuda")
            pid = torch.tensor(table[b], device="cuda")[at // page]
            for h in range(H):
                want[b, h * gqa:(h + 1) * gqa, t] = attention(q[b, h * gqa:(h + 1) * gqa, t].to(F64), k[pid, h, at % page], v[pid, h, at % page], D ** -0.5)[0]
    rel = lambda x: float((x - want).norm() / want.norm())
    mine, rounding = rel(out), rel(want.to(BF16).to(F64))
    assert mine <= 1.02 * math.sqrt(rounding ** 2 + (0.0 if bits == 16 else 2.0 ** -22)), (mine, rounding)
