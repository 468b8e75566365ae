"""GPU tests of the attention of drafted trees where its bounded waits run out: the status is set, what depends on such a wait is NaN, what does not is as ever,
and so is the next launch."""
import pytest
import torch

import qb200
from test_gpu_tree_attention import BF16, ints, make_pool, make_table, make_tree

pytestmark = pytest.mark.gpu
CODES = range(600, 615)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("D,H,gqa,T,page,wide,strided", [
    (128, 2, 4, 4, 16, False, False),       # 16 rows a tile; eight boxes a block
    (64, 2, 8, 4, 128, False, True),        # 32; scales read by the readers
    (128, 1, 8, 8, 64, False, False),       # 64
    (128, 2, 4, 32, 32, True, True),        # 128
])
def test_waits_that_run_out(bits, D, H, gqa, T, page, wide, strided):
    L = qb200.lib()
    torch.manual_seed(bits + T)
    lens = [3000, 40, 777, 129, T]
    P = sum(-(-n // page) for n in lens) + 2
    kp, vp = make_pool(P, H, page, D, bits), make_pool(P, H, page, D, bits)
    if strided and bits != 16:              # rows of scales a few elements apart
        def apart(t):
            room = torch.zeros(*t.shape[:-1], 5, dtype=t.dtype, device="cuda")
            room[..., 1:1 + t.shape[-1]] = t
            return room[..., 1:1 + t.shape[-1]]
        kp, vp = [(p[0], apart(p[1]), apart(p[2])) for p in (kp, vp)]
    table = make_table(lens, page, 160 * 1024 // page if wide else 3100 // page + 1, P)
    table[0][5] = -1
    trees = [make_tree(T, T, b) for b in range(len(lens))]
    # sequences behind one another, so that a block of the device has several pieces, and parts of tiles that are joined
    rows = [0, 1, 2, 3, 4] * 12
    q = torch.randn(len(rows), H * gqa, T, D, device="cuda").to(BF16)
    args = (q, kp, vp, ints(table), ints(lens), ints([trees[r] for r in rows]), bits, 64, 0.1)
    kw = dict(rows=ints(rows), window=600, sinks=3)
    good = qb200.kv_pages_tree_attention(*args, **kw)
    assert L.qb200_debug_tc_status() == 0 and not torch.isnan(good).any()
    try:
        for polls in (-1, 1, 2, 5, 40):
            y = torch.full_like(good, 7.0)
            L.qb200_debug_wait_polls(polls)
            qb200.kv_pages_tree_attention(*args, out=y, **kw)
            L.qb200_debug_wait_polls(0)
            status, done = L.qb200_debug_tc_status(), ~torch.isnan(y)
            assert status in CODES or (polls > 0 and status == 0)
            assert torch.equal(y[done], good[done])
            assert (status == 0) <= bool(done.all())
            assert polls > 0 or not bool(done.any())
            L.qb200_debug_tc_reset()
            assert torch.equal(qb200.kv_pages_tree_attention(*args, **kw), good)
            assert L.qb200_debug_tc_status() == 0
    finally:
        L.qb200_debug_wait_polls(0)
        L.qb200_debug_tc_reset()
