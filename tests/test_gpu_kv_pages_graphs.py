"""GPU tests of the paged calls as nodes of a graph behind other nodes than kernels: copies from the host, fills, and streams that join."""
import pytest
import torch

import qb200
from test_gpu_kv_pages import BF16, I32, ints, make_pool, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 16])
def test_a_tick_behind_copies_and_joined_streams(bits):
    """Tokens from pinned memory, keys made on one stream and values on another, the results read back: replayed with other inputs, against the
    same calls one by one."""
    torch.manual_seed(bits)
    page, H, D, M, N = 16, 2, 64, 8, 3
    host = torch.empty(N, H, 1, D, dtype=BF16).pin_memory()
    back = torch.empty(N, 4, 1, D, dtype=BF16).pin_memory()
    start = [t for p in (make_pool(N * M, H, page, D, bits), make_pool(N * M, H, page, D, bits)) for t in p]
    rows, ones = ints([2, 0, 1]), ints([1, 1, 1])
    q = torch.randn(N, 4, 1, D, device="cuda").to(BF16)

    class State:
        def __init__(self):
            pools = [None if t is None else t.clone() for t in start]
            self.k, self.v = tuple(pools[:3]), tuple(pools[3:])
            self.table, self.lens, self.refs = torch.full((N, M), -1, dtype=I32, device="cuda"), ints([0] * N), ints([0] * N * M)
            self.x, self.val = (torch.zeros(N, H, 1, D, dtype=BF16, device="cuda") for _ in range(2))
            self.out = torch.empty_like(q)
            self.ws = torch.empty(qb200.kv_pages_decode_attention_workspace_size(N, 4, H, D), dtype=torch.uint8, device="cuda")

        def tick(self, side=None):
            self.x.copy_(host, non_blocking=True)
            pos, copies = qb200.kv_pages_reserve(self.table, self.lens, self.refs, page, rows, ones)
            if side is not None:
                side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                self.val.copy_(self.x)
                self.val.mul_(-2.0)
            qb200.kv_pages_copy(tensors(self.k) + tensors(self.v), copies)
            if side is not None:
                torch.cuda.current_stream().wait_stream(side)
            qb200.kv_pages_append(self.k, self.v, self.x, self.val, self.table, pos, bits, 64, rows=rows)
            self.out.zero_()
            qb200.kv_pages_decode_attention(q, self.k, self.v, self.table, self.lens, bits, 64, 0.1, window=20, sinks=2, rows=rows, workspace=self.ws, out=self.out)
            back.copy_(self.out, non_blocking=True)
            alone = qb200.window_attention(self.x, self.x, self.val, 0.1)
            return alone

    one, two, spare = State(), State(), State()
    host.normal_()
    side, s = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        spare.tick(side)                        # (first calls set their kernels up)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            alone = two.tick(side)
    for step in range(40):
        host.copy_(torch.randn(N, H, 1, D))
        want = one.tick()
        torch.cuda.synchronize()
        expect = back.clone()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(back, expect) and torch.equal(one.out, two.out), step
        assert torch.equal(alone, want) and torch.equal(alone, two.val), step
        for a, b in zip([one.table, one.lens, one.refs] + tensors(one.k) + tensors(one.v), [two.table, two.lens, two.refs] + tensors(two.k) + tensors(two.v)):
            assert torch.equal(a.view(torch.int16) if a.dtype == BF16 else a, b.view(torch.int16) if b.dtype == BF16 else b), step
    assert one.lens.tolist() == [40, 40, 40] and qb200.lib().qb200_debug_tc_status() == 0
