"""GPU tests of the operators on drafted tokens with calls in flight on several streams, and in graphs that are replayed at once: each as by itself."""
import pytest
import torch

import qb200
from test_gpu_tree_attention import BF16, ints, make_pool, make_table, make_tree

pytestmark = pytest.mark.gpu
I32 = torch.int32


def tree_calls():
    torch.manual_seed(21)
    calls = []
    for i, (bits, D, gqa, T) in enumerate([(4, 128, 4, 8), (16, 64, 8, 8), (8, 128, 4, 32), (16, 128, 4, 32)]):
        page, lens = 64, [3000, 700, 129, 50]
        P = sum(-(-n // page) for n in lens) + 1
        kp, vp = make_pool(P, 2, page, D, bits), make_pool(P, 2, page, D, bits)
        q = torch.randn(4, 2 * gqa, T, D, device="cuda").to(BF16)
        args = (q, kp, vp, ints(make_table(lens, page, 2560, P)), ints(lens), ints([make_tree(T, T, i + b) for b in range(4)]), bits, 64, 0.09)
        ws = torch.empty(qb200.kv_pages_tree_attention_workspace_size(4, 2 * gqa, 2, T, D), dtype=torch.uint8, device="cuda")
        out = torch.empty_like(q)
        calls.append((lambda a=args, w=ws, o=out: qb200.kv_pages_tree_attention(*a, workspace=w, out=o), out))
    return calls


def sample_calls():
    g = torch.Generator(device="cuda").manual_seed(22)
    calls = []
    for N, V, dtype, k, p in ((3, 128256, torch.bfloat16, 50, 0.9), (40, 32001, torch.float32, 0, 0.997), (150, 20000, torch.float16, 0, 1.0), (1, 262144, torch.float32, 0, 1.0)):
        x = (torch.randn(N, V, device="cuda", generator=g) * 3).to(dtype)
        u, t = torch.rand(N, device="cuda", generator=g), torch.full((N,), 0.8, device="cuda")
        kk, pp = torch.full((N,), k, dtype=I32, device="cuda"), torch.full((N,), p, device="cuda")
        out = torch.empty(N, dtype=I32, device="cuda")
        calls.append((lambda a=(x, u, t, kk, pp), o=out: o.copy_(qb200.sample(*a)), out))
    return calls


@pytest.mark.parametrize("calls", [tree_calls, sample_calls])
def test_calls_on_streams_and_graphs_at_once(calls):
    calls = calls()
    want = []
    for call, out in calls:
        call()
        want.append(out.clone())
    graphs = []
    for call, out in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call()
            call()
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for runs in ([c for c, _ in calls], [g.replay for g in graphs]):
        for _ in range(10):
            for (_, out), run, st in zip(calls, runs, streams):
                with torch.cuda.stream(st):
                    out.fill_(0)
                    run()
                    run()
        torch.cuda.synchronize()
        for (_, out), w in zip(calls, want):
            assert torch.equal(out, w)
    assert qb200.lib().qb200_debug_tc_status() == 0
