"""A CUDA error that one entry reports does not come back from the next one."""
import ctypes as C

import pytest
import torch

import qb200

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("entry", ["pages", "rms_norm"])
def test_a_failed_launch_is_reported_once(entry):
    """The launch that fails: into the legacy stream while a stream that synchronises with it is being captured, which CUDA answers with
    an error on the host.  Capture by the driver's entries, which keep no last error of their own."""
    cu = C.CDLL("libcuda.so.1")
    table, lens, refs, rows = ints([[-1, -1]]), ints([0]), ints([0, 0]), ints([0])
    x, w = torch.randn(4, 128, device="cuda").to(torch.bfloat16), torch.ones(128, device="cuda").to(torch.bfloat16)
    y = torch.empty_like(x)
    d = [qb200.desc(t) for t in (table, lens, refs, rows, y, x, w)]
    t, l, f, r, dy, dx, dw = (C.byref(e) for e in d)
    none = C.byref(qb200.desc(None))
    L = qb200.lib()
    call = (lambda: L.qb200_kv_pages_free(t, l, f, 16, r, none, none, None)) if entry == "pages" else (lambda: L.qb200_rms_norm(dy, dx, dw, 1e-5, None))
    want = qb200.quantize(x, 64, 4)
    torch.cuda.synchronize()
    s, graph = C.c_void_p(), C.c_void_p()
    assert cu.cuStreamCreate(C.byref(s), 0) == 0 and cu.cuStreamBeginCapture_v2(s, 2) == 0
    try:
        status = call()
    finally:
        cu.cuStreamEndCapture(s, C.byref(graph))
        cu.cuStreamDestroy_v2(s)
    assert status == 6
    got = qb200.quantize(x, 64, 4)               # (its launcher asks for the last error)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert call() == 0
    torch.cuda.synchronize()
