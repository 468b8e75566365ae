"""What the prompt attention's entry refuses, without a GPU."""
import ctypes as C

import pytest
import torch

import qb200 as q
from test_kv_pages import BF16, I32, NONE, ref, t


def attend(res=None, qq=None, k=None, v=None, scale=0.1, window=0, sinks=0, lens=NONE):
    qq = qq or t(BF16, [2, 4, 8, 128])
    k = k or t(BF16, [2, 2, 9, 128])
    return q.lib().qb200_window_attention(*ref(res or qq, qq, k, v or k), scale, window, sinks, *ref(lens), None)


@pytest.mark.parametrize("status,kw", [
    (1, dict(qq=t(q.FLOAT32, [2, 4, 8, 128]))), (1, dict(v=t(q.FLOAT16, [2, 2, 9, 128]))), (2, dict(qq=t(BF16, [2, 4, 128]))), (2, dict(res=t(BF16, [2, 4, 7, 128]))),
    (2, dict(v=t(BF16, [2, 2, 8, 128]))), (2, dict(qq=t(BF16, [2, 3, 8, 128]))), (2, dict(k=t(BF16, [1, 2, 9, 128]))), (2, dict(k=t(BF16, [2, 2, 9, 64]))),
    (1, dict(qq=t(BF16, [2, 4, 8, 96]), k=t(BF16, [2, 2, 9, 96]))), (5, dict(window=-1)), (5, dict(sinks=-2)), (1, dict(scale=0.0)), (1, dict(scale=-0.5)),
    (1, dict(scale=float("nan"))), (1, dict(scale=float("inf"))), (2, dict(k=t(BF16, [2, 2, 7, 128]))), (2, dict(lens=t(I32, [3]))), (4, dict(lens=t(q.INT64, [2]))),
    (2, dict(k=t(BF16, [2, 2, 0, 128]), lens=t(I32, [2]))), (1, dict(k=t(BF16, [2, 2, 9, 128], ptr=0x1008))), (1, dict(k=t(BF16, [2, 2, 9, 128], stride=[2400, 1200, 132, 1]))),
    (1, dict(k=t(BF16, [2, 2, 9, 128], stride=[0, 0, 0, 1]))), (3, dict(k=t(BF16, [2, 2, 9, 128], stride=[5000, 2500, 256, 2]))),
    (3, dict(res=t(BF16, [2, 4, 8, 128], stride=[0, 1024, 128, 1]))), (5, dict(k=t(BF16, [2, 2, 9, 128], ptr=None))), (1, dict(qq=t(BF16, [2, 4, 1 << 31, 128]), lens=t(I32, [2]))),
])
def test_refusals(status, kw):
    assert attend(**kw) == status, q.lib().qb200_last_error()


def test_nothing_to_do():
    assert attend(qq=t(BF16, [2, 4, 0, 128])) == 0 and attend(qq=t(BF16, [0, 4, 8, 128]), k=t(BF16, [0, 2, 9, 128])) == 0
    x = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="CUDA"):
        q.window_attention(x, x, x, 0.1)
