"""How many rows of test_gpu_sample.py lie on a border, where the weights' rounding decides and the token is not looked at: next to none.  Those rows' log-probabilities
are of the token that came out."""
import inspect

import pytest
import torch

import qb200
import test_gpu_sample as rows
from sample_rows import logprob

pytestmark = pytest.mark.gpu
# Rows whose borders fall among equal logits by construction (a random number or a share that is a ratio of small whole numbers meets a sum of equal weights)
TIES = {"test_equal_logits_go_by_index": 0.1}


def cases():
    names = ["test_sizes_and_settings", "test_large_vocabularies", "test_every_setting_by_itself_and_together", "test_equal_logits_go_by_index",
             "test_masks_and_what_is_not_finite"]
    for name in names:
        takes = inspect.signature(getattr(rows, name)).parameters
        for V in ([7, 255, 4097, 16001, 50001] if "V" in takes else [None]):
            for dtype in (rows.DTYPES if "dtype" in takes else [None]):
                yield name, {k: v for k, v in dict(V=V, dtype=dtype).items() if v is not None}


@pytest.mark.parametrize("name,kw", list(cases()))
def test_rows_that_lie_on_a_border(name, kw, monkeypatch):
    seen, sampled = [], []
    plain, sample = rows.plain, qb200.sample

    def counted(x, *a):
        token, margin = plain(x, *a)
        seen.append((len(x), margin, x))
        return token, margin

    def kept(*a, **k):
        out = sample(*a, **k)
        if k.get("want_logprobs"):
            sampled.extend(zip(out[0].tolist(), out[1].tolist()))
        return out

    monkeypatch.setattr(rows, "plain", counted)
    monkeypatch.setattr(qb200, "sample", kept)
    getattr(rows, name)(**kw)
    assert len(seen) == len(sampled) > 0
    on = [i for i, (V, margin, _) in enumerate(seen) if margin <= V * 2.0 ** -44]
    assert len(on) <= TIES.get(name, 0.0) * len(seen), f"{len(on)} of {len(seen)} rows"
    for i in on:
        V, _, x = seen[i]
        token, lp = sampled[i]
        y = logprob(torch.tensor(x, dtype=torch.float64).numpy(), token)
        assert abs(lp - y) <= 2.0 ** -22 * abs(y) + V * 2.0 ** -44 + 2.0 ** -21
