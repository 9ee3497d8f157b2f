"""Attention over coded pages where a step mixes single tokens with portions, at the sizes at which the kernels change."""
import math

import numpy as np
import pytest
import torch

from tests.plain import cache8 as plain
from tests.test_cache8_gpu import DEV, Setup, rts  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,starts,nh,nkv,hd,P,window,cap", [
    ([1, 1, 40], [30, 200, 50], 71, 1, 64, 128, 0, 0.0),          # more than 64 query heads a kv head, pages of 128
    ([1, 40, 1], [9, 70, 33], 130, 1, 32, 16, 0, 30.0),           # more than 128
    ([1, 1, 3, 20], [100, 5, 40, 0], 140, 2, 48, 48, 25, 0.0),    # two groups of 70, pages of 48, a window
    ([1, 1, 40], [30, 200, 50], 100, 1, 64, 32, 0, 50.0),         # what the portion kernel still takes
    ([1, 1, 40], [30, 200, 50], 64, 1, 64, 128, 0, 50.0),         # and what the prompt kernel does
])
def test_single_tokens_in_front_of_portions(rts, lens, starts, nh, nkv, hd, P, window, cap):
    """Against the definition.  Codes are arbitrary bytes: values of another request's keys, or of none, are off by the order of
    the largest value; probabilities, tanh.approx and the result's rounding by 0.012 of it at most (scores of a few units)."""
    from glint_b200 import ops_cache8
    rt = rts["bfloat16"]
    s = Setup(rt, lens, starts, nkv, hd, P, seed=nh, window=window)
    q = (0.1 * torch.randn(sum(lens), nh * hd, generator=torch.Generator().manual_seed(nh))).to(rt.dtype)
    out = ops_cache8.attention(rt, s.cache, s.step, q.to(DEV), nh, 1.0 / math.sqrt(hd), softcap=cap, window=window)
    rt.check_status()
    got, qd = (t.double().cpu().numpy().reshape(-1, nh, hd) for t in (out, q))
    for r, (n, start) in enumerate(zip(lens, starts)):
        for i in sorted({0, n // 2, n - 1}):
            lo = max(0, start + i - window + 1) if window else 0
            for head in sorted({0, 1, nh // 2, nh - 1}):
                k, v = s.values(0, r, head // (nh // nkv)), s.values(1, r, head // (nh // nkv))
                want = plain.attend(qd[s.cu[r] + i, head], k, v, 1.0 / math.sqrt(hd), cap, lo, start + i + 1)
                err = np.abs(got[s.cu[r] + i, head] - want).max()
                assert err <= 0.012 * np.abs(v[lo:start + i + 1]).max(), (r, i, head, err)
