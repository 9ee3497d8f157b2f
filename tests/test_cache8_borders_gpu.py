"""Keys whose page's scale, or whose code, hangs on the last bits of the rotation: what the definition in 64 bits says."""
import math

import numpy as np
import pytest
import torch

from tests.plain import cache8 as plain
from tests.test_cache8_gpu import DEV, Setup, _turns, rts  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def _key_next_to(power, pos, turn, amp, rng):
    """A pair of float32 numbers that rotation brings within a few 2^-24 of (+-power, something smaller)."""
    angle = 2.0 * math.pi * math.fmod(pos * turn, 1.0)
    c, s = math.cos(angle), math.sin(angle)
    x, y = rng.choice([-1.0, 1.0]) * power / amp, rng.uniform(-0.9, 0.9) * power / amp
    return np.float32(x * c + y * s), np.float32(y * c - x * s)


@pytest.mark.parametrize("hd,P,pairs,inter,amp", [(64, 16, 32, False, 1.0), (128, 16, 32, True, 1.3), (256, 32, 128, False, 1.0), (96, 16, 48, False, 0.8),
                                                  (256, 16, 33, True, 1.0), (10, 8, 5, False, 1.0), (128, 256, 64, False, 1.0)])
def test_scales_next_to_a_power_of_two(rts, hd, P, pairs, inter, amp):
    """Every page has one key within a few 2^-24 of a power of two, half of them below: the scales and all codes are, to the last,
    those of the definition (the test's own 64 bits are off by 2^-50 or so; no value here is that near)."""
    from glint_b200 import ops_cache8
    rt, nkv, pages, start = rts["bfloat16"], 2, 24, 0
    T = pages * P
    rng = np.random.default_rng(hd + P)
    turns = _turns(pairs)
    x = (0.25 * rng.standard_normal((T, 3 * nkv, hd))).clip(-0.45, 0.45).astype(np.float32)
    for page in range(pages):
        for h in range(nkv):
            p, j = page * P + int(rng.integers(0, P)), int(rng.integers(0, pairs))
            a, b = (2 * j, 2 * j + 1) if inter else (j, j + pairs)
            x[p, nkv + h, a], x[p, nkv + h, b] = _key_next_to(1.0, p, float(turns[j]), amp, rng)
    s = Setup(rt, [T], [start], nkv, hd, P, seed=1)
    ops_cache8.append(rt, s.cache, s.step, torch.from_numpy(x.reshape(T, -1)).to(DEV), turns.to(DEV), nkv,
                      layout="interleaved" if inter else "half", amplitude=amp)
    rt.check_status()
    codes, scales = s.cache.k.cpu().numpy(), s.cache.k_scale.double().cpu().numpy()
    below = 0
    for h in range(nkv):
        y = np.stack([plain.rotate(x[t, nkv + h].astype(np.float64), t, turns.numpy(), inter, amp) for t in range(T)])
        for page in range(pages):
            part = y[page * P:(page + 1) * P]
            top = np.abs(part).max()
            assert top == 1.0 or 2.0 ** -40 < abs(top - 1.0) < 2.0 ** -21      # (position 0 turns nothing: exactly 1)
            below += top < 1.0
            e, i = plain.exponent(top), int(s.table[0, page])
            assert scales[i, h] == 2.0 ** e, (h, page, top - 1.0)
            assert np.array_equal(codes[i, h], (np.floor(part * 2.0 ** -e) + 128).astype(np.int64)), (h, page, top - 1.0)
    assert 0.25 * nkv * pages <= below <= 0.75 * nkv * pages
