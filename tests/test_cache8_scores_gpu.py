"""Attention over coded pages where scores reach the soft cap and few keys have the weight: against the definition, within the error
that the kernels' own roundings allow at that row, and far from what a result without the cap, or without the scores, would be."""
import math

import numpy as np
import pytest
import torch

from tests.test_cache8_gpu import ATTENDS, DEV, Setup, rts  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def _softmax(s):
    w = np.exp(s - s.max())
    return w / w.sum()


def bound_of(kind, q, k, v, raw, s, cap, multiplier):
    """(expected output, most that a kernel's may be off, per dim).

    A change d_i of score i moves the output by sum w_i d_i (v_i - out) to first order, at most by exp(2 max d) times that much.
    A probability's relative rounding r moves it by r sum w_i |v_i| at most.  The scores:
    * the product's sum in 32 bits, at most 2^-24 a step and 2^-18 in all for up to 64 steps, relative to sum |q_d k_d|;
    * "tiled": tanh.approx, 2^-11 relative; "single": exponential and reciprocal to 2^-20 of the cap together, and queries as integers of 16
      bits: elements below 2^-7 of the row's largest are off by half of 2^-14 of it (a bfloat16 number above is exact);
      "32-bit": a few ulp, 2^-20;
    * the exponential, in log2 units of up to 2^7: 2^-16.
    Probabilities: 8 bits of bfloat16 ("tiled", 2^-8 with its half step), 11 of a half ("single", 2^-11), 32 (2^-18 for all sums).  Then
    the result's own rounding, 2^-8, and 2^-18 of the largest value for partial results and what underflows."""
    w = _softmax(s)
    out = w @ v
    size = (np.abs(k) @ np.abs(q)) * multiplier
    d = 2.0 ** -18 * size + 2.0 ** -16
    if kind == "single":
        low = np.where(np.abs(q) < 2.0 ** -7 * np.abs(q).max(), 2.0 ** -15 * np.abs(q).max(), 0.0)
        d = d + (np.abs(k) @ low) * multiplier + cap * 2.0 ** -20
    elif cap:
        d = d + np.abs(s) * (2.0 ** -11 if kind == "tiled" else 2.0 ** -20)
    moved = math.exp(2 * d.max()) * ((w * d) @ np.abs(v - out))
    r = {"tiled": 2.0 ** -8, "single": 2.0 ** -11, "32-bit": 2.0 ** -18}[kind]
    rounding = 0.0 if kind == "32-bit" else 2.0 ** -8
    return out, moved + r * (w @ np.abs(v)) + rounding * np.abs(out) + 2.0 ** -18 * np.abs(v).max()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("reach", [0.75, 2.5])
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_scores_up_to_the_cap(rts, dtype, reach, case):
    """Queries as large as brings the largest scores to 0.75 or 2.5 times the cap (10 or 30 without one)."""
    from glint_b200 import ops_cache8
    lens, starts, nh, nkv, hd, P, window, cap = ATTENDS[case]
    rt = rts[dtype]
    s = Setup(rt, lens, starts, nkv, hd, P, seed=case, window=window)
    T, G, multiplier = sum(lens), nh // nkv, 1.0 / math.sqrt(hd)
    largest = (reach * cap if cap else 13.0 * reach) / 16.0      # keys of up to 8, a root mean square of 4.6: 16 a unit at 3.5 deviations
    q = (largest * torch.randn(T, nh * hd, generator=torch.Generator().manual_seed(case))).to(rt.dtype)
    out = ops_cache8.attention(rt, s.cache, s.step, q.to(DEV), nh, multiplier, softcap=cap, window=window)
    rt.check_status()
    got, qd = (t.double().cpu().numpy().reshape(T, nh, hd) for t in (out, q))
    kind = "32-bit" if dtype == "float32" else "single" if max(lens) == 1 and hd % 16 == 0 and hd <= 256 and P % 16 == 0 else "tiled"
    rows = capped = told = 0
    for r in sorted({0, len(lens) // 2, len(lens) - 1}):
        n, start = lens[r], starts[r]
        for h in sorted({0, nkv - 1}):
            k, v = s.values(0, r, h), s.values(1, r, h)
            for i in sorted({0, n // 3, n - 1}):
                lo, hi = max(0, start + i - window + 1) if window else 0, start + i + 1
                for head in sorted({h * G, h * G + G - 1}):
                    query = qd[s.cu[r] + i, head]
                    raw = (k[lo:hi] @ query) * multiplier
                    scores = cap * np.tanh(raw / cap) if cap else raw
                    want, bound = bound_of(kind, query, k[lo:hi], v[lo:hi], raw, scores, cap, multiplier)
                    err = np.abs(got[s.cu[r] + i, head] - want)
                    assert (err <= bound).all(), (r, i, head, (err / bound).max())
                    if hi - lo >= 16:
                        rows += 1
                        capped += (np.abs(_softmax(raw) @ v[lo:hi] - want) > 2 * bound).any()
                        told += (np.abs(v[lo:hi].mean(axis=0) - want) > 2 * bound).any()
    # what a kernel without the cap, or one that does not look at its scores, would give lies outside
    assert told == rows and (not cap or capped >= (0.4 if reach > 1 else 0.05) * rows), (rows, capped, told)


@pytest.mark.parametrize("lens,starts,hd", [([150], [0], 64), ([130], [1500], 128), ([150], [400], 256), ([130], [1500], 256)])
def test_values_too_large_for_the_sums_of_portions_are_reported(rts, lens, starts, hd):
    """Scores at +cap over values of up to 2^(7 + e): inside the range the mean of the values, beyond it a report, and the same values
    without a cap, or as single tokens, are right.  A page that is not finite is no such report."""
    from glint_b200 import ops_cache8
    from glint_b200.errors import KernelError
    rt, nh, nkv, P = rts["bfloat16"], 4, 2, 16
    T = sum(lens)
    s = Setup(rt, lens, starts, nkv, hd, P, seed=9)
    s.cache.k.fill_(255)
    s.cache.k_scale.fill_(1.0)
    s.codes[1][:] = 255
    s.cache.v.fill_(255)
    q = torch.full((T, nh * hd), 8.0, dtype=torch.bfloat16, device=DEV)
    one = ops_cache8.StepArrays(*[torch.tensor(a, dtype=torch.int32, device=DEV) for a in ([starts[0] + T - 1], [0], [starts[0] + T - 1], [0, 1])],
                                s.step.tensors["block_table"], 1, starts[0] + T)
    for e in (0, 28, 70, 100):
        s.cache.v_scale.fill_(2.0 ** e)
        value = 127.5 * 2.0 ** e
        calls = [(s.step, q, 55.0, e < 30), (s.step, q, 0.0, e < 84), (one, q[:1], 55.0, True), (one, q[:1], 0.0, True)]
        for step, rows, cap, fine in calls:
            out = ops_cache8.attention(rt, s.cache, step, rows.contiguous(), nh, 1.0, softcap=cap).double()
            if fine:
                rt.check_status()
                assert ((out - value).abs() <= 2.0 ** -6 * value).all(), (e, cap)
            elif e == 70:
                with pytest.raises(KernelError, match="overflow"):
                    rt.check_status()
            else:                                   # past what is promised: right, or reported
                try:
                    rt.check_status()
                except KernelError:
                    continue
                assert ((out - value).abs() <= 2.0 ** -6 * value).all(), (e, cap)
    s.cache.v_scale.fill_(float("nan"))
    out = ops_cache8.attention(rt, s.cache, s.step, q, nh, 1.0, softcap=55.0)
    assert out.isnan().all()
    rt.check_status()
