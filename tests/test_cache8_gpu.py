"""The 8-bit key/value cache's operators against a plain 64-bit restatement: rotate and append, widen, attend; alone,
in a run as a step makes it, and in the engine."""
import math

import numpy as np
import pytest
import torch

from tests.plain import cache8 as plain

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def rts():
    from glint_b200.runtime import Runtime
    return {d: Runtime(DEV, d) for d in ("bfloat16", "float32")}


class Setup:
    """Requests with ``starts`` cached tokens that bring ``lens`` more, in shuffled pages of a pool with some to spare
    (filled with arbitrary bytes: nothing may depend on what a page held before)."""

    def __init__(self, rt, lens, starts, nkv, hd, page, seed=0, window=0, history=True):
        from glint_b200 import ops_cache8
        rng = np.random.default_rng(seed)
        self.rt, self.lens, self.starts, self.nkv, self.hd, self.P = rt, lens, starts, nkv, hd, page
        R = len(lens)
        self.spans = [(max(0, s - window + 1) // page if window else 0, (s + n - 1) // page + 1) for n, s in zip(lens, starts)]
        need = sum(b - a for a, b in self.spans)
        pages = need + 3
        order = rng.permutation(pages)
        self.table = np.full((R, max(b for _, b in self.spans) + 1), -1, dtype=np.int32)
        at = 0
        for r, (a, b) in enumerate(self.spans):
            self.table[r, a:b] = order[at:at + b - a]
            at += b - a
        self.spare = [int(p) for p in order[at:]]
        self.codes = [rng.integers(0, 256, size=(pages, nkv, page, hd), dtype=np.uint8) for _ in range(2)]
        self.e = [rng.integers(-9, -3, size=(pages, nkv)) for _ in range(2)]
        d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
        self.cache = ops_cache8.Cache8(
            d(self.codes[0]), d(self.codes[1]), d((2.0 ** self.e[0]).astype(np.float32)), d((2.0 ** self.e[1]).astype(np.float32)),
            torch.zeros(pages, nkv, page, hd, dtype=rt.dtype, device=DEV), torch.zeros(pages, nkv, page, hd, dtype=rt.dtype, device=DEV))
        self.positions = np.concatenate([np.arange(s, s + n) for n, s in zip(lens, starts)]).astype(np.int32)
        cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        self.cu = cu
        single = [s + 1 for n, s in zip(lens, starts)]
        lead = next((i for i, n in enumerate(lens) if n != 1), R)
        self.step = ops_cache8.StepArrays(d(self.positions), d(np.repeat(np.arange(R), lens).astype(np.int32)),
                                          d(np.asarray(starts, np.int32)), d(cu), d(self.table), max(lens),
                                          max(n + s for n, s in zip(lens, starts)), contexts=single[:lead])

    def page(self, which, r, place, h):
        i = self.table[r, place]
        return plain.Page(self.P, self.hd, self.codes[which][i, h], int(self.e[which][i, h]))

    def values(self, which, r, h):
        """Keys or values of request r from position 0 (NaN where its pages were given back)."""
        a, b = self.spans[r]
        out = np.full((b * self.P, self.hd), np.nan)
        for place in range(a, b):
            out[place * self.P:(place + 1) * self.P] = self.page(which, r, place, h).values()
        return out


def _qkv(T, nh, nkv, hd, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, nh + 2 * nkv, hd, generator=g) * torch.exp(spread * torch.randn(T, nh + 2 * nkv, 1, generator=g))
    return x.reshape(T, (nh + 2 * nkv) * hd).contiguous()


def _turns(pairs, theta=10000.0):
    return torch.from_numpy(theta ** (-np.arange(pairs) / max(pairs, 1)) / (2 * np.pi))


APPENDS = [  # lens, starts, nh, nkv, hd, page, pairs, interleaved, amplitude
    ([1], [0], 2, 1, 16, 16, 8, False, 1.0),
    ([1], [37], 8, 4, 256, 16, 128, False, 1.0),
    ([1, 1, 1, 1, 1], [0, 15, 16, 31, 1000], 4, 2, 64, 16, 32, False, 1.0),
    ([50], [0], 4, 4, 48, 16, 24, True, 1.0),
    ([50], [13], 6, 2, 96, 16, 24, False, 1.3),
    ([1, 1, 70, 3, 33], [5, 100, 7, 16, 31], 4, 1, 80, 32, 20, True, 0.8),
    ([17, 2], [99000, 130000], 16, 8, 128, 16, 64, False, 1.0),
    ([200], [61], 2, 2, 32, 64, 16, False, 1.0),
    ([40], [3], 3, 1, 10, 8, 5, False, 1.0),                # a head size that no vector form takes, small pages
    ([9], [0], 2, 1, 6, 3, 1, True, 1.0),                   # odd pages, one pair of three turned
    ([5, 6], [2, 0], 2, 2, 64, 16, 0, False, 1.0),          # nothing turned
    ([300], [250], 4, 2, 256, 256, 128, False, 1.0),        # pages of 256
    ([40, 1], [5, 7], 6, 2, 128, 16, 32, True, 1.2),        # heads of 64, 128 and 256, all or some of them turned
    ([20, 1], [5, 14], 2, 1, 128, 16, 24, False, 0.9),
    ([1, 30], [9, 3], 4, 2, 256, 16, 32, False, 1.0),
    ([30], [3], 4, 2, 256, 32, 33, False, 1.0),
    ([30], [3], 5, 1, 256, 16, 128, True, 1.0),
    ([30], [30], 3, 1, 64, 16, 7, True, 1.0),
    ([30], [30], 3, 1, 256, 16, 0, False, 1.0),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_against_the_definition(rts, dtype, case):
    """Codes: the kernel's 32-bit rotation is off by at most 4 ulp of the pair's length (two products, a sum, and
    cosine and sine each within an ulp), so a code differs by at most 1, and only where the 64-bit value lies that near a
    border.  Queries: the same 4 ulp (2^-22 of the pair's length) and a rounding to bfloat16 (2^-8 of the result).  The
    exponent of a page can differ only if its largest magnitude is that near a power of two: not at these seeds."""
    from glint_b200 import ops_cache8
    lens, starts, nh, nkv, hd, P, pairs, inter, amp = APPENDS[case]
    rt = rts[dtype]
    s = Setup(rt, lens, starts, nkv, hd, P, seed=case)
    T = sum(lens)
    qkv, turns = _qkv(T, nh, nkv, hd, case), _turns(pairs)
    q = ops_cache8.append(rt, s.cache, s.step, qkv.to(DEV), turns.to(DEV), nh, layout="interleaved" if inter else "half",
                          amplitude=amp)
    rt.check_status()
    x = qkv.double().numpy().reshape(T, nh + 2 * nkv, hd)
    got_q = q.double().cpu().numpy().reshape(T, nh, hd)
    unit = 2.0 ** -8 if dtype == "bfloat16" else 0.0
    for t in range(0, T, max(1, T // 40)):
        for h in range(nh):
            want = plain.rotate(x[t, h], int(s.positions[t]), turns.numpy(), inter, amp)
            top = max(amp, 1.0) * np.abs(x[t, h]).max() * 1.5
            assert np.all(np.abs(got_q[t, h] - want) <= unit * np.abs(want) + 2.0 ** -22 * top)
    codes = [s.cache.k.cpu().numpy(), s.cache.v.cpu().numpy()]
    scales = [s.cache.k_scale.double().cpu().numpy(), s.cache.v_scale.double().cpu().numpy()]
    touched = set()
    for r, (n, start) in enumerate(zip(lens, starts)):
        for h in range(nkv):
            for which in range(2):
                for place in range(start // P, (start + n - 1) // P + 1):
                    page, i = s.page(which, r, place, h), int(s.table[r, place])
                    touched.add(i)
                    new = range(max(start, place * P), min(start + n, (place + 1) * P))
                    for p in new:
                        t = s.cu[r] + p - start
                        row = x[t, nh + nkv + h] if which else plain.rotate(x[t, nh + h], p, turns.numpy(), inter, amp)
                        page.add(p - place * P, row)
                    assert scales[which][i, h] == page.scale
                    if which:                                            # values are not turned: exact
                        assert np.array_equal(codes[which][i, h], page.codes)
                    else:
                        far = np.abs(codes[which][i, h].astype(int) - page.codes)
                        assert far.max() <= 1 and far.sum() <= 2 + 2e-3 * far.size
    for i in range(codes[0].shape[0]):
        if i not in touched:                                             # other pages stay as they were
            for which in range(2):
                assert np.array_equal(codes[which][i], s.codes[which][i])
                assert np.array_equal(scales[which][i], 2.0 ** s.e[which][i])


@pytest.mark.parametrize("nkv,hd,P,pairs,inter,amp", [(4, 256, 16, 128, False, 1.0), (4, 128, 16, 32, True, 1.3), (4, 64, 32, 32, False, 0.7),
                                                      (3, 96, 16, 48, True, 1.0), (3, 256, 16, 33, False, 1.0), (2, 10, 8, 5, False, 1.0)])
def test_codes_are_those_of_the_definition_to_the_last(rts, nkv, hd, P, pairs, inter, amp):
    """Codes of rotated keys next to a border between two are decided in 64 bits: 400 tokens at far positions, every code as the
    definition has it.  (The scale comes from 32 bits: pages whose largest magnitude lies within 2^-20 of a power of two are left out.)"""
    from glint_b200 import ops_cache8
    rt, T, start, nh = rts["bfloat16"], 400, 90001, nkv
    s = Setup(rt, [T], [start], nkv, hd, P, seed=hd, window=1)
    qkv, turns = _qkv(T, nh, nkv, hd, 3, 0.5), _turns(pairs)
    ops_cache8.append(rt, s.cache, s.step, qkv.to(DEV), turns.to(DEV), nh, layout="interleaved" if inter else "half", amplitude=amp)
    rt.check_status()
    codes = s.cache.k.cpu().numpy()
    x, n = qkv.double().numpy().reshape(T, nh + 2 * nkv, hd), 0
    for h in range(nkv):
        y = np.stack([plain.rotate(x[t, nh + h], start + t, turns.numpy(), inter, amp) for t in range(T)])
        first = -(-start // P) * P - start                       # the first page begun in this step
        for t in range(first, T, P):
            part = y[t:t + P]
            mantissa = math.frexp(np.abs(part).max())[0]
            if min(mantissa - 0.5, 1.0 - mantissa) < 2.0 ** -20:
                continue
            e = plain.exponent(np.abs(part).max())
            want = (np.floor(part * 2.0 ** -e) + 128).astype(np.int64)
            got = codes[s.table[0, (start + t) // P], h, :len(part)]
            assert np.array_equal(got, want), (h, t, np.abs(got - want).max(), (got != want).sum())
            n += 1
    assert n > 0.9 * nkv * ((T - first) // P)


@pytest.mark.parametrize("P,hd", [(16, 64), (32, 256), (8, 10)])
def test_append_does_not_depend_on_the_cuts(rts, P, hd):
    """75 tokens at once, one by one, and in odd portions leave the same codes and scales, bit for bit."""
    from glint_b200 import ops_cache8
    rt, T, nh, nkv = rts["bfloat16"], 75, 2, 2
    qkv, turns = _qkv(T, nh, nkv, hd, 3).to(DEV), _turns(hd // 2).to(DEV)
    seen = []
    for cuts in ([75], [1] * 75, [7, 30, 1, 1, 20, 16]):
        caches, at = None, 0
        for n in cuts:
            s = Setup(rt, [n], [at], nkv, hd, P, seed=5)
            whole = Setup(rt, [75], [0], nkv, hd, P, seed=5)
            if caches is None:
                caches = whole
            step = ops_cache8.StepArrays(s.step.tensors["positions"], s.step.tensors["token_seq"], s.step.tensors["seq_start"],
                                         s.step.tensors["cu_seqlens"], caches.step.tensors["block_table"], n, at + n)
            ops_cache8.append(rt, caches.cache, step, qkv[at:at + n].contiguous(), turns, nh)
            at += n
        rt.check_status()
        c = caches.cache
        seen.append([t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)])
    for other in seen[1:]:
        for a, b in zip(seen[0], other):
            # rows behind the last token hold what they held (the same arbitrary bytes in all three)
            assert torch.equal(a, b)


def test_append_extreme_magnitudes(rts):
    """Zeros, the smallest and the largest numbers, powers of two: codes and scales exactly by the definition (nothing
    is turned, so nothing is rounded)."""
    from glint_b200 import ops_cache8
    rt, hd, P = rts["float32"], 16, 16
    tops = [0.0, 1e-45, 1e-38, 2.0 ** -114, 2.0 ** -113, 1.0, 2.0, 1.9999999, 127.99999, 128.0, 1e30, 3.4028234e38]
    for first, second in [(a, b) for a in tops for b in (0.0, 1e-38, 1.0, 2.0, 3.4028234e38)]:
        s = Setup(rt, [2], [0], 1, hd, P, seed=1)
        x = np.linspace(-1.0, 1.0, 3 * hd, dtype=np.float64).reshape(1, 3, hd).repeat(2, 0)
        x[0], x[1] = x[0] * first, -x[1] * second
        x = x.astype(np.float32)
        ops_cache8.append(rt, s.cache, s.step, torch.from_numpy(x.reshape(2, -1).copy()).to(DEV),
                          torch.zeros(0, dtype=torch.float64, device=DEV), 1)
        for which, (codes, scale) in enumerate([(s.cache.k, s.cache.k_scale), (s.cache.v, s.cache.v_scale)]):
            page = s.page(which, 0, 0, 0)
            for i in range(2):
                page.add(i, x[i, 1 + which].astype(np.float64))
            i = int(s.table[0, 0])
            assert float(scale[i, 0].double()) == page.scale, (first, second)
            assert np.array_equal(codes[i, 0].cpu().numpy(), page.codes), (first, second)
    rt.check_status()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("place", ["key", "value"])
def test_what_is_not_finite_reaches_its_own_request_only(rts, bad, place):
    """A key or value that is not finite makes its page's scale NaN and the outputs of queries that see the page NaN;
    other requests, heads and pages are as without it, also where the poisoned page is page 0 of the pool; a page
    begun anew is sound again."""
    from glint_b200 import ops_cache8
    rt, nh, nkv, hd = rts["bfloat16"], 4, 2, 64
    outs = []
    for poison in (False, True):
        s = Setup(rt, [20, 40], [0, 0], nkv, hd, 16, seed=2)
        swap = int(s.table[0, 1])                            # request 0's second page becomes page 0
        t = s.table.copy()
        t[s.table == 0] = swap
        t[0, 1] = 0
        s.table = t
        s.step.tensors["block_table"].copy_(torch.from_numpy(t))
        qkv = _qkv(60, nh, nkv, hd, 4, 0.2)
        if poison:
            qkv.view(60, nh + 2 * nkv, hd)[17, nh + (nkv if place == "value" else 0) + 1, 5] = bad
        ops_cache8.append(rt, s.cache, s.step, qkv.to(DEV), torch.zeros(0, dtype=torch.float64, device=DEV), nh)
        scale = s.cache.v_scale if place == "value" else s.cache.k_scale
        assert bool(torch.isnan(scale[0, 1])) == poison and not bool(torch.isnan(scale[0, 0]))
        q = torch.randn(60, nh * hd, generator=torch.Generator().manual_seed(1)).to(DEV, torch.bfloat16)
        s.step.begin()
        outs.append(ops_cache8.attention(rt, s.cache, s.step, q, nh, 0.125).float().cpu().view(60, nh, hd))
        # the same as single tokens: the last token of each request
        one = ops_cache8.StepArrays(*[torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([19, 39], [0, 1], [19, 39], [0, 1, 2])],
                                    s.step.tensors["block_table"], 1, 40, contexts=[20, 40])
        single = ops_cache8.attention(rt, s.cache, one, q[[19, 59]].contiguous(), nh, 0.125).float().cpu().view(2, nh, hd)
        assert bool(torch.isnan(single[0, 2:]).all()) == poison and torch.isfinite(single[0, :2]).all()
        assert torch.isfinite(single[1]).all()
        if poison:
            again = Setup(rt, [4], [16], nkv, hd, 16, seed=2)
            step = ops_cache8.StepArrays(*[again.step.tensors[n] for n in ("positions", "token_seq", "seq_start", "cu_seqlens")],
                                         s.step.tensors["block_table"][:1].contiguous(), 4, 20)
            ops_cache8.append(rt, s.cache, step, _qkv(4, nh, nkv, hd, 9).to(DEV), torch.zeros(0, dtype=torch.float64, device=DEV), nh)
            assert torch.isfinite(s.cache.k_scale[0]).all() and torch.isfinite(s.cache.v_scale[0]).all()
    clean, poisoned = outs
    assert torch.isfinite(clean).all()
    assert torch.isnan(poisoned[16:20, 2:]).all()
    keep = torch.ones(60, nh, dtype=torch.bool)
    keep[16:20, 2:] = False
    assert torch.equal(clean[keep], poisoned[keep])
    rt.check_status()


def test_bad_pages_and_orders_are_reported_and_nothing_is_written(rts):
    from glint_b200 import ops_cache8
    from glint_b200.errors import KernelError
    rt, nh, nkv, hd = rts["bfloat16"], 2, 1, 32
    for change, what in [(lambda s: s.step.tensors["block_table"].fill_(-1), "no page"),
                         (lambda s: s.step.tensors["block_table"].fill_(10 ** 6), "no page"),
                         (lambda s: s.step.tensors["positions"].fill_(4), "ascending"),
                         (lambda s: s.step.tensors["token_seq"].copy_(torch.tensor([1, 0, 0], dtype=torch.int32)), "ascending")]:
        s = Setup(rt, [2, 1], [3, 0], nkv, hd, 16, seed=3)
        change(s)
        ops_cache8.append(rt, s.cache, s.step, _qkv(3, nh, nkv, hd, 1).to(DEV), _turns(16).to(DEV), nh)
        with pytest.raises(KernelError, match=what):
            rt.check_status()
        if what == "no page":
            assert np.array_equal(s.cache.k.cpu().numpy(), s.codes[0]) and np.array_equal(s.cache.v.cpu().numpy(), s.codes[1])
    s = Setup(rt, [2, 3], [3, 20], nkv, hd, 16, seed=3)
    s.step.tensors["block_table"].fill_(-1)
    ops_cache8.unpack(rt, s.cache, s.step)
    with pytest.raises(KernelError, match="attention read"):
        rt.check_status()
    assert not s.cache.k_wide.any() and not s.cache.v_wide.any()
    s = Setup(rt, [2, 3], [3, 20], nkv, hd, 16, seed=3)
    short = ops_cache8.StepArrays(*[s.step.tensors[m] for m in ("positions", "token_seq", "seq_start", "cu_seqlens", "block_table")], 3, 16)
    ops_cache8.unpack(rt, s.cache, short)
    with pytest.raises(KernelError, match="more tokens than its step"):
        rt.check_status()
    q = torch.zeros(2, nh * hd, dtype=torch.bfloat16, device=DEV)
    s = Setup(rt, [1, 1], [3, 20], nkv, hd, 16, seed=3)
    s.step.tensors["block_table"].fill_(10 ** 6)
    ops_cache8.attention(rt, s.cache, s.step, q, nh, 1.0)
    with pytest.raises(KernelError, match="attention read"):
        rt.check_status()


def test_positions_outside_the_block_table_are_reported():
    """Single tokens at positions that the block table has no room for, or below zero: reported, and the others' results are
    what they are without them, up to the order of their sums (a few ulp of 32 bits of values up to 8, before the result's
    rounding)."""
    from glint_b200 import ops_cache8
    from glint_b200.errors import KernelError
    from glint_b200.runtime import Runtime
    rt, nh, nkv, hd = Runtime(DEV, "bfloat16"), 2, 1, 32
    q = (0.1 * torch.randn(3, nh * hd, generator=torch.Generator().manual_seed(1))).to(DEV, torch.bfloat16)
    for P in (16, 128):
        for window in (0, 20):
            s = Setup(rt, [1, 1, 1], [3, 40, 20], nkv, hd, P, seed=3)
            good = ops_cache8.attention(rt, s.cache, s.step, q, nh, 1.0, window=window)
            rt.check_status()
            for bad in (-1, -1000, -2 ** 31, 16 * 128, 2 ** 31 - 1):
                s.step.tensors["positions"][1] = bad
                out = ops_cache8.attention(rt, s.cache, s.step, q, nh, 1.0, window=window)
                with pytest.raises(KernelError, match="attention read"):
                    rt.check_status()
                far = (out[[0, 2]].float() - good[[0, 2]].float()).abs()
                assert (far <= 2.0 ** -7 * good[[0, 2]].float().abs() + 2.0 ** -17).all()
                if bad < 0:
                    assert not out[1].any()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("lens,starts,nkv,hd,P,window", [([1], [0], 1, 16, 16, 0), ([3, 1, 40], [0, 50, 30], 2, 48, 16, 0),
                                                         ([5, 20], [100, 63], 3, 10, 7, 20), ([9], [200], 2, 128, 64, 64)])
def test_unpack_is_exact_and_leaves_other_pages(rts, dtype, lens, starts, nkv, hd, P, window):
    from glint_b200 import ops_cache8
    rt = rts[dtype]
    s = Setup(rt, lens, starts, nkv, hd, P, seed=hd, window=window)
    s.cache.k_wide.fill_(3.5)
    s.cache.v_wide.fill_(-3.5)
    k, v = ops_cache8.unpack(rt, s.cache, s.step, window=window)
    rt.check_status()
    k, v = k.double().cpu().numpy(), v.double().cpu().numpy()
    used = {int(s.table[r, p]) for r, (a, b) in enumerate(s.spans) for p in range(a, b)}
    for i in range(k.shape[0]):
        for h in range(nkv):
            if i in used:
                assert np.array_equal(k[i, h], (s.codes[0][i, h] - 127.5) * 2.0 ** s.e[0][i, h])
                assert np.array_equal(v[i, h], (s.codes[1][i, h] - 127.5) * 2.0 ** s.e[1][i, h])
            else:
                assert (k[i, h] == 3.5).all() and (v[i, h] == -3.5).all()


ATTENDS = [  # lens, starts, nh, nkv, hd, page, window, cap
    ([1], [0], 2, 1, 16, 16, 0, 0.0),
    ([1], [1999], 8, 4, 256, 16, 0, 50.0),
    ([1] * 5, [0, 15, 16, 130, 700], 4, 2, 64, 16, 0, 30.0),
    ([1] * 9, [3, 100, 200, 300, 400, 999, 5, 64, 63], 16, 8, 128, 16, 100, 50.0),
    ([1] * 40, list(range(0, 1200, 30)), 8, 4, 256, 16, 0, 50.0),
    ([1] * 20, list(range(10, 2010, 100)), 6, 2, 48, 16, 0, 0.0),
    ([1] * 70, [500 + 3 * i for i in range(70)], 16, 8, 96, 32, 333, 50.0),
    ([1] * 3, [900, 30, 64], 5, 1, 80, 64, 0, 50.0),
    ([1] * 3, [900, 30, 64], 24, 1, 64, 16, 0, 0.0),              # more query heads than a pass of the kernel takes
    ([1] * 2, [50, 300], 2, 1, 256, 128, 0, 0.0),                 # pages of 128
    ([1] * 2, [50, 300], 2, 1, 320, 16, 0, 0.0),                  # a head size that no tensor-core kernel takes
    ([1] * 2, [50, 90], 4, 2, 36, 12, 40, 20.0),                  # nor this one, nor these pages
    ([5], [300], 8, 4, 256, 16, 0, 0.0),
    ([200], [0], 4, 2, 128, 16, 0, 50.0),
    ([1, 1, 70, 3, 33], [5, 400, 7, 16, 31], 4, 1, 64, 16, 50, 50.0),
    ([1] * 12 + [150, 2], [100 * i for i in range(12)] + [77, 5], 16, 8, 256, 16, 0, 50.0),
    ([130, 65], [1000, 64], 6, 3, 80, 32, 200, 0.0),
    ([40], [100], 4, 4, 96, 64, 0, 0.0),
    ([40, 1], [100, 3], 4, 2, 64, 48, 30, 10.0),                  # pages that the tiled kernel does not take
    ([2 + i % 7 for i in range(75)], [(5 * i) % 200 for i in range(75)], 4, 2, 64, 16, 0, 50.0),     # more requests than a warp has lanes
    ([1] * 3 + [3] * 40 + [90, 20], [9, 100, 40] + [(11 * i) % 90 for i in range(40)] + [70, 130], 12, 4, 112, 32, 0, 0.0),
    ([130], [1500], 4, 2, 64, 16, 0, 50.0),                       # keys split over blocks, ...
    ([130], [1500], 4, 2, 64, 16, 0, 56.0),                       # ... with a running maximum
    ([100, 40], [2000, 1000], 6, 2, 128, 16, 0, 0.0),
    ([150, 3], [1700, 1200], 2, 1, 256, 64, 900, 0.0),            # ... through a window
    ([90] + [2] * 40, [2600] + [700 + i for i in range(40)], 10, 2, 48, 16, 0, 30.0),
    ([70, 3], [100, 7], 40, 1, 64, 16, 0, 50.0),                  # groups that do not divide 128, or fill it
    ([20], [60], 128, 1, 32, 16, 0, 0.0),
    ([80], [40], 4, 2, 16, 16, 0, 50.0),                          # head sizes between the usual ones
    ([80], [140], 4, 2, 240, 64, 0, 50.0),
    ([80], [140], 2, 1, 192, 32, 0, 0.0),
    ([150, 1, 1], [30, 4, 200], 4, 2, 64, 16, 1, 0.0),            # a window of one
    ([700], [1500], 34, 17, 48, 32, 0, 50.0),                     # a few blocks more than SMs
    ([1100], [900], 16, 16, 128, 16, 0, 56.0),
]


def _attention_case(rts, dtype, case, seed=0, level=1.0):
    from glint_b200 import ops_cache8
    lens, starts, nh, nkv, hd, P, window, cap = ATTENDS[case]
    rt = rts[dtype]
    s = Setup(rt, lens, starts, nkv, hd, P, seed=case + seed, window=window)
    T = sum(lens)
    g = torch.Generator().manual_seed(case)
    q = (level * 0.1 * torch.randn(T, nh * hd, generator=g)).to(rt.dtype)
    out = ops_cache8.attention(rt, s.cache, s.step, q.to(DEV), nh, 1.0 / math.sqrt(hd), softcap=cap, window=window)
    return s, q, out


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention_against_the_definition(rts, dtype, case):
    """Codes are arbitrary bytes, so keys and values are of about 128 * 2^e: values of 1/4 to 4, scores of order 1.

    float32: sums of up to 320 products in 32-bit, 2^-24 each and of random sign: 2^-24 * 320 relative to |q||k| is the worst;
    2e-4 of the largest value covers scores of a few units and the sums over keys.
    bfloat16: keys, values and queries are exact in the products; probabilities are rounded to 8 or 11 bits
    (2^-9 of each at most, so 2^-9 of the largest value), tanh.approx (2^-11 relative, of a capped score below 10: 0.005 in the
    exponent at worst, so 0.005 of the largest value) and the result's own rounding (2^-9): 0.012 of the largest value."""
    s, q, out = _attention_case(rts, dtype, case)
    rts[dtype].check_status()
    lens, starts, nh, nkv, hd, P, window, cap = ATTENDS[case]
    got = out.double().cpu().numpy().reshape(-1, nh, hd)
    qd = q.double().numpy().reshape(-1, nh, hd)
    assert np.isfinite(got).all()
    for r, (n, start) in enumerate(zip(lens, starts)):
        for h in range(nkv):
            k, v = s.values(0, r, h), s.values(1, r, h)
            for i in sorted({0, n // 3, n - 1}):
                p = start + i
                lo = max(0, p - window + 1) if window else 0
                for head in range(h * (nh // nkv), (h + 1) * (nh // nkv)):
                    want = plain.attend(qd[s.cu[r] + i, head], k, v, 1.0 / math.sqrt(hd), cap, lo, p + 1)
                    bound = (2e-4 if dtype == "float32" else 0.012) * np.abs(v[lo:p + 1]).max()
                    err = np.abs(got[s.cu[r] + i, head] - want).max()
                    assert err <= bound, (r, i, head, err, bound)


@pytest.mark.parametrize("lens,starts,hd,cap", [([150], [0], 256, 50.0), ([150], [0], 64, 55.0), ([130], [1500], 128, 55.0), ([1], [70], 128, 55.0)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("e", [-43, 0, 28])
def test_scores_that_all_reach_the_cap(rts, lens, starts, hd, cap, sign, e):
    """Every score at +cap or at -cap, over values of up to 2^-36, 2^7 and 2^35: the mean of the values.  Probabilities are
    equal, so that only their own rounding and the result's is left (2^-9 each), and tanh.approx does not matter: 0.012 of the
    largest value as elsewhere."""
    from glint_b200 import ops_cache8
    rt, nh, nkv, P = rts["bfloat16"], 4, 2, 16
    s = Setup(rt, lens, starts, nkv, hd, P, seed=9)
    s.codes[0][:] = 255
    s.cache.k.fill_(255)
    s.e[0][:], s.e[1][:] = 0, e
    s.cache.k_scale.fill_(1.0)
    s.cache.v_scale.fill_(2.0 ** e)
    q = torch.full((sum(lens), nh * hd), 8.0 * sign, dtype=torch.bfloat16, device=DEV)
    out = ops_cache8.attention(rt, s.cache, s.step, q, nh, 1.0, softcap=cap)
    rt.check_status()
    got = out.double().cpu().numpy().reshape(-1, nh, hd)
    for i in sorted({0, lens[0] // 2, lens[0] - 1}):
        for head in range(nh):
            v = s.values(1, 0, head // 2)[:starts[0] + i + 1]
            err = np.abs(got[i, head] - v.mean(axis=0)).max()
            assert err <= 0.012 * np.abs(v).max(), (i, head, err / np.abs(v).max())


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("lens,starts", [([0, 5, 0, 70, 1], [10, 3, 0, 20, 6]), ([1, 0, 0, 130], [400, 500, 0, 900]), ([1, 0, 1], [30, 9, 700]),
                                         ([0, 0], [5, 0]), ([], [])])
def test_requests_without_tokens_and_steps_without_requests(rts, dtype, lens, starts):
    """Requests that bring no token of a step, and steps without any: the others as the definition has them (tolerances as
    above)."""
    from glint_b200 import ops_cache8
    rt, nh, nkv, hd, P = rts[dtype], 4, 2, 64, 16
    T = sum(lens)
    if not lens:
        i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=DEV)
        cache = ops_cache8.Cache8.empty(2, nkv, P, hd, rt.dtype)
        step = ops_cache8.StepArrays(i32(0), i32(0), i32(0), i32(1), i32(0, 2), 0, 0)
    else:
        s = Setup(rt, lens, starts, nkv, hd, P, seed=3)
        cache, step = s.cache, s.step
    q = (0.1 * torch.randn(T, nh * hd, generator=torch.Generator().manual_seed(1))).to(rt.dtype)
    out = ops_cache8.attention(rt, cache, step, q.to(DEV), nh, 0.125, softcap=30.0)
    ops_cache8.unpack(rt, cache, step)
    rt.check_status()
    assert out.shape == q.shape
    got, qd = (t.double().cpu().numpy().reshape(-1, nh, hd) for t in (out, q))
    for r, (n, start) in enumerate(zip(lens, starts)):
        for i in sorted({0, n - 1}) if n else ():
            for head in range(nh):
                k, v = s.values(0, r, head // 2), s.values(1, r, head // 2)
                want = plain.attend(qd[s.cu[r] + i, head], k, v, 0.125, 30.0, 0, start + i + 1)
                bound = (2e-4 if dtype == "float32" else 0.012) * np.abs(v[:start + i + 1]).max()
                assert np.abs(got[s.cu[r] + i, head] - want).max() <= bound, (r, i, head)
    q2 = ops_cache8.append(rt, cache, step, _qkv(T, nh, nkv, hd, 1).to(DEV), _turns(32).to(DEV), nh)
    rt.check_status()
    assert q2.shape == q.shape


@pytest.mark.parametrize("case", [2, 4, 8, 14])
def test_attention_repeats_itself(rts, case):
    _, _, a = _attention_case(rts, "bfloat16", case)
    _, _, b = _attention_case(rts, "bfloat16", case)
    assert torch.equal(a, b)


def test_attention_over_pages_of_very_different_scales(rts):
    """Values whose pages' scales lie up to 2^40 apart, the large ones behind keys that get no weight (score -60 against
    0): the small ones' result keeps its precision, whichever comes first."""
    from glint_b200 import ops_cache8
    rt, nh, nkv, hd, P, n = rts["bfloat16"], 2, 1, 64, 16, 96
    for big_page in (0, 2, 5):
        for gap in (3, 6, 12, 40):
            s = Setup(rt, [1], [n - 1], nkv, hd, P, seed=gap)
            x = np.zeros((n, 2, hd))
            rng = np.random.default_rng(gap)
            x[:, 1] = rng.uniform(0.5, 1.0, size=(n, hd))
            x[big_page * P:(big_page + 1) * P, 1] *= 2.0 ** gap
            x[:, 0, 0] = 1.0
            x[big_page * P:(big_page + 1) * P, 0, 0] = -1.0
            q = torch.zeros(1, nh * hd)
            q[:, 0] = 30.0
            q[:, hd] = 90.0
            w = Setup(rt, [n], [0], nkv, hd, P, seed=gap)
            qkv = torch.cat([torch.zeros(n, nh * hd), torch.from_numpy(x.reshape(n, -1)).float()], 1)
            step = ops_cache8.StepArrays(*[w.step.tensors[m] for m in ("positions", "token_seq", "seq_start", "cu_seqlens")],
                                         s.step.tensors["block_table"], n, n)
            ops_cache8.append(rt, s.cache, step, qkv.to(DEV), torch.zeros(0, dtype=torch.float64, device=DEV), nh)
            got = ops_cache8.attention(rt, s.cache, s.step, q.to(DEV, torch.bfloat16), nh, 1.0)
            rt.check_status()
            k8, v8 = plain.coded(x[:, :1], P)[:, 0], plain.coded(x[:, 1:], P)[:, 0]
            for head in range(nh):
                want = plain.attend(q.double().numpy()[0, head * hd:(head + 1) * hd], k8, v8, 1.0, 0.0, 0, n)
                err = np.abs(got.double().cpu().numpy()[0, head * hd:(head + 1) * hd] - want).max()
                # rounding of the probabilities and of the result, as above; the large page's weight is e^-60 or less
                assert err <= 0.012 * np.abs(want).max(), (big_page, gap, head, err)


@pytest.mark.parametrize("lens,starts,cap", [([90], [40], 50.0), ([90], [40], 0.0), ([130], [1500], 0.0), ([1] * 4, [40, 700, 3, 90], 50.0)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_query_that_is_not_finite_reaches_its_own_row_only(rts, lens, starts, cap, bad):
    """Bit for bit: the other heads and tokens are what they are without it; its own row is not a number (infinity times codes
    of both signs is none either)."""
    from glint_b200 import ops_cache8
    rt, nh, nkv, hd = rts["bfloat16"], 4, 2, 64
    s = Setup(rt, lens, starts, nkv, hd, 16, seed=2)
    q = (0.1 * torch.randn(sum(lens), nh * hd, generator=torch.Generator().manual_seed(1))).to(DEV, torch.bfloat16)
    want = ops_cache8.attention(rt, s.cache, s.step, q, nh, 0.125, softcap=cap).view(-1, nh, hd)
    t, head = min(2, sum(lens) - 1), 1
    q.view(-1, nh, hd)[t, head, 5:7] = bad
    got = ops_cache8.attention(rt, s.cache, s.step, q, nh, 0.125, softcap=cap).view(-1, nh, hd)
    rt.check_status()
    assert got[t, head].isnan().all()
    got[t, head] = want[t, head]
    assert torch.equal(got, want)


@pytest.mark.parametrize("cap", [50.0, 0.0])
def test_portions_replayed_from_a_graph(rts, cap):
    """Append and attention of portions captured once for contexts of up to 2,000 tokens and replayed at others."""
    from glint_b200 import ops_cache8
    rt, nh, nkv, hd, P, lens = rts["bfloat16"], 4, 2, 128, 16, [70, 33]
    turns = _turns(hd // 2).to(DEV)
    s = Setup(rt, lens, [1900, 1800], nkv, hd, P, seed=6)
    qkv = _qkv(sum(lens), nh, nkv, hd, 1).to(DEV)
    names = ("k", "v", "k_scale", "v_scale")
    fresh = [getattr(s.cache, m).clone() for m in names]
    t = s.step.tensors

    def once():
        q = ops_cache8.append(rt, s.cache, s.step, qkv, turns, nh)
        return ops_cache8.attention(rt, s.cache, s.step, q, nh, 0.1, softcap=cap)

    def reset(starts, seed):
        t["positions"].copy_(torch.cat([torch.arange(a, a + n, dtype=torch.int32) for a, n in zip(starts, lens)]))
        t["seq_start"].copy_(torch.tensor(starts, dtype=torch.int32))
        qkv.copy_(_qkv(sum(lens), nh, nkv, hd, seed))
        for m, f in zip(names, fresh):
            getattr(s.cache, m).copy_(f)
        s.step.begin()
    once()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for starts, seed in (([1900, 1800], 2), ([0, 5], 3), ([700, 1799], 4)):
        reset(starts, seed)
        graph.replay()
        replayed = [out.clone()] + [getattr(s.cache, m).clone() for m in names]
        reset(starts, seed)
        eager = [once()] + [getattr(s.cache, m) for m in names]
        for a, b in zip(replayed, eager):
            assert torch.equal(a, b)
    rt.check_status()


def test_more_single_tokens_than_a_launch_takes(rts):
    """1,100 single tokens (a launch takes 1,024): every one as if it were alone, up to the order of its sums, which depends on
    the launch (a few ulp of 32 bits before the result's rounding: at most the two nearest bfloat16 values apart)."""
    from glint_b200 import ops_cache8
    rt, n, nh, nkv, hd = rts["bfloat16"], 1100, 2, 1, 16
    starts = [(7 * i) % 50 for i in range(n)]
    s = Setup(rt, [1] * n, starts, nkv, hd, 16, seed=4)
    q = (0.1 * torch.randn(n, nh * hd, generator=torch.Generator().manual_seed(2))).to(DEV, torch.bfloat16)
    out = ops_cache8.attention(rt, s.cache, s.step, q, nh, 0.25)
    t = s.step.tensors
    for i in (0, 500, 1023, 1024, 1099):
        one = ops_cache8.StepArrays(t["positions"][i:i + 1].contiguous(), torch.zeros(1, dtype=torch.int32, device=DEV),
                                    t["seq_start"][i:i + 1].contiguous(), torch.tensor([0, 1], dtype=torch.int32, device=DEV),
                                    t["block_table"][i:i + 1].contiguous(), 1, starts[i] + 1, contexts=[starts[i] + 1])
        alone = ops_cache8.attention(rt, s.cache, one, q[i:i + 1].contiguous(), nh, 0.25)
        far = (alone[0].float() - out[i].float()).abs()
        assert (far <= 2.0 ** -7 * alone[0].float().abs()).all()
    rt.check_status()


def test_pages_beyond_32_bit_offsets(rts):
    """A pool of 4.9e9 codes: requests in its last pages give, bit for bit, what they give in a small pool."""
    from glint_b200 import ops_cache8
    rt, nh, nkv, hd, P, pages = rts["bfloat16"], 4, 2, 256, 16, 600_000
    turns = _turns(hd // 2).to(DEV)
    outs = []
    for base, total in ((0, 16), (pages - 16, pages)):
        cache = ops_cache8.Cache8.empty(total, nkv, P, hd)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
        table = i32([[base + p for p in range(16)]])
        qkv = _qkv(201, nh, nkv, hd, 5, 0.3).to(DEV)
        got = []
        for a, b in ((0, 200), (200, 201)):
            step = ops_cache8.StepArrays(i32(list(range(a, b))), i32([0] * (b - a)), i32([a]), i32([0, b - a]), table, b - a, b,
                                         contexts=[b] if b - a == 1 else [])
            q = ops_cache8.append(rt, cache, step, qkv[a:b].contiguous(), turns, nh)
            got += [q, ops_cache8.attention(rt, cache, step, q, nh, 0.0625, softcap=50.0)]
        k, v = ops_cache8.unpack(rt, cache, step)
        outs.append([t.clone() for t in got] + [cache.k[base:base + 13].clone(), cache.v[base:base + 13].clone(),
                                               cache.k_scale[base:base + 13].clone(), k[base:base + 12].clone(), v[base:base + 12].clone()])
        del cache, k, v
        torch.cuda.empty_cache()
    rt.check_status()
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_a_step_as_it_is_made(rts):
    """Append, then attention of the appended tokens, for a portion, single tokens behind it and the mixture: against the
    definition over what the pages hold (read back), and on a stream of its own."""
    from glint_b200 import ops_cache8
    rt, nh, nkv, hd, P = rts["bfloat16"], 8, 4, 128, 16
    s = Setup(rt, [75, 40], [0, 0], nkv, hd, P, seed=8)
    side = torch.cuda.Stream()
    table = s.step.tensors["block_table"]
    table_np = s.table
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    turns = _turns(hd // 2).to(DEV)
    cursor = [0, 0]
    plan = [[60, 0], [1, 30], [1, 1], [13, 9]]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for which, lens in enumerate(plan):
            rows = [r for r in range(2) if lens[r]]
            ns, starts = [lens[r] for r in rows], [cursor[r] for r in rows]
            pos = np.concatenate([np.arange(a, a + n) for a, n in zip(starts, ns)])
            step = ops_cache8.StepArrays(i32(pos), i32(np.repeat(np.arange(len(rows)), ns)), i32(starts),
                                         i32(np.concatenate([[0], np.cumsum(ns)])), table[rows].contiguous(), max(ns),
                                         max(a + n for a, n in zip(starts, ns)),
                                         contexts=[starts[0] + 1] if ns[0] == 1 else [])
            q = ops_cache8.append(rt, s.cache, step, _qkv(sum(ns), nh, nkv, hd, 20 + which, 0.3).to(DEV), turns, nh)
            out = ops_cache8.attention(rt, s.cache, step, q, nh, 0.1, softcap=50.0)
            k = (s.cache.k.double() - 127.5) * s.cache.k_scale.double()[:, :, None, None]
            v = (s.cache.v.double() - 127.5) * s.cache.v_scale.double()[:, :, None, None]
            side.synchronize()
            k, v, qd, got = (t.double().cpu().numpy() for t in (k, v, q, out))
            t = 0
            for r, n, a in zip(rows, ns, starts):
                for i in sorted({0, n - 1}):
                    for h in range(nkv):
                        ids = table_np[r, :(a + i) // P + 1]
                        kk, vv = k[ids, h].reshape(-1, hd), v[ids, h].reshape(-1, hd)
                        for head in (2 * h, 2 * h + 1):
                            want = plain.attend(qd[t + i, head * hd:(head + 1) * hd], kk, vv, 0.1, 50.0, 0, a + i + 1)
                            assert np.abs(got[t + i, head * hd:(head + 1) * hd] - want).max() <= 0.012 * np.abs(vv[:a + i + 1]).max()
                t += n
                cursor[r] = a + n
    rt.check_status()


def test_graph_replays_with_other_values(rts):
    """Append and attention of single tokens captured once and replayed at other positions give what eager calls give."""
    from glint_b200 import ops_cache8
    rt, nh, nkv, hd, P, n = rts["bfloat16"], 8, 4, 256, 16, 24
    turns = _turns(hd // 2).to(DEV)
    s = Setup(rt, [1] * n, [200] * n, nkv, hd, P, seed=6)
    qkv = _qkv(n, nh, nkv, hd, 1).to(DEV)
    names = ("k", "v", "k_scale", "v_scale")
    fresh = [getattr(s.cache, m).clone() for m in names]
    t = s.step.tensors

    def once():
        q = ops_cache8.append(rt, s.cache, s.step, qkv, turns, nh)
        return ops_cache8.attention(rt, s.cache, s.step, q, nh, 0.0625, softcap=50.0)

    def reset(seed, top):
        pos = torch.from_numpy(np.random.default_rng(seed).integers(0, top, size=n).astype(np.int32)).to(DEV)
        t["positions"].copy_(pos)
        t["seq_start"].copy_(pos)
        qkv.copy_(_qkv(n, nh, nkv, hd, seed).to(DEV))
        for m, f in zip(names, fresh):
            getattr(s.cache, m).copy_(f)
        s.step.begin()
    once()
    reset(1, 200)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for seed, top in ((2, 200), (3, 20), (4, 200)):
        reset(seed, top)
        graph.replay()
        replayed = [out.clone()] + [getattr(s.cache, m).clone() for m in names]
        reset(seed, top)
        eager = [once()] + [getattr(s.cache, m) for m in names]
        for a, b in zip(replayed, eager):
            assert torch.equal(a, b)
    rt.check_status()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("inter,rot,amp", [(True, 64, 1.0), (True, 24, 1.25), (False, 32, 0.5), (False, 64, 1.0)])
def test_rotary_forms_into_wide_pages(rts, dtype, inter, rot, amp):
    """The kernel that takes every rotary form, writing pages of the activations' type (4 ulp of 32 bits and the
    storage's rounding, as for queries), and queries only when there is no pool."""
    from glint_b200 import ops
    rt, nh, nkv, hd, P = rts[dtype], 4, 2, 64, 16
    s = Setup(rt, [20, 3], [77, 5], nkv, hd, P, seed=3)
    t = s.step.tensors
    qkv, turns = _qkv(23, nh, nkv, hd, 2, 0.3), _turns(rot // 2)
    q = torch.empty(23, nh * hd, dtype=rt.dtype, device=DEV)
    k, v = (torch.zeros(s.cache.num_pages, nkv, P, hd, dtype=rt.dtype, device=DEV) for _ in range(2))
    ops.rope_append(qkv.to(DEV), t["positions"], t["token_seq"], t["block_table"], turns.to(DEV), q, k, v, nh, nkv, hd, P,
                    s.cache.num_pages, rt.status, interleaved=inter, amplitude=amp)
    alone = torch.empty_like(q)
    ops.rope_append(qkv.to(DEV), t["positions"], t["token_seq"], t["block_table"], turns.to(DEV), alone, None, None, nh, nkv,
                    hd, P, s.cache.num_pages, rt.status, interleaved=inter, amplitude=amp)
    rt.check_status()
    assert torch.equal(q, alone)
    x = qkv.double().numpy().reshape(23, nh + 2 * nkv, hd)
    unit = 2.0 ** -8 if dtype == "bfloat16" else 0.0
    gq, gk, gv = q.double().cpu().numpy().reshape(23, nh, hd), k.double().cpu().numpy(), v.double().cpu().numpy()
    for i in range(23):
        r = 0 if i < 20 else 1
        p = int(s.positions[i])
        page, row = s.table[r, p // P], p % P
        for h in range(nh + nkv):
            want = plain.rotate(x[i, h], p, turns.numpy(), inter, amp)
            got = gq[i, h] if h < nh else gk[page, h - nh, row]
            assert np.all(np.abs(got - want) <= unit * np.abs(want) + 2.0 ** -22 * 1.5 * np.abs(x[i, h]).max())
        for h in range(nkv):
            assert np.all(np.abs(gv[page, h, row] - x[i, nh + nkv + h]) <= unit * np.abs(x[i, nh + nkv + h]))


# ---- in the engine -------------------------------------------------------------------------------------------------


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    from tests.helpers import make_model_dir
    return make_model_dir(tmp_path_factory.mktemp("cache8"), "C")


def _plain_with_codes(folder, tokens, coded):
    """The plain implementation with keys and values as the coded cache keeps them (pages of 16)."""
    from tests.plain import model
    c, w = model.read_config(folder), model.read_weights(folder, torch.float64)

    def attention(n, lw, c, layer):
        T, nh, nkv, hd = n.shape[0], c["heads"], c["kv_heads"], c["head_dim"]
        turn = lambda m, heads: model.rope_adjacent(n @ model.permute_qk_rows(m, heads, hd).T, list(range(T)), hd, c["theta"],
                                                    c["rope_factor"]).reshape(T, heads, hd).numpy()
        q, k, v = turn(lw["q"], nh), turn(lw["k"], nkv), (n @ lw["v"].T).reshape(T, nkv, hd).numpy()
        if coded:
            k, v = plain.coded(k, 16), plain.coded(v, 16)
        out = np.zeros((T, nh, hd))
        for p in range(T):
            lo = max(0, p - c["window"] + 1) if c["window"] is not None and layer % 2 == 0 else 0
            for h in range(nh):
                out[p, h] = plain.attend(q[p, h], k[:, h // (nh // nkv)], v[:, h // (nh // nkv)], c["scale"], c["attn_cap"], lo, p + 1)
        return torch.from_numpy(out.reshape(T, -1)) @ lw["o"].T
    real = model.attention
    model.attention = attention
    try:
        return model.forward(c, w, tokens).numpy()
    finally:
        model.attention = real


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_engine_against_the_plain_implementation_with_codes(folder, dtype):
    """A whole prompt in one step, so that every page is complete when it is read.  What the codes change in the logits
    is the yardstick: a code at a border that 32-bit arithmetic puts on the other side is a full step off where the codes
    themselves are a third of a step off on average, and fewer than 1 in 1000 are, so such borders move the logits by
    less than a tenth of what the codes do; a tenth more is left for 32-bit sums.  A wrong page, scale or head would move
    them by many times as much.  bfloat16 adds its own bound (0.025 of the largest logit)."""
    from glint_b200.engine.loading import build_engine, load_model
    from glint_b200.engine.step import StepEntry
    from tests.helpers import TINY, random_tokens, tolerance
    toks = random_tokens(75, TINY["C"][0]["vocab_size"], 3)
    want, without = _plain_with_codes(folder, toks, True), _plain_with_codes(folder, toks, False)
    moved = np.abs(want - without).max()
    assert moved > 1e-4 * np.abs(want).max()
    model = load_model(folder, dtype, cache_dtype="int8")
    engine = build_engine(model, 256, num_slots=2)
    assert engine.cache.views[0].k.dtype == torch.uint8
    slot = engine.open()
    got = engine.step([StepEntry(slot, toks, list(range(75)))]).double().cpu().numpy()
    model.rt.check_status()
    bound = 0.2 * moved if dtype == "float32" else tolerance(dtype, want)
    assert np.abs(got - want).max() <= bound, (np.abs(got - want).max(), moved)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_engine_under_cuts_in_batches_and_graphs(folder, dtype):
    """Prompts cut into portions, single tokens through graphs and mixed batches: logits as near to the wide cache's as
    the codes allow.  Reading a page before it is complete uses a finer or equal scale, so the bound is twice what the codes
    change in a whole prompt, and bfloat16's own."""
    from glint_b200.engine.loading import build_engine, load_model
    from glint_b200.engine.step import StepEntry
    from tests.helpers import TINY, random_tokens, tolerance
    toks = [random_tokens(n, TINY["C"][0]["vocab_size"], n) for n in (75, 60, 33)]
    ends = [(_plain_with_codes(folder, t, True), _plain_with_codes(folder, t, False)) for t in toks]
    model = load_model(folder, dtype, cache_dtype="int8")
    engine = build_engine(model, 512, num_slots=4)
    slots = [engine.open() for _ in toks]
    at = [0, 0, 0]
    seen = {}
    rng = np.random.default_rng(2)
    while any(a < len(t) for a, t in zip(at, toks)):
        entries = []
        for i, t in enumerate(toks):
            n = min(len(t) - at[i], 1 if min(at) > 20 else int(rng.integers(1, 20)))
            if n > 0:
                entries.append((i, StepEntry(slots[i], t[at[i]:at[i] + n], [n - 1])))
        entries.sort(key=lambda e: len(e[1].tokens))
        logits = engine.step([e for _, e in entries]).double().cpu().numpy()
        for row, (i, e) in zip(logits, entries):
            at[i] += len(e.tokens)
            seen[i, at[i] - 1] = row.copy()
    model.rt.check_status()
    assert engine.graph_counts["replayed"] > 0
    for (i, p), row in seen.items():
        want, without = ends[i]
        moved = np.abs(want - without).max()
        bound = 2 * moved if dtype == "float32" else 2 * moved + tolerance(dtype, want)
        assert np.abs(row - without[p]).max() <= bound, (i, p)


def test_entry_point_and_commands(folder, capsys):
    from glint_b200 import LLM
    from glint_b200.bench import check_generate
    from glint_b200.cli import main
    from tests.helpers import TINY, random_tokens
    llm = LLM(folder, dtype="bfloat16", cache_tokens=1024, max_active=4, cache_dtype="int8")
    assert all(g.name.endswith("/int8") for g in llm.engine.cache.groups)
    prompts = [random_tokens(n, TINY["C"][0]["vocab_size"], n) for n in (5, 40, 90)]
    check_generate(llm, prompts, new_tokens=12)
    with pytest.raises(ValueError, match="cache dtype"):
        LLM(folder, cache_dtype="int4")
    with pytest.raises(ValueError, match="keeps its cache"):
        LLM(model=llm.model, cache_dtype="auto", cache_tokens=256)
    assert main(["generate", "-f", folder, "-t", "5,17,3", "-m", "4", "--cache-dtype", "int8"]) == 0
    assert "Generated token ids: [5, 17, 3" in capsys.readouterr().out


def test_rotary_forms_through_the_engine(folder):
    """A model whose position parts are given another form: interleaved pairs over part of the head with yarn scaling, over
    wide and coded pages, decoding after a prompt as in one go (32-bit, so 2e-5 of the largest logit for the wide pages)."""
    from glint_b200.config import load_config
    from glint_b200.engine.loading import build_engine
    from glint_b200.engine.model import CausalLM
    from glint_b200.engine.step import StepEntry
    from glint_b200.runtime import Runtime
    from glint_b200.weights import load_weights
    from tests.helpers import TINY, random_tokens
    toks = random_tokens(50, TINY["C"][0]["vocab_size"], 8)
    out = {}
    for cache_dtype in (None, "int8"):
        config = load_config(folder)
        spec = config.model_spec()
        for b in spec.blocks:
            for part in vars(b).values():
                if getattr(part, "params", None) and "position" in part.params:
                    part.params["position"].params.update(layout="interleaved", rotary_dim=32,
                                                          scaling={"kind": "yarn", "factor": 4.0, "original_context": 64})
        model = CausalLM(spec, Runtime(DEV, "float32", "auto", cache_dtype))
        model.config = config
        load_weights(model, folder)
        assert model.blocks[0].mixer.position.only
        engine = build_engine(model, 256, num_slots=2)
        s = engine.open()
        whole = engine.step([StepEntry(s, toks, [49])]).clone()
        engine.close(s)
        s = engine.open()
        engine.step([StepEntry(s, toks[:40], [])])
        for t in toks[40:]:
            last = engine.step([StepEntry(s, [t], [0])])
        out[cache_dtype] = (whole.cpu(), last.clone().cpu())
        model.rt.check_status()
    whole, last = out[None]
    assert (whole - last).abs().max() <= 2e-5 * max(1.0, whole.abs().max().item())
    assert (out["int8"][0] - whole).abs().max() <= 0.05 * whole.abs().max()
