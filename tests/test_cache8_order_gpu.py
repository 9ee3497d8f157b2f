"""The coded cache's operators behind kernels that write a step's arrays: what they read is what those kernels leave."""
import pytest
import torch

from tests.test_cache8_gpu import DEV, Setup, _qkv, _turns, rts  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,starts", [([1] * 8, [40 * i + 3 for i in range(8)]), ([60, 20], [7, 300])])
def test_arrays_written_by_a_kernel_that_lets_its_successor_begin(rts, lens, starts):
    """Positions, starts, table and turns come from kernels directly in front of every call (the ones that place values release
    their successor before they write); attention, append and widening give, bit for bit, what they give once the device is idle."""
    from glint_b200 import ops, ops_cache8
    rt, nh, nkv, hd, P = rts["bfloat16"], 8, 4, 128, 16
    T, R = sum(lens), len(lens)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    qkv = _qkv(T, nh, nkv, hd, 1, 0.3).to(DEV)
    turns = _turns(hd // 2).to(DEV)
    results = []
    for idle in (True, False):
        s = Setup(rt, lens, [a + 40 for a in starts], nkv, hd, P, seed=6)
        t = s.step.tensors
        table = t["block_table"].clone()
        rows = {n: torch.arange(t[n].numel(), dtype=torch.int32, device=DEV) for n in ("positions", "seq_start", "block_table")}
        own = torch.empty_like(turns)
        wait = torch.cuda.synchronize if idle else (lambda: None)
        got = []
        for at in range(40):
            sources = {"positions": i32([a + at + k for a, n in zip(starts, lens) for k in range(n)]),
                       "seq_start": i32([a + at for a in starts]), "block_table": table.view(-1)}
            torch.cuda.synchronize()
            def behind_the_writers(call):
                own.zero_()
                for n in rows:
                    t[n].zero_()
                own.copy_(turns)
                for n in rows:
                    ops.place_tokens(t[n].view(-1), rows[n], sources[n], rows[n])
                s.step.begin()
                wait()
                got.append(call())
                wait()
                return got[-1]
            q = behind_the_writers(lambda: ops_cache8.append(rt, s.cache, s.step, qkv, own, nh))
            behind_the_writers(lambda: ops_cache8.attention(rt, s.cache, s.step, q, nh, 0.1, softcap=50.0))
            behind_the_writers(lambda: torch.stack(ops_cache8.unpack(rt, s.cache, s.step)))
        got += [t.clone() for t in (s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale)]
        rt.check_status()
        results.append(got)
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_portions_between_products_and_beside_others(rts, hd):
    """Portions in front of tiled products, which take tensor memory of their own while they wait, and at the same time portions
    over another cache on another stream: bit for bit what each gives alone."""
    from glint_b200 import ops_cache8, ops_tensor
    rt, nh, nkv, P = rts["bfloat16"], 8, 4, 16
    g = torch.Generator().manual_seed(hd)
    setups = [Setup(rt, [300, 40], [150, 900], nkv, hd, P, seed=s) for s in (1, 2)]
    q = (0.2 * torch.randn(340, nh * hd, generator=g)).to(DEV, torch.bfloat16)
    w = (0.05 * torch.randn(256, nh * hd, generator=g)).to(DEV, torch.bfloat16)

    def once(s, product):
        out = ops_cache8.attention(rt, s.cache, s.step, q, nh, 0.1, softcap=50.0)
        y = torch.empty(340, 256, dtype=torch.float32, device=DEV)
        if product:
            ops_tensor.gemm(out, w, y, status=rt.status, force_splits=1, path="tcgen05")
        return (out, y) if product else (out,)
    want = []
    for k, s in enumerate(setups):
        want.append(once(s, k == 0))
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in setups]
    got = [[], []]
    for _ in range(20):
        for k, (s, stream) in enumerate(zip(setups, streams)):
            with torch.cuda.stream(stream):
                got[k].append(once(s, k == 0))
    torch.cuda.synchronize()
    rt.check_status()
    for k in range(2):
        for outs in got[k]:
            for a, b in zip(outs, want[k]):
                assert torch.equal(a, b)


@pytest.mark.parametrize("lens,starts", [([1] * 6, [0] * 6), ([200, 1], [0, 0])])
def test_layers_that_share_scratch(rts, lens, starts):
    """Three layers' appends and attention, step after step on one stream, over caches that share their wide pages and scratch: bit for
    bit what caches of their own give."""
    from glint_b200 import ops_cache8
    rt, nh, nkv, hd, P, layers = rts["bfloat16"], 4, 2, 128, 16, 3
    R, pages = len(lens), 40
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1))[:R * (pages // R)].view(R, -1).to(DEV, torch.int32)
    turns = _turns(hd // 2).to(DEV)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    results = []
    for shared in (False, True):
        caches = [ops_cache8.Cache8.empty(pages, nkv, P, hd)]
        caches += [ops_cache8.Cache8.empty(pages, nkv, P, hd, like=caches[0] if shared else None) for _ in range(layers - 1)]
        at, outs = list(starts), []
        for step_no in range(4):
            ns = lens if step_no == 0 else [1 + step_no % 2] * R
            pos = [a + k for a, n in zip(at, ns) for k in range(n)]
            cu = [sum(ns[:r]) for r in range(R + 1)]
            step = ops_cache8.StepArrays(i32(pos), i32([r for r, n in enumerate(ns) for _ in range(n)]), i32(at), i32(cu), table, max(ns),
                                         max(a + n for a, n in zip(at, ns)))
            for layer, cache in enumerate(caches):
                q = ops_cache8.append(rt, cache, step, _qkv(len(pos), nh, nkv, hd, 10 * step_no + layer, 0.3).to(DEV), turns, nh)
                outs.append(ops_cache8.attention(rt, cache, step, q, nh, 0.1, softcap=50.0))
            at = [a + n for a, n in zip(at, ns)]
        rt.check_status()
        results.append(outs + [getattr(c, n) for c in caches for n in ("k", "v", "k_scale", "v_scale")])
    for a, b in zip(*results):
        assert torch.equal(a, b)
