"""Caches in 8 bits that share their wide pages and scratch, and what the cache takes in memory.  No GPU."""
import pytest
import torch

from glint_b200 import ops_cache8
from glint_b200.cache import CodedKVNeed, PagedKVNeed, cache_bytes_per_token
from glint_b200.errors import KernelError
from tests.test_cache8 import _pretend, _tensors


def _bytes(caches):
    """Of pools and scales, each storage once."""
    seen = {}
    for c in caches:
        for t in (c.k, c.v, c.k_scale, c.v_scale, c.k_wide, c.v_wide):
            seen[t.data_ptr()] = t.numel() * t.element_size()
    return sum(seen.values())


def test_layers_share_the_wide_pages(monkeypatch):
    _pretend(monkeypatch)
    make = lambda like=None: ops_cache8.Cache8.empty(6, 2, 16, 64, device="cpu", like=like)
    first = make()
    layers = [first] + [make(first) for _ in range(7)]
    for c in layers[1:]:
        assert c.k_wide is first.k_wide and c.v_wide is first.v_wide and c.scratch is first.scratch
        assert c.struct.partials == first.struct.partials and c.struct.arrive == first.struct.arrive
        assert c.struct.k_wide == first.struct.k_wide and c.struct.k != first.struct.k and c.struct.k_scale != first.struct.k_scale
    assert len({c.k.data_ptr() for c in layers}) == 8
    wide = 8 * 2 * first.k.numel() * 2
    scales = 8 * 2 * 6 * 2 * 4
    assert _bytes(layers) == wide // 2 + wide // 8 + scales               # codes, one layer's worth of wide pages
    own = make()
    assert own.scratch is not first.scratch and own.k_wide.data_ptr() != first.k_wide.data_ptr()


@pytest.mark.parametrize("sizes,dtype", [((7, 2, 16, 64), torch.bfloat16), ((6, 1, 16, 64), torch.bfloat16), ((6, 2, 32, 64), torch.bfloat16),
                                         ((6, 2, 16, 32), torch.bfloat16), ((6, 2, 16, 64), torch.float32)])
def test_what_cannot_be_shared_is_refused(monkeypatch, sizes, dtype):
    _pretend(monkeypatch)
    first = ops_cache8.Cache8.empty(6, 2, 16, 64, device="cpu")
    with pytest.raises(KernelError, match="share"):
        ops_cache8.Cache8.empty(*sizes, dtype=dtype, device="cpu", like=first)
    with pytest.raises(KernelError, match="one device"):
        ops_cache8.Cache8(*_tensors(), tuple(t.to("meta") for t in first.scratch))


@pytest.mark.parametrize("layers,times", [(42, 1.83), (26, 1.73), (46, 1.84)])
def test_tokens_in_the_same_memory(layers, times):
    """What the documents say: alternating layers with and without a window are two groups, each with one layer's pages wide."""
    per = {}
    for need in (PagedKVNeed, CodedKVNeed):
        kinds = [need(8, 256, 4096), need(8, 256, None)]
        per[need] = cache_bytes_per_token([kinds[i % 2] for i in range(layers)], [None] * layers, 2)
    assert abs(per[PagedKVNeed] / per[CodedKVNeed] - times) < 0.01
