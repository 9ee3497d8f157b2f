"""The 8-bit key/value cache on the host: its format, what it declares, what is refused before any launch, and the
frequencies of scaled rotary encodings.  No GPU."""
import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from glint_b200 import ops_cache8
from glint_b200.cache import CacheManager, CodedKVNeed, PagedKVNeed, cache_bytes_per_token
from glint_b200.errors import ConfigError, GlintError, KernelError
from tests.plain import cache8 as plain


@pytest.mark.parametrize("seed", range(4))
def test_a_page_depends_on_its_tokens_and_not_on_their_cuts(seed):
    """Shifting codes when the scale grows gives the codes at the final scale at once, and a value lies within half a
    step (at most 1/128 of the largest magnitude) of what it stands for."""
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((16, 24)) * np.exp(2.0 * rng.standard_normal((16, 1)))).astype(np.float32)
    page = plain.Page(16, 24)
    for i in range(16):
        page.add(i, x[i])
    e = plain.exponent(np.abs(x).max())
    assert page.e == e
    assert np.array_equal(page.q, np.floor(x.astype(np.float64) / 2.0 ** e))
    assert page.q.min() >= -128 and page.q.max() <= 127
    assert np.abs(page.values() - x).max() <= 2.0 ** e / 2 <= np.abs(x).max() / 128
    as_bf16 = torch.from_numpy(page.values()).to(torch.bfloat16).double().numpy()
    assert np.array_equal(as_bf16, page.values())                        # widening is exact


@pytest.mark.parametrize("top", [1.0, 2.0, np.nextafter(np.float32(2), np.float32(0)), 127.99999, 128.0, 3.4e38, 1e-38, 1e-45])
def test_scale_at_the_borders(top):
    e = plain.exponent(top)
    assert abs(np.float64(np.float32(top))) < 128 * 2.0 ** e
    assert e == plain.LOWEST or np.float64(np.float32(top)) >= 64 * 2.0 ** e


def test_declaration_and_accounting():
    a, b = CodedKVNeed(4, 64, None), CodedKVNeed(4, 64, 100)
    wide = PagedKVNeed(4, 64, None)
    assert a.group_key() != wide.group_key() and a.group_key() != b.group_key()
    assert a.readable_by(b) and not a.readable_by(wide) and not wide.readable_by(a)
    assert a.bytes_per_token(2) == 2 * 4 * 64 + 2                        # codes, and 8 scales' bytes over 16 tokens
    # two layers of one group share the wide pages, a third layer of another group has its own
    assert cache_bytes_per_token([a, a, b], [None] * 3, 2) == 3 * a.bytes_per_token(2) + 2 * 2 * 2 * 4 * 64
    assert cache_bytes_per_token([wide, wide], [None, None], 2) == 2 * 2 * 4 * 64 * 2
    m = CacheManager([a, a, b], [None, None, None], num_slots=2, num_pages=6, page_size=16, max_positions=64,
                     dtype=torch.bfloat16, device="cpu")
    assert len(m.groups) == 2 and m.bytes_per_token() == 3 * a.bytes_per_token(2) + 2 * 2 * 2 * 4 * 64
    v0, v1, v2 = m.views
    assert v0.k.dtype == torch.uint8 and v0.k.shape == (6, 4, 16, 64) and v0.k_scale.shape == (6, 4)
    assert v0.k_wide.data_ptr() == v1.k_wide.data_ptr() != v2.k_wide.data_ptr() and v0.k_wide.dtype == torch.bfloat16
    assert v0.k.data_ptr() != v1.k.data_ptr()
    with pytest.raises(GlintError, match="shapes differ"):
        CacheManager([a, wide], [None, 0], 2, 6, 16, 64, torch.bfloat16, "cpu")
    with pytest.raises(GlintError, match="shapes differ"):
        CacheManager([wide, a], [None, 0], 2, 6, 16, 64, torch.bfloat16, "cpu")


def test_odd_heads_are_refused_when_declared():
    PagedKVNeed(4, 33, None)
    with pytest.raises(GlintError, match="even"):
        CodedKVNeed(4, 33, None)


def test_cache_dtype_names():
    from glint_b200.runtime import parse_cache_dtype
    assert parse_cache_dtype(None) is None and parse_cache_dtype("auto") is None and parse_cache_dtype("int8") == "int8"
    with pytest.raises(KernelError, match="cache dtype"):
        parse_cache_dtype("int4")


def _pretend(monkeypatch):
    """Host checks with tensors that only claim to be on the device: nothing is launched."""
    def require(t, dtype, name):
        if t is not None and dtype is not None and t.dtype != dtype:
            raise KernelError(f"{name} must be {dtype}, is {t.dtype}")
        if t is not None and not t.is_contiguous():
            raise KernelError(f"{name} must be contiguous")
    monkeypatch.setattr(ops_cache8.ops, "require", require)

    def no_launch():
        raise AssertionError("a refused call reached the launch")
    monkeypatch.setattr(ops_cache8, "_lib", no_launch)


def _tensors(pages=3, nkv=2, P=16, hd=32):
    shape = (pages, nkv, P, hd)
    return [torch.zeros(shape, dtype=torch.uint8), torch.zeros(shape, dtype=torch.uint8), torch.zeros(shape[:2]),
            torch.zeros(shape[:2]), torch.zeros(shape, dtype=torch.bfloat16), torch.zeros(shape, dtype=torch.bfloat16)]


def _step(T=3, pages=3, **kw):
    i = lambda *v: torch.tensor(v, dtype=torch.int32)
    args = dict(positions=i(*range(T)), token_seq=i(*[0] * T), seq_start=i(0), cu_seqlens=i(0, T),
                block_table=torch.zeros(1, pages, dtype=torch.int32), max_seq_len=T, max_context=T)
    args.update(kw)
    return ops_cache8.StepArrays(**args)


def test_a_cpu_tensor_is_refused():
    with pytest.raises(KernelError, match="CUDA"):
        ops_cache8.Cache8(*_tensors())


def test_cache_refusals(monkeypatch):
    _pretend(monkeypatch)
    ops_cache8.Cache8(*_tensors())
    for k, bad, what in [(0, torch.zeros(3, 2, 16, 32, dtype=torch.int8), "uint8"),
                         (1, torch.zeros(3, 2, 16, 30, dtype=torch.uint8), "fit"),
                         (2, torch.zeros(3, 1), "fit"), (3, torch.zeros(3, 2, dtype=torch.float64), "float32"),
                         (4, torch.zeros(3, 2, 8, 32, dtype=torch.bfloat16), "fit"),
                         (5, torch.zeros(3, 2, 16, 32), "bfloat16"),
                         (0, torch.zeros(3, 2, 32, 16, dtype=torch.uint8).transpose(2, 3), "contiguous")]:
        t = _tensors()
        t[k] = bad
        with pytest.raises(KernelError, match=what):
            ops_cache8.Cache8(*t)
    with pytest.raises(KernelError, match="even"):
        ops_cache8.Cache8(*_tensors(hd=33))
    for k in (0, 1, 4, 5):                        # kernels move these 2 to 16 bytes at a time
        t = _tensors()
        t[k] = torch.zeros(t[k].numel() + 1, dtype=t[k].dtype)[1:].view(t[k].shape)
        with pytest.raises(KernelError, match="16 bytes"):
            ops_cache8.Cache8(*t)


def test_step_refusals(monkeypatch):
    _pretend(monkeypatch)
    _step()
    for kw in (dict(token_seq=torch.zeros(2, dtype=torch.int32)), dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)),
               dict(block_table=torch.zeros(2, 3, dtype=torch.int32)), dict(max_seq_len=4), dict(max_context=2),
               dict(max_seq_len=0), dict(contexts=[1, 1])):
        with pytest.raises(KernelError):
            _step(**kw)
    with pytest.raises(KernelError, match="int32"):
        _step(positions=torch.zeros(3, dtype=torch.int64))


def test_call_refusals(monkeypatch):
    """Every refusal comes before the launch."""
    _pretend(monkeypatch)
    cache, step = ops_cache8.Cache8(*_tensors()), _step()
    rt = SimpleNamespace(dtype=torch.bfloat16, device_index=-1, native=None)
    qkv, turns = torch.zeros(3, (4 + 4) * 32), torch.zeros(16, dtype=torch.float64)
    q = torch.zeros(3, 4 * 32, dtype=torch.bfloat16)
    for args, kw, what in [((qkv, turns, 3), {}, "evenly"), ((qkv, turns, 0), {}, "evenly"),
                           ((qkv[:, :-32].contiguous(), turns, 4), {}, "qkv"), ((qkv[:2], turns, 4), {}, "qkv"),
                           ((qkv.double(), turns, 4), {}, "float32"), ((qkv, turns.float(), 4), {}, "float64"),
                           ((qkv, torch.zeros(17, dtype=torch.float64), 4), {}, "turns"),
                           ((qkv, torch.zeros(32, dtype=torch.float64)[::2], 4), {}, "contiguous"),
                           ((qkv, turns, 4), dict(layout="pairs"), "layout"), ((qkv, turns, 4), dict(q_out=q.float()), "q_out"),
                           ((qkv, turns, 4), dict(q_out=q[:2]), "q_out")]:
        with pytest.raises(KernelError, match=what):
            ops_cache8.append(rt, cache, step, *args, **kw)
    for args, kw, what in [((q, 3, 1.0), {}, "evenly"), ((q.float(), 4, 1.0), {}, "bfloat16"), ((q[:2], 4, 1.0), {}, "q "),
                           ((q, 4, 1.0), dict(window=-1), "window"), ((q, 4, 1.0), dict(out=q[:, :64].contiguous()), "out")]:
        with pytest.raises(KernelError, match=what):
            ops_cache8.attention(rt, cache, step, *args, **kw)
    far = _step(max_context=49)                                          # three pages of 16 hold 48 positions
    with pytest.raises(KernelError, match="block table"):
        ops_cache8.attention(rt, cache, far, q, 4, 1.0)
    with pytest.raises(KernelError, match="block table"):
        ops_cache8.unpack(rt, cache, far)
    with pytest.raises(KernelError, match="wide"):
        ops_cache8.unpack(SimpleNamespace(dtype=torch.float32, device_index=-1), cache, step)
    with pytest.raises(KernelError, match="one device"):
        ops_cache8.unpack(SimpleNamespace(dtype=torch.bfloat16, device_index=0), cache, step)


# ---- scaled rotary frequencies -----------------------------------------------------------------------------------

FREQ = 10000.0 ** (-np.arange(0, 64, 2) / 64.0)


def test_single_operation_refusals(monkeypatch):
    _pretend(monkeypatch)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)
    good = dict(qkv=torch.zeros(3, 8 * 32), positions=i32(3), token_seq=i32(3), block_table=i32((1, 3)), turns=torch.zeros(16, dtype=torch.float64),
                q_out=torch.zeros(3, 4 * 32), k_pool=torch.zeros(3, 2, 16, 32, dtype=torch.uint8), v_pool=torch.zeros(3, 2, 16, 32, dtype=torch.uint8),
                nh=4, nkv=2, hd=32, page_size=16, num_pages=3, status=None, k_scale=torch.zeros(3, 2), v_scale=torch.zeros(3, 2))
    for name, bad, what in [("positions", i32(2), "fit"), ("token_seq", i32(4), "fit"), ("q_out", torch.zeros(2, 4 * 32), "fit"),
                            ("turns", torch.zeros(17, dtype=torch.float64), "fit"), ("num_pages", 4, "pages"),
                            ("v_pool", torch.zeros(2, 2, 16, 32, dtype=torch.uint8), "pages"), ("v_scale", torch.zeros(2, 2), "scales"),
                            ("k_pool", torch.zeros(3, 2, 16, 32), "uint8")]:
        with pytest.raises(KernelError, match=what):
            ops_cache8.ops.rope_append(**dict(good, **{name: bad}))


def test_bands_keep_the_fast_and_slow_the_slow():
    from glint_b200.parts.positions import scaled_frequencies
    got, amplitude = scaled_frequencies(FREQ, {"kind": "bands", "factor": 8.0, "original_context": 4096}, 10000.0, 64)
    assert amplitude == 1.0
    for f, g in zip(FREQ, got):
        turns = 4096 * f / (2 * math.pi)
        want = f if turns >= 4 else f / 8 if turns <= 1 else ((turns - 1) / 3) * f + (1 - (turns - 1) / 3) * f / 8
        assert abs(g - want) <= 1e-15 * f * 8


def test_yarn_ramp_and_amplitude():
    from glint_b200.parts.positions import scaled_frequencies
    got, amplitude = scaled_frequencies(FREQ, {"kind": "yarn", "factor": 4.0, "original_context": 2048}, 10000.0, 64)
    assert abs(amplitude - (0.1 * math.log(4.0) + 1.0)) < 1e-15
    ratio = got / FREQ
    assert ratio[0] == 1.0 and abs(ratio[-1] - 0.25) < 1e-15 and np.all(np.diff(ratio) <= 0)
    turns = 2048 * FREQ / (2 * math.pi)
    assert np.all(ratio[turns > 40] == 1.0) and np.all(np.abs(ratio[turns < 0.7] - 0.25) < 1e-15)
    _, named = scaled_frequencies(FREQ, {"kind": "yarn", "factor": 4.0, "original_context": 2048, "amplitude": 1.0}, 1e4, 64)
    assert named == 1.0


@pytest.mark.parametrize("bad", [{"kind": "none", "factor": 2, "original_context": 10}, {"factor": 2, "original_context": 10},
                                 {"kind": "bands", "factor": 0.5, "original_context": 10},
                                 {"kind": "bands", "factor": 2, "original_context": 0},
                                 {"kind": "bands", "factor": 2, "original_context": 10, "low": 4, "high": 4},
                                 {"kind": "yarn", "factor": 2, "original_context": 10, "beta_fast": 1, "beta_slow": 2}])
def test_scalings_that_are_refused(bad):
    from glint_b200.parts.positions import scaled_frequencies
    with pytest.raises(ConfigError):
        scaled_frequencies(FREQ, bad, 10000.0, 64)


def test_rotary_part_refuses_a_layout_it_does_not_know():
    from glint_b200.parts.positions import Rotary
    from glint_b200.weights.random_init import MetaRuntime
    part = Rotary(MetaRuntime(), {"head_dim": 64, "theta": 1e4, "layout": "interleaved"}, {})
    assert part.only and part.rope.interleaved == 1 and part.rope.rotary_dim == 64
    assert not Rotary(MetaRuntime(), {"head_dim": 64, "theta": 1e4}, {}).only
    with pytest.raises(ConfigError, match="layout"):
        Rotary(MetaRuntime(), {"head_dim": 64, "theta": 1e4, "layout": "twisted"}, {})
