"""Which kernels attention over coded pages hands a step's tokens to, with the entry points replaced by recorders: no GPU,
nothing is launched (block tables without pages leave the widening nothing to do)."""
import ctypes
from ctypes import c_float, c_int, c_longlong, c_void_p

import pytest

from glint_b200 import native

P, I, F = c_void_p, c_int, c_float
TABLE, CU = 1 << 20, 1 << 21                        # addresses that nobody follows
SIGNATURES = {                                      # entry: (argument types, places of (table, tokens or requests, offsets))
    "attention_decode8": ([P] * 8 + [I, P] + [I] * 6 + [F, F, I, I, I, P, P, I, P, I, P], (7, 10, None)),
    "attention_decode": ([P] * 6 + [I, P] + [I] * 6 + [F, F, I, I, P, P], (5, 8, None)),
    "attention_portion": ([P] * 6 + [I, P] + [I] * 10 + [F, F, I, I, P, c_longlong, P, I, P], (5, 10, 3)),
    "attention_prefill": ([P] * 6 + [I, P] + [I] * 7 + [F, F, I, P, P], (5, 8, 3)),
    "attention_tcgen05": ([P] * 6 + [I, P] + [I] * 8 + [F, F, I, P, P], (5, 9, 3)),
}


def _lib():
    lib = native.lib()
    lib.glint_op_attention.argtypes = [P, P, P, P, P, I, I, I, F, F, I, P]
    return lib


def _calls(lens, starts, nh, nkv, hd, page, window=0, copied=0):
    """(entry, first request, tokens or requests, whether it counts tokens, its argument before the stream) of every call that
    attention makes."""
    calls, keep = [], []
    rt = native.RuntimeStruct()
    rt.tensor_cores, rt.dtype, rt.sms = 1, 1, 148
    R = len(lens)
    for name, (types, (table, count, offsets)) in SIGNATURES.items():
        def record(*args, name=name, table=table, count=count, offsets=offsets):
            row = 0 if offsets is None else (args[offsets] - CU) // 4
            assert args[table] == TABLE
            calls.append((name, row, args[count], offsets is None, args[-2]))
            return 0
        fn = ctypes.CFUNCTYPE(c_int, *types)(record)
        keep.append(fn)
        setattr(rt.tensor, name, ctypes.cast(fn, c_void_p).value)
    for name, types, result, answer in [
            ("attention_decode8_supported", [I] * 4, c_int, lambda nh, nkv, hd, page: int(hd % 16 == 0 and hd <= 256 and page % 16 == 0)),
            ("attention_decode8_workspace", [I] * 4, c_longlong, lambda *_: 0),
            ("attention_portion_supported", [I] * 4, c_int,
             lambda nh, nkv, hd, page: int(nh // nkv <= 128 and hd % 16 == 0 and hd <= 256 and page in (16, 32, 64)))]:
        fn = ctypes.CFUNCTYPE(result, *types)(answer)
        keep.append(fn)
        setattr(rt.tensor, name, ctypes.cast(fn, c_void_p).value)
    step = native.StepStruct()
    step.num_tokens, step.num_seqs, step.max_seq_len = sum(lens), R, max(lens)
    step.max_context = max(n + s for n, s in zip(lens, starts))
    step.leading_single = next((i for i, n in enumerate(lens) if n != 1), R)
    step.leading_single_context = max([s + 1 for s in starts[:step.leading_single]] or [0])
    step.copied = copied
    step.num_groups, step.cu_seqlens, step.block_table[0], step.max_pages[0] = 1, CU, TABLE, 0
    view = native.ViewStruct()
    view.page_size, view.num_pages = page, 8
    view.k_scale = view.v_scale = view.k_wide = view.v_wide = view.partials = view.arrive = 1 << 22
    view.k = view.v = 1 << 22
    view.partial_floats, view.arrive_ints = 1 << 24, native.CACHE8_ARRIVE
    a = ctypes.addressof
    assert _lib().glint_op_attention(a(rt), a(step), 1 << 22, a(view), 1 << 22, nh, nkv, hd, 1.0, 0.0, window, None) == 0
    return calls


SIZES = [(8, 4, 64, 16), (40, 1, 64, 16), (64, 1, 64, 48), (64, 1, 64, 128), (71, 1, 64, 128), (71, 1, 64, 48), (128, 1, 64, 128),
         (100, 1, 32, 16), (130, 1, 32, 16), (260, 2, 32, 64), (256, 1, 16, 128)]


@pytest.mark.parametrize("nh,nkv,hd,page", SIZES)
@pytest.mark.parametrize("lens,starts", [([1, 1, 40], [30, 200, 50]), ([1] * 12 + [300, 5], [400] * 12 + [0, 3]), ([1, 40, 1], [9, 9, 9]),
                                         ([40], [10]), ([1] * 5, [4, 90, 3, 2, 1]), ([1, 3], [4000, 5000])])
def test_every_token_goes_to_one_kernel_with_its_own_request(nh, nkv, hd, page, lens, starts):
    """Kernels that find a token's request by its row in the step are given all of its tokens, or those in front; kernels that
    count requests, the requests behind.  (Tables here have no columns, a row is 0 bytes: offsets tell the first request.)"""
    calls = _calls(lens, starts, nh, nkv, hd, page)
    owners = [r for r, n in enumerate(lens) for _ in range(n)]
    seen = []
    for name, row, count, by_token, _ in calls:
        if by_token:
            seen += list(range(count))
        else:
            assert row + count == len(lens), name
            seen += [t for t, r in enumerate(owners) if r >= row]
    assert sorted(seen) == list(range(sum(lens))), calls


@pytest.mark.parametrize("lens,starts", [([1, 1, 400], [3000, 2000, 50]), ([1] * 5, [4, 90, 3, 2, 1]), ([400], [0])])
def test_only_copied_arrays_are_read_before_the_wait(lens, starts):
    """A step's arrays may be read under the kernel in front only where no kernel writes them: the engine's, which come by a copy.
    Those of a caller's own are not marked so."""
    for copied in (0, 1):
        calls = _calls(lens, starts, 8, 4, 64, 16, copied=copied)
        assert calls and all(name in ("attention_decode8", "attention_portion") for name, *_ in calls)
        assert [c[-1] for c in calls] == [copied] * len(calls)


def test_who_marks_the_arrays_as_copied(monkeypatch):
    import torch
    from glint_b200 import ops_cache8
    from tests.test_cache8 import _pretend, _step
    _pretend(monkeypatch)
    assert _step().struct.copied == 0
    i = torch.zeros(1, dtype=torch.int32)
    ctx = type("Context", (), dict(num_tokens=1, num_seqs=1, max_seq_len=1, max_context=1, leading_single=1, leading_single_context=1,
                                   num_logit_rows=1, uneven=0, block_tables=[], token_ids=i, positions=i, token_seq=i, seq_slot=i,
                                   seq_start=i, cu_seqlens=i, logit_rows=i))
    assert native.fill_step(native.StepStruct(), ctx, 1).copied == 1
