"""Python face of the key/value cache held in 8 bits (csrc/cache8.cu): rotate and append, widen, attend.

A page holds ``page_size`` tokens of one kv head as codes of 8 bits with one scale ``s`` (a power of two), for keys
and for values each: code ``c`` stands for ``(c - 127.5) * s`` and is made by ``floor(x / s) + 128``.  A page's scale
is the smallest that holds its largest magnitude below ``128 s``; when a later token needs a larger one, the codes
before it are shifted, which gives exactly the codes they would have got at once.  So a page depends on its tokens
only, not on how they were cut into steps; a value is off by at most half a step, and is exact in bfloat16.

The calls launch on the current stream of the runtime's device, with the kernels the runtime chooses.  ``Cache8`` and
``StepArrays`` are made once for a layer's pages and a step's arrays and only point at them: what the arrays hold is
read by the kernels.  A ``Cache8`` holds scratch: wide pools for portions, twice the bytes of the codes, and partial results.  The
layers of a model share one (``Cache8.empty(..., like=first)``); with its own each would hold more than pages of bfloat16.  Calls
on one ``Cache8``, or on several that share scratch, belong on one stream, or on streams that wait for each other, graphs among
them.
"""
from __future__ import annotations

import ctypes
from ctypes import c_double, c_float, c_int, c_void_p
from dataclasses import dataclass

import torch

from . import native, ops
from .errors import KernelError

LAYOUTS = {"half": False, "interleaved": True}

_F32, _F64 = torch.float32, torch.float64

_routed = None


def _lib():
    """The core library with the routed operations of the coded cache typed (structures go by address)."""
    global _routed
    if _routed is None:
        lib = native.lib()
        P, I, F = c_void_p, c_int, c_float
        lib.glint_op_rope_append_with.argtypes = [P, P, P, P, P, I, I, I, P, I, I, c_double, P]
        lib.glint_op_cache8_unpack.argtypes = [P, P, P, I, I, I, P]
        lib.glint_op_attention.argtypes = [P, P, P, P, P, I, I, I, F, F, I, P]
        for f in (lib.glint_op_rope_append_with, lib.glint_op_cache8_unpack, lib.glint_op_attention):
            f.restype = c_int
        _routed = lib
    return _routed


@dataclass
class Cache8:
    """One layer's pages: ``k``, ``v`` uint8 [pages, kv heads, page size, head size], ``k_scale``, ``v_scale`` float32
    [pages, kv heads], and ``k_wide``, ``v_wide``, scratch of the codes' shape in the runtime's dtype.  The wide pools
    have to be finite when the cache is made (zeros).  ``scratch``: another cache's, of the same shape; made here unless given."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    k_wide: torch.Tensor
    v_wide: torch.Tensor
    scratch: tuple = None

    def __post_init__(self):
        for name in ("k", "v"):
            ops.require(getattr(self, name), torch.uint8, name)
            ops.require(getattr(self, name + "_scale"), torch.float32, name + "_scale")
            ops.require(getattr(self, name + "_wide"), self.k_wide.dtype, name + "_wide")
        if self.k.dim() != 4 or min(self.k.shape) < 1:
            raise KernelError(f"a coded cache is [pages, kv heads, page size, head size], not {tuple(self.k.shape)}")
        self.num_pages, self.nkv, self.page_size, self.hd = self.k.shape
        for name, shape in (("v", self.k.shape), ("k_scale", self.k.shape[:2]), ("v_scale", self.k.shape[:2]),
                            ("k_wide", self.k.shape), ("v_wide", self.k.shape)):
            if tuple(getattr(self, name).shape) != tuple(shape):
                raise KernelError(f"{name} {tuple(getattr(self, name).shape)} does not fit codes {tuple(self.k.shape)}")
        if self.hd % 2:
            raise KernelError(f"a coded cache takes even head sizes, not {self.hd}")
        if any(t.device != self.k.device for t in (self.v, self.k_scale, self.v_scale, self.k_wide, self.v_wide)):
            raise KernelError("the tensors of a coded cache belong to one device")
        if any(t.data_ptr() % 16 for t in (self.k, self.v, self.k_wide, self.v_wide)):
            raise KernelError("the pools of a coded cache begin at multiples of 16 bytes")
        if self.scratch is None:
            self.scratch = native.cache8_scratch(self.nkv, self.hd, self.k.device)
        partials, arrive = self.scratch
        if any(t.device != self.k.device for t in self.scratch):
            raise KernelError("the tensors of a coded cache belong to one device")
        self.struct = native.ViewStruct(self.k.data_ptr(), self.v.data_ptr(), self.page_size, self.num_pages, 0, 1,
                                        self.k_scale.data_ptr(), self.v_scale.data_ptr(), self.k_wide.data_ptr(),
                                        self.v_wide.data_ptr(), partials.data_ptr(), partials.numel(), arrive.data_ptr(),
                                        arrive.numel())
        self.addr, self.dtype, self.device_index = ctypes.addressof(self.struct), self.k_wide.dtype, self.k.get_device()
        self.device = self.k.device

    @classmethod
    def empty(cls, num_pages, num_kv_heads, page_size, head_dim, dtype=torch.bfloat16, device="cuda:0", like=None):
        """A cache that holds nothing yet.  ``like``: a cache of the same sizes, dtype and device, say another layer's, whose wide
        pools and scratch this one shares."""
        shape = (num_pages, num_kv_heads, page_size, head_dim)
        made = [torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(2)]
        made += [torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in range(2)]
        if like is None:
            return cls(*made, *[torch.zeros(shape, dtype=dtype, device=device) for _ in range(2)])
        if tuple(like.k.shape) != shape or like.dtype != dtype or like.device != made[0].device:
            raise KernelError(f"a cache of {shape} with wide pools of {dtype} on {made[0].device} cannot share those of one of "
                              f"{tuple(like.k.shape)}, {like.dtype} on {like.device}")
        return cls(*made, like.k_wide, like.v_wide, like.scratch)


class StepArrays:
    """The arrays of a step (int32, on the device) for calls that bring their own: ``positions`` and ``token_seq`` per
    token (a request's tokens stand together, in ascending positions; requests in the order of their rows), ``seq_start``
    (tokens cached before the step) and ``cu_seqlens`` (token offsets, one more, the last of them the number of tokens) per
    request, ``block_table`` [requests, pages].  Every token is a request's: a row of padding would be one like the others.
    ``max_seq_len`` is the most tokens of a request, ``max_context`` at least the largest position plus one; ``contexts``:
    the contexts of the requests in front that bring a single token, for planning launches.  A page that a step writes
    belongs to one of its requests; pages that are only read may be several requests'.  ``begin()`` starts a new step: the
    arrays may hold other values, and what was planned for the old ones is not used.  Kernels in front on the stream may write
    them (``positions += 1``), also in a captured graph: the calls read them behind those kernels' end."""

    def __init__(self, positions, token_seq, seq_start, cu_seqlens, block_table, max_seq_len, max_context, contexts=()):
        from .engine.step import _uneven
        named = {"positions": positions, "token_seq": token_seq, "seq_start": seq_start, "cu_seqlens": cu_seqlens,
                 "block_table": block_table}
        for name, t in named.items():
            ops.require(t, torch.int32, name)
            if t.device != positions.device:
                raise KernelError(f"{name} belongs to another device than positions")
        T, R = positions.numel(), seq_start.numel()
        if block_table.dim() != 2 or block_table.shape[0] != R or cu_seqlens.numel() != R + 1 or token_seq.numel() != T:
            raise KernelError(f"step arrays do not fit: {T} positions, {token_seq.numel()} token rows, {R} requests, "
                              f"{cu_seqlens.numel()} offsets, block table {tuple(block_table.shape)}")
        if T and not (1 <= max_seq_len <= T and max_context >= max_seq_len and R >= 1):
            raise KernelError(f"max_seq_len {max_seq_len} and max_context {max_context} do not fit {T} tokens")
        contexts = [int(c) for c in contexts]
        # the requests in front bring a token each; where some bring more, those stand behind
        if len(contexts) > min(R, T) or (contexts and max_seq_len > 1 and len(contexts) == min(R, T)):
            raise KernelError(f"{len(contexts)} contexts of single tokens do not fit {R} requests of {T} tokens, up to {max_seq_len} each")
        if contexts and not 1 <= min(contexts) <= max(contexts) <= max_context:
            raise KernelError(f"contexts from {min(contexts)} to {max(contexts)} do not lie within 1 and {max_context}")
        self.tensors, self.num_tokens, self.device_index = named, T, positions.get_device()
        s = self.struct = native.StepStruct()
        s.num_tokens, s.num_seqs, s.max_seq_len, s.max_context = T, R, int(max_seq_len), int(max_context)
        s.leading_single, s.leading_single_context = (R if max_seq_len == 1 else len(contexts)), max(contexts or [0])
        s.uneven = _uneven(contexts)
        s.num_groups = 1
        s.positions, s.token_seq = positions.data_ptr(), token_seq.data_ptr()
        s.seq_start, s.cu_seqlens = seq_start.data_ptr(), cu_seqlens.data_ptr()
        s.block_table[0], s.max_pages[0] = block_table.data_ptr(), block_table.shape[1]
        self.addr, self.max_context, self.table_pages = ctypes.addressof(s), int(max_context), block_table.shape[1]
        self.begin()

    def begin(self):
        self.struct.id = native.next_step_id()


# A step of a few tokens is bound by the host: the checks below compare what is cheap to read (a fraction of a microsecond
# each) and leave the wording of a refusal to the functions that raise it.


def _check(rt, cache, step, window=0):
    if cache.dtype is not rt.dtype:
        raise KernelError(f"the wide pools are {cache.dtype}, the runtime is {rt.dtype}")
    if not cache.device_index == step.device_index == rt.device_index:
        raise KernelError(f"the cache (device {cache.device_index}), the step ({step.device_index}) and the runtime "
                          f"({rt.device_index}) belong to one device")
    if window < 0:
        raise KernelError(f"a window of {window} tokens")
    if step.max_context > step.table_pages * cache.page_size:
        raise KernelError(f"a context of {step.max_context} exceeds the block table of {step.table_pages} pages of "
                          f"{cache.page_size}")


def _rows(t, rows, width, dtype, name, index):
    if t.dtype is dtype and t.get_device() == index and t.shape == (rows, width) and t.is_contiguous():
        return
    ops.require(t, dtype, name)
    if t.dim() != 2 or tuple(t.shape) != (rows, width):
        raise KernelError(f"{name} {tuple(t.shape)} is not [{rows}, {width}]")
    raise KernelError(f"{name} belongs to device {t.get_device()}, the runtime to {index}")


_current_device = ops._raw_device or torch.cuda.current_device
_current_stream = ops._raw_stream or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(rt, what, fn, *args):
    """One routed operation on the current stream of the runtime's device."""
    index = rt.device_index
    if _current_device() == index:
        rc = fn(*args, _current_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _current_stream(index))
    if rc != 0:
        raise KernelError(f"{what}: {ops.error_string(rc)} (code {rc})")


def _heads(num_heads, cache):
    raise KernelError(f"{num_heads} query heads do not share {cache.nkv} kv heads evenly")


def append(rt, cache, step, qkv, turns, num_heads, q_out=None, layout="half", amplitude=1.0):
    """Rotate the queries and keys of a finished product ``qkv`` float32 [tokens, (heads + 2 kv heads) * head size], write
    the queries to ``q_out`` (made here in the runtime's dtype unless given; returned) and code keys and values into
    their pages.  ``turns`` float64 [pairs]: turns per position of the first ``2 pairs`` dims of a head, which are
    paired (j, j + pairs) in the layout "half" and (2j, 2j + 1) in the layout "interleaved"; the angles are computed
    in 64 bits.  ``amplitude`` scales the turned dims.  A key or value that is not finite makes its page's scale NaN."""
    _check(rt, cache, step)
    if num_heads < 1 or num_heads % cache.nkv:
        _heads(num_heads, cache)
    interleaved = LAYOUTS.get(layout)
    if interleaved is None:
        raise KernelError(f"rotary layout {layout!r} is none of {sorted(LAYOUTS)}")
    T, hd, index = step.num_tokens, cache.hd, rt.device_index
    width = num_heads * hd
    if qkv.dtype is not _F32 or qkv.get_device() != index or qkv.shape != (T, width + 2 * cache.nkv * hd) or not qkv.is_contiguous():
        _rows(qkv, T, width + 2 * cache.nkv * hd, _F32, "qkv", index)
    pairs = turns.numel()
    if turns.dtype is not _F64 or turns.get_device() != index or turns.dim() != 1 or 2 * pairs > hd or not turns.is_contiguous():
        ops.require(turns, torch.float64, "turns")
        raise KernelError(f"turns {tuple(turns.shape)} on device {turns.get_device()} do not fit heads of {hd} on device {index}")
    if q_out is None:
        q_out = torch.empty_strided((T, width), (width, 1), dtype=rt.dtype, device=cache.device)   # the cheapest
    else:
        _rows(q_out, T, width, rt.dtype, "q_out", index)
    _call(rt, "cache8 append", (_routed or _lib()).glint_op_rope_append_with, rt.native_addr, step.addr, qkv.data_ptr(),
          q_out.data_ptr(), cache.addr, num_heads, cache.nkv, hd, turns.data_ptr(), 2 * pairs, interleaved, amplitude)
    return q_out


def unpack(rt, cache, step, window=0):
    """The values of every page that the step's tokens can reach (through ``window``, or all before them), at the same
    places of the wide pools (returned); other places are left as they were."""
    window = window or 0
    _check(rt, cache, step, window)
    _call(rt, "cache8 unpack", (_routed or _lib()).glint_op_cache8_unpack, rt.native_addr, step.addr, cache.addr, cache.nkv,
          cache.hd, window)
    return cache.k_wide, cache.v_wide


def attention(rt, cache, step, q, num_heads, multiplier, softcap=0.0, window=0, out=None):
    """Attention of the step's queries ``q`` [tokens, heads * head size] (the runtime's dtype) over the coded pages, keys
    and values of the step among them: scores times ``multiplier``, soft cap, keys of the last ``window`` positions (0:
    all).  Returns ``out`` [tokens, heads * head size].

    Range in bfloat16: single tokens take whatever the pages hold.  Portions keep their precision for values between 2^-36 and
    2^36 where there is a soft cap of up to 55, and of up to 2^90 without one; sums that overflow are reported by
    ``Runtime.check_status`` (code 7).  Their capped scores are off by up to 2^-11 relative."""
    window = window or 0
    _check(rt, cache, step, window)
    if num_heads < 1 or num_heads % cache.nkv:
        _heads(num_heads, cache)
    T, hd, index = step.num_tokens, cache.hd, rt.device_index
    _rows(q, T, num_heads * hd, rt.dtype, "q", index)
    if out is None:
        out = torch.empty_like(q)
    else:
        _rows(out, T, num_heads * hd, rt.dtype, "out", index)
    _call(rt, "cache8 attention", (_routed or _lib()).glint_op_attention, rt.native_addr, step.addr, q.data_ptr(), cache.addr,
          out.data_ptr(), num_heads, cache.nkv, hd, multiplier, softcap or 0.0, window)
    return out
