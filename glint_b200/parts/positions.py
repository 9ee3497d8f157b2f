"""Rotary position encoding, applied where keys enter the cache.

Pair (j, j + rot/2) of a head turns by (pos / factor) * theta^(-2j/head_dim), all in 32-bit
(src/tensor/ops.rs:212-245).  The reference permutes the q/k rows at load and turns adjacent
pairs; that is the same rotation of the same pairs (src/transformer/weights.rs:473-530, test
:626-671), and q.k does not change under a permutation common to both, so the file's row
order is kept here.  Keys are cached after the rotation (src/transformer/forward.rs:569-572).

Beside that form, ``layout`` "interleaved" turns the pairs (2j, 2j + 1), ``rotary_dim`` a part of the head, and
``scaling`` changes the frequencies for contexts beyond those a model was trained on (``scaled_frequencies``).
"""
from __future__ import annotations

import numpy as np
import torch

from .. import ops
from ..errors import ConfigError
from ..native import TrigTable, rope_struct
from .base import Part
from .registry import register_part


def scaled_frequencies(freq, scaling, theta, head_dim):
    """(frequencies, amplitude) of a rotary encoding whose contexts are ``scaling["factor"]`` times longer than the
    ``scaling["original_context"]`` tokens a model was trained on.  Slow pairs turn ``factor`` times slower, fast pairs as
    before; the kinds differ in the ramp between them:

    * "bands": by the turns n = original_context * freq / 2 pi that a pair makes over the original context: all slow
      up to ``low`` turns (default 1), as before from ``high`` (default 4), linear in n between;
    * "yarn": linear in the pair's index, between the indices that make ``beta_fast`` (default 32) and ``beta_slow``
      (default 1) turns; the turned dims are scaled by ``amplitude`` (default 0.1 ln(factor) + 1).
    """
    kind = scaling.get("kind")
    factor, context = float(scaling["factor"]), float(scaling["original_context"])
    if not (factor >= 1.0 and context > 0.0):
        raise ConfigError(f"rotary scaling wants a factor of at least 1 and a positive original context, not {scaling}")
    freq = np.asarray(freq, dtype=np.float64)
    if kind == "bands":
        low, high = float(scaling.get("low", 1.0)), float(scaling.get("high", 4.0))
        if not 0.0 < low < high:
            raise ConfigError(f"rotary scaling by bands wants 0 < low < high, not {low} and {high}")
        keep = np.clip((context * freq / (2.0 * np.pi) - low) / (high - low), 0.0, 1.0)
        amplitude = float(scaling.get("amplitude", 1.0))
    elif kind == "yarn":
        fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
        if not fast > slow > 0.0:
            raise ConfigError(f"yarn scaling wants beta_fast > beta_slow > 0, not {fast} and {slow}")
        # the index whose pair makes n turns: freq = theta^(-2j / head_dim) = 2 pi n / context
        index = [head_dim * np.log(context / (2.0 * np.pi * n)) / (2.0 * np.log(theta)) for n in (fast, slow)]
        first, last = max(np.floor(index[0]), 0.0), min(np.ceil(index[1]), head_dim - 1.0)
        j = np.arange(freq.size, dtype=np.float64)
        keep = 1.0 - np.clip((j - first) / max(last - first, 1e-3), 0.0, 1.0)
        amplitude = float(scaling.get("amplitude", 0.1 * np.log(factor) + 1.0))
    else:
        raise ConfigError(f"unknown rotary scaling {kind!r} (known: bands, yarn)")
    return freq * keep + freq / factor * (1.0 - keep), amplitude


class Rotary(Part):
    def __init__(self, rt, params, tensors):
        super().__init__(rt, params, tensors)
        self.head_dim = int(params["head_dim"])
        self.rotary_dim = int(params.get("rotary_dim", self.head_dim)) & ~1
        self.theta = float(params["theta"])
        self.factor = float(params.get("factor", 1.0))
        # freq_j = 1 / theta^(2j / head_dim) in 32-bit, as the reference computes it
        i = np.arange(0, self.rotary_dim, 2, dtype=np.float32)
        inv = np.float32(1.0) / np.power(np.float32(self.theta), i / np.float32(self.head_dim), dtype=np.float32)
        self.layout = params.get("layout", "half")
        if self.layout not in ("half", "interleaved"):
            raise ConfigError(f"unknown rotary layout {self.layout!r} (known: half, interleaved)")
        self.amplitude = 1.0
        freq = inv.astype(np.float64)
        if params.get("scaling"):
            freq, self.amplitude = scaled_frequencies(freq, params["scaling"], self.theta, self.head_dim)
        self.inv_freq = torch.from_numpy(freq.astype(np.float32)).to(rt.device)
        # turns per position, for the kernel that takes every form and computes its angles in 64 bits
        self.turns = torch.from_numpy(freq / self.factor / (2.0 * np.pi)).to(rt.device)
        self.only = self.layout != "half" or self.amplitude != 1.0          # no other kernel has these forms
        self.rope = rope_struct(self.turns, self.layout == "interleaved", self.amplitude, self.only)

    def lower(self, prog, x, w_qkv, q_out, view, nh, nkv, hd):
        """The q/k/v product of ``x``, the rotation of q and k, q into ``q_out``, k and v into the pages of
        ``view`` (only q when the view does not write), as one operation: the runtime takes one kernel
        where there is one for these sizes (the weight-streaming product for a few single tokens, the tiled
        product for heads in steps of 256, both with the rotation and the cache write in their epilogue) and
        else the product followed by the rotation kernel (always when the pages of ``view`` are coded)."""
        key = ("rope_table", self.theta, self.factor, self.rotary_dim, self.head_dim, repr(self.params.get("scaling")))
        trig = self.rt.shared.get(key)                # the step's table of angles, shared by all layers with these parameters
        if trig is None:
            trig = self.rt.shared[key] = TrigTable(self.rt, self.rotary_dim // 2)
        trig.reserve(prog.capacity)
        tmp = prog.value("mixer.qkv", w_qkv.shape[0], torch.float32)
        prog.qkv_rope(x, w_qkv, q_out, tmp, view, nh, nkv, hd, self.inv_freq, self.factor, self.rotary_dim, trig, self.rope)

    def encode_and_store(self, qkv, ctx, q_out, view, nh, nkv, hd):
        """Rotate q and k of a finished product ``qkv``; q goes to ``q_out``; k and v go into the pages of
        ``view`` (only q when the view does not write)."""
        writes = view.writes
        coded = getattr(view, "k_scale", None) is not None
        if coded or self.only:
            ops.rope_append(qkv, ctx.positions, ctx.token_seq, ctx.block_table(view.group), self.turns, q_out,
                            view.k if writes else None, view.v if writes else None, nh, nkv, hd, view.page_size,
                            view.num_pages, self.rt.status, view.k_scale if coded and writes else None,
                            view.v_scale if coded and writes else None, self.layout == "interleaved", self.amplitude)
            return
        ops.rope_kv_write(qkv, ctx.positions, ctx.token_seq, ctx.block_table(view.group), self.inv_freq,
                          self.factor, self.rotary_dim, q_out, view.k if writes else None,
                          view.v if writes else None, nh, nkv, hd, view.page_size, view.num_pages,
                          self.rt.status)


register_part("position", "rope", Rotary)
