"""Keys and values of one layer in 4 bits, and attention over them.

A row is held in groups of 32 columns: the group's smallest value and its step (largest - smallest) / 15, both float16, and a code of
0 .. 15 per column.  128 columns take 80 bytes, 3.2 times less than in bfloat16.  Rows are quantised as they are written; the attention
reads the codes themselves.
"""
from __future__ import annotations

import ctypes as C
import struct

from . import abi
from .abi import check, lib
from .ops import on_device, reorder_states, type_code

GROUP = 32
_strides = struct.Struct("3q").pack     # (of sequence, position and head, as the C entry points take them)
DIMS = (32, 64, 96, 128, 192, 256)


class Cache4:
    """``max_seq`` positions (rounded up to 16) of ``batch`` sequences: ``kv_heads`` heads of ``dim`` columns.

    The caller keeps the sequences' lengths, as for the models' own caches: ``past`` is what they hold before a call, one number for
    all or an int32 tensor [batch] on the device (a captured call reads it anew at every replay; values are kept within the cache).
    Calls are ordered by the current stream."""

    def __init__(self, batch: int, kv_heads: int, max_seq: int, dim: int):
        if batch < 1 or kv_heads < 1 or max_seq < 1 or batch > 65535 or kv_heads > 65535 or max_seq > 1 << 26:
            raise ValueError(f"a cache of {batch} sequences, {kv_heads} heads and {max_seq} positions")
        if dim not in DIMS:
            raise ValueError(f"heads of {dim} columns: {', '.join(map(str, DIMS))} are supported")
        torch = abi.require_cuda()
        self.batch, self.kv_heads, self.dim = batch, kv_heads, dim
        self.max_seq = (max_seq + 15) // 16 * 16
        make = lambda n, t: torch.zeros((batch, kv_heads, self.max_seq, n), dtype=t, device="cuda")
        self.k_codes, self.v_codes = make(dim // 2, torch.uint8), make(dim // 2, torch.uint8)
        self.k_step, self.k_least, self.v_step, self.v_least = (make(dim // GROUP, torch.float16) for _ in range(4))
        self._c = abi.Cache4(batch, kv_heads, self.max_seq, dim, *(t.data_ptr() for t in self._tensors()))
        self._ref = C.byref(self._c)
        self._device = self.k_codes.get_device()

    def _tensors(self):
        return self.k_codes, self.v_codes, self.k_step, self.k_least, self.v_step, self.v_least

    def states(self):
        """For ``ops.reorder_states``: the tensors, each with the axis its positions run along.  Positions lie in tiles of 16: a
        ``length`` given with them has to be rounded up to that (``reorder`` does it)."""
        return [(t, 2) for t in self._tensors()]

    def reorder(self, beams, length=None):
        """``ops.reorder_states`` of this cache: sequence b * width + w becomes what b * width + beams[b, w] was, in its first
        ``length`` positions (all of them unless given)."""
        reorder_states(self.states(), beams, None if length is None else min(-(-length // 16) * 16, self.max_seq))

    def _here(self):
        device, stream = abi.device_and_stream()
        if device != self._device:
            raise ValueError(f"the cache is on {self.k_codes.device}, not on the current CUDA device")
        return device, stream

    def _past(self, past, seq, device):
        """(number, address of the lengths or None), checked."""
        if hasattr(past, "data_ptr"):
            on_device("past", past, device, 1, abi._torch.int32)
            if past.shape[0] != self.batch or not past.is_contiguous():
                raise ValueError(f"past of shape {tuple(past.shape)} for {self.batch} sequences")
            if seq > self.max_seq:
                raise ValueError(f"{seq} positions in a cache of {self.max_seq}")
            return 0, past.data_ptr()
        if past < 0 or past + seq > self.max_seq:
            raise ValueError(f"positions {past} to {past + seq} in a cache of {self.max_seq}")
        return past, None

    def _rows(self, name, x, heads, device):
        """Positions and strides of rows [batch, seq, heads, dim], checked."""
        shape = x.shape
        if x.get_device() != device or len(shape) != 4:
            on_device(name, x, device, 4)
        b, s, h, d = shape
        if b != self.batch or h != heads or d != self.dim:
            raise ValueError(f"{name} of shape {(b, s, h, d)}, expected {(self.batch, 'positions', heads, self.dim)}")
        sb, ss, sh, sd = x.stride()
        if sd != 1:
            raise ValueError(f"the columns of {name} have to lie side by side")
        return s, _strides(sb, ss, sh)

    def append(self, k, v, past):
        """Rows k and v [batch, seq, kv_heads, dim] (float32, bfloat16 or float16, any strides with columns side by side) are quantised
        into the positions from ``past`` on; with a tensor of lengths, positions behind the end of the cache are left out."""
        device, stream = self._here()
        (seq, ks), (v_seq, vs) = self._rows("k", k, self.kv_heads, device), self._rows("v", v, self.kv_heads, device)
        if seq != v_seq or k.dtype is not v.dtype:
            raise ValueError(f"k is {k.dtype} {tuple(k.shape)}, v is {v.dtype} {tuple(v.shape)}")
        code = type_code(k.dtype)
        number, lengths = self._past(past, seq, device)
        if seq:
            status = lib.rotor_b200_cache4_append(self._ref, k.data_ptr(), v.data_ptr(), code, ks, vs, seq, number, lengths, stream)
            if status:
                check(status, "cache4_append")

    def read(self, begin: int, end: int, dtype=None):
        """What positions begin .. end - 1 stand for: keys and values [batch, kv_heads, end - begin, dim] (float32 unless told).
        float16 holds 65504 where a code stands for a little more."""
        _, stream = self._here()
        dtype = dtype or abi._torch.float32
        if not 0 <= begin <= end <= self.max_seq:
            raise ValueError(f"positions {begin} to {end} of a cache of {self.max_seq}")
        code, shape = type_code(dtype), (self.batch, self.kv_heads, end - begin, self.dim)
        k = self.k_step.new_empty(shape, dtype=dtype)
        v = abi._torch.empty_like(k)
        if end > begin:
            status = lib.rotor_b200_cache4_read(self._ref, begin, end, k.data_ptr(), v.data_ptr(), code, stream)
            if status:
                check(status, "cache4_read")
        return k, v

    def attend(self, q, past, *, scale=None, window: int = 0, sinks=None, longest=None):
        """Causal attention of queries [batch, seq, heads, dim] that sit at the positions from ``past`` on (their own keys and values
        appended before) -> the same shape and type.

        Query head h reads KV head h // (heads // kv_heads).  ``scale`` of the scores: 1 / sqrt(dim) unless given.  ``window`` > 0: a
        query sees that many positions, its own included.  ``sinks`` float32 [heads]: exp(sink) joins the softmax's denominator.
        ``longest``: with a tensor of lengths, the most that a sequence holds, by which the work is divided (the cache's size unless
        given); longer lengths are taken as it.  A query that sees no position gives zeros.

        Prompts of 16-bit types run a kernel whose waits are bounded: after a synchronise ``abi.device_status()`` raises where one ran out
        and left outputs unwritten."""
        device, stream = self._here()
        heads = q.shape[2] if q.dim() == 4 else 0
        seq, strides = self._rows("q", q, heads, device)
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"{heads} query heads cannot share {self.kv_heads} key/value heads evenly")
        code = type_code(q.dtype)
        number, lengths = self._past(past, seq, device)
        if window < 0:
            raise ValueError(f"a window of {window} positions")
        if sinks is not None:
            on_device("sinks", sinks, device, 1, abi._torch.float32)
            if sinks.shape[0] != heads or not sinks.is_contiguous():
                raise ValueError("one sink per query head is needed")
            sinks = sinks.data_ptr()
        out = abi._torch.empty_like(q) if q.is_contiguous() else q.new_empty(q.shape)
        if seq == 0:
            return out
        bound = number if lengths is None else self.max_seq if longest is None else min(max(int(longest), 0), self.max_seq)
        scale = self.dim ** -0.5 if scale is None else float(scale)
        call = self._ref, q.data_ptr(), code, strides, heads, seq, number, lengths, bound, scale, window, sinks, out.data_ptr()
        status = lib.rotor_b200_cache4_attend(*call, None, 0, stream)
        if status == abi.ERR_WORKSPACE:      # (nothing has been launched; few tokens need none)
            need = lib.rotor_b200_cache4_attend_workspace_bytes(self._ref, code, heads, seq, bound, window)
            workspace = q.new_empty(need, dtype=abi._torch.uint8)
            status = lib.rotor_b200_cache4_attend(*call, workspace.data_ptr(), need, stream)
        if status:
            check(status, "cache4_attend")
        return out
