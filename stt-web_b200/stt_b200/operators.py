"""Decode operators that stand beside the model, over device tensors: the 8-bit K/V cache with its
attention, and beam search's selection and reordering.

Tensors are CUDA tensors of any library whose objects have torch's ``data_ptr()``, ``shape``,
``stride()``, ``dtype`` and ``get_device()`` (torch itself is not imported).  Calls are queued on ``stream`` (the integer
handle of a CUDA stream, 0 = the legacy default stream) and do not wait for the device; the tensors must
stay alive until it has run them.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

from ._lib import (BEAM_STATES, BEAM_STEP, KV8_BATCH, KV8_TENSOR, STT_E_INVALID_ARG, SttError, check, lib,
                   stt_kv8_cache_info)

_NAMES = {"torch.float32": 0, "torch.bfloat16": 1, "torch.float16": 2, "torch.int32": 3, "torch.uint8": 4}
_F32, _I32, _U8 = 0, 3, 4
_codes = {}  # the same by dtype object: these checks are a good part of a small call's time


def _code(dtype) -> int:
    code = _codes.get(dtype)
    if code is None:
        code = _codes[dtype] = _NAMES.get(str(dtype), -1)
    return code


def _refuse(where: str, why: str):
    raise SttError(STT_E_INVALID_ARG, where, why)


def _dtype(t, where: str) -> int:
    code = _code(t.dtype)
    if not 0 <= code <= 2:
        _refuse(where, f"dtype {t.dtype} unknown: f32, bf16 and f16 are")
    return code


def _on(t, device: int, where: str):
    if t.get_device() != device:  # -1 off the GPUs
        _refuse(where, f"a tensor is on {t.device}, the operator on cuda:{device}")


def _whole(t, n: int, device: int, where: str, what: str, code: int = _I32) -> int:
    """Address of a contiguous device array of n entries."""
    if _codes.get(t.dtype) == code and t.numel() == n and t.is_contiguous() and t.get_device() == device:
        return t.data_ptr()
    if _code(t.dtype) != code or t.numel() != n or not t.is_contiguous():
        _refuse(where, f"{what} must be {n} contiguous {('f32', '', '', 'int32', 'uint8')[code]} values")
    _on(t, device, where)
    return t.data_ptr()


# places of a call's batch and its two tensors among the packed arguments
_A = KV8_BATCH.size
_B = _A + KV8_TENSOR.size


class Kv8Cache:
    """K and V of ``n_seqs`` sequences as signed bytes with a power-of-two scale for each block of 16
    tokens and head (stt_kv8_* of include/stt_b200.h).  ``memory``: a device tensor of ``bytes()``
    bytes that holds the cache, or None for memory of the library's own.  Calls on one cache must not
    overlap in time."""

    def __init__(self, n_seqs: int, n_kv_heads: int, head_dim: int, capacity: int, device: int = 0, memory=None):
        self._h = None
        need = self.bytes(n_seqs, n_kv_heads, head_dim, capacity)
        where = "stt_kv8_cache_create"
        if memory is not None:
            _on(memory, device, where)
            if not memory.is_contiguous() or memory.numel() * memory.element_size() < need:
                _refuse(where, f"the memory must be contiguous and hold {need} bytes")
        h = C.c_void_p()
        check(lib().stt_kv8_cache_create(device, n_seqs, n_kv_heads, head_dim, capacity,
                                         memory.data_ptr() if memory is not None else None, C.byref(h)), where)
        self._h = h
        self.memory = memory
        self._prepare()
        self.n_seqs, self.n_kv_heads, self.head_dim, self.capacity, self.device = n_seqs, n_kv_heads, head_dim, capacity, device

    def _prepare(self) -> None:
        L = lib()
        self._append, self._read, self._attention = L.stt_kv8_append_device, L.stt_kv8_read_device, L.stt_kv8_attention_device
        self._args = C.create_string_buffer(_B + KV8_TENSOR.size)
        self._at = C.addressof(self._args)

    @staticmethod
    def bytes(n_seqs: int, n_kv_heads: int, head_dim: int, capacity: int) -> int:
        out = C.c_size_t()
        check(lib().stt_kv8_cache_bytes(n_seqs, n_kv_heads, head_dim, capacity, C.byref(out)), "stt_kv8_cache_bytes")
        return out.value

    def close(self) -> None:
        if self._h:
            lib().stt_kv8_cache_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def info(self) -> stt_kv8_cache_info:
        o = stt_kv8_cache_info()
        check(lib().stt_kv8_cache_get_info(self._h, C.byref(o)), "stt_kv8_cache_get_info")
        return o

    def status(self) -> None:
        """Waits for the device; raises SttError for what the calls since the last check reported."""
        check(lib().stt_kv8_cache_status(self._h), "stt_kv8_cache_status")

    def _tensor(self, t, at: int, where: str, heads: int = 0):
        """Packs tensor t into place `at` of the call's arguments; returns (n, tokens, heads)."""
        shape, strides = t.shape, t.stride()
        if len(shape) == 4 and shape[3] == self.head_dim and strides[3] == 1 and (not heads or shape[2] == heads):
            code = _codes.get(t.dtype, -1)
            if not 0 <= code <= 2:
                code = _dtype(t, where)
            if t.get_device() != self.device:
                _on(t, self.device, where)
            KV8_TENSOR.pack_into(self._args, at, t.data_ptr(), strides[0], strides[1], strides[2], code, 0)
            return shape[:3]
        _refuse(where, f"tensors are [n, tokens, {heads or 'heads'}, {self.head_dim}] with the last dimension contiguous, got "
                       f"{tuple(shape)} with strides {tuple(strides)}")

    def _batch(self, n: int, tokens: int, pos, count, seqs, where: str):
        d = self.device
        KV8_BATCH.pack_into(self._args, 0, 0 if seqs is None else _whole(seqs, n, d, where, "seqs"),
                            _whole(pos, n, d, where, "pos"), 0 if count is None else _whole(count, n, d, where, "count"), n, tokens)

    def append(self, k, v, pos, count=None, seqs=None, stream: int = 0) -> None:
        """Writes k and v [n, tokens, n_kv_heads, head_dim]: row i's count[i] tokens (None: all) at the
        positions pos[i] on of sequence seqs[i] (None: i)."""
        where = "stt_kv8_append_device"
        shape = self._tensor(k, _A, where, self.n_kv_heads)
        if self._tensor(v, _B, where, self.n_kv_heads) != shape:
            _refuse(where, f"k is {tuple(k.shape)}, v {tuple(v.shape)}")
        self._batch(shape[0], shape[1], pos, count, seqs, where)
        at = self._at
        code = self._append(self._h, at, at + _A, at + _B, stream)
        if code:
            check(code, where)

    def read(self, k, v, pos, count=None, seqs=None, stream: int = 0) -> None:
        """Reads the values of a range of tokens into k and v [n, tokens, n_kv_heads, head_dim]."""
        where = "stt_kv8_read_device"
        shape = self._tensor(k, _A, where, self.n_kv_heads)
        if self._tensor(v, _B, where, self.n_kv_heads) != shape:
            _refuse(where, f"k is {tuple(k.shape)}, v {tuple(v.shape)}")
        self._batch(shape[0], shape[1], pos, count, seqs, where)
        at = self._at
        code = self._read(self._h, at, at + _A, at + _B, stream)
        if code:
            check(code, where)

    def attention(self, q, out, pos, count=None, seqs=None, start=None, window: int = 0, scale: Optional[float] = None,
                  stream: int = 0) -> None:
        """Causal attention of q [n, tokens, heads, head_dim], whose K and V an append with the same
        pos, count and seqs has written, into ``out`` of the same shape (any of the dtypes).
        scale None: 1 / sqrt(head_dim)."""
        where = "stt_kv8_attention_device"
        shape = self._tensor(q, _A, where)
        if self._tensor(out, _B, where) != shape:
            _refuse(where, f"q is {tuple(q.shape)}, out {tuple(out.shape)}")
        n, tokens, heads = shape
        self._batch(n, tokens, pos, count, seqs, where)
        at = self._at
        code = self._attention(self._h, at, at + _A, heads,
                               None if start is None else _whole(start, n, self.device, where, "start"), window,
                               1.0 / math.sqrt(self.head_dim) if scale is None else scale, at + _B, stream)
        if code:
            check(code, where)

    def reorder(self, parents, held=None, stream: int = 0) -> None:
        """Sequence g * beams + b becomes what sequence g * beams + parents[g, b] was, in place;
        ``held`` [groups, beams]: positions that each sequence's new contents have (None: the whole ring)."""
        where = "stt_kv8_reorder_device"
        if len(parents.shape) != 2:
            _refuse(where, "parents must be [groups, beams]")
        g, b = parents.shape
        d = self.device
        check(lib().stt_kv8_reorder_device(self._h, _whole(parents, g * b, d, where, "parents"), g, b,
                                           None if held is None else _whole(held, g * b, d, where, "held"), stream), where)


class BeamSelector:
    """Beam search's selection (stt_beam_select_device), with workspace for up to ``max_batch``
    utterances, ``max_beams`` (at most 32) beams and ``max_vocab`` tokens.  Calls on one selector must
    not overlap in time."""

    def __init__(self, max_batch: int, max_beams: int, max_vocab: int, device: int = 0):
        self._h = None
        h = C.c_void_p()
        check(lib().stt_beam_create(device, max_batch, max_beams, max_vocab, C.byref(h)), "stt_beam_create")
        self._h = h
        self.device = device
        self._prepare()

    def _prepare(self) -> None:
        self._select = lib().stt_beam_select_device
        self._args = C.create_string_buffer(BEAM_STEP.size)
        self._at = C.addressof(self._args)

    def close(self) -> None:
        if self._h:
            lib().stt_beam_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def status(self) -> None:
        """Waits for the device; raises SttError if a beam had a NaN or +inf logit or score."""
        check(lib().stt_beam_status(self._h), "stt_beam_status")

    def select(self, logits, scores, next_scores, parents, tokens, done=None, next_done=None, eos: int = -1,
               stream: int = 0) -> None:
        """logits [batch * beams, vocab] (rows may be strided), scores f32 [batch, beams]; writes the
        best ``beams`` continuations of each utterance, best first: next_scores (f32), parents and
        tokens (int32), next_done (uint8, may be None).  done (uint8): beams that ended, whose only
        continuation is ``eos``."""
        where = "stt_beam_select_device"
        if len(logits.shape) != 2 or len(scores.shape) != 2:
            _refuse(where, "logits must be [batch * beams, vocab] and scores [batch, beams]")
        rows, vocab = logits.shape
        batch, beams = scores.shape
        stride = logits.stride()
        if rows != batch * beams or (stride[1] != 1 and vocab > 1):
            _refuse(where, f"logits {tuple(logits.shape)} with strides {tuple(stride)} for {batch} x {beams} beams")
        d = self.device
        _on(logits, d, where)
        BEAM_STEP.pack_into(
            self._args, 0, logits.data_ptr(), stride[0] if rows > 1 else vocab, _dtype(logits, where), batch, beams, vocab,
            _whole(scores, rows, d, where, "scores", _F32), 0 if done is None else _whole(done, rows, d, where, "done", _U8),
            _whole(next_scores, rows, d, where, "next_scores", _F32), _whole(parents, rows, d, where, "parents"),
            _whole(tokens, rows, d, where, "tokens"),
            0 if next_done is None else _whole(next_done, rows, d, where, "next_done", _U8), eos, 0)
        code = self._select(self._h, self._at, stream)
        if code:
            check(code, where)


def beam_reorder(states, parents, held=None, stream: int = 0) -> None:
    """Row g * beams + b of ``states`` [groups * beams, segments, units, ...] becomes what row
    g * beams + parents[g, b] was, in place.  ``held`` [groups, beams]: the first units of each segment
    that count (None: all); the rest stays.  Everything behind the first two dimensions is contiguous."""
    where = "stt_beam_reorder_device"
    shape, stride = states.shape, states.stride()
    if len(parents.shape) != 2 or len(shape) < 3:
        _refuse(where, "states must be [groups * beams, segments, units, ...] and parents [groups, beams]")
    groups, beams = parents.shape
    inner = 1
    for size, step in zip(reversed(shape[2:]), reversed(stride[2:])):
        if size > 1 and step != inner:
            _refuse(where, f"states of strides {tuple(stride)} are not contiguous behind the segments")
        inner *= size
    if shape[0] != groups * beams or 0 in shape:
        _refuse(where, f"states {tuple(shape)} for {groups} x {beams} beams")
    size = states.element_size()
    d = states.get_device()
    if d < 0:
        _refuse(where, f"the states are on {states.device}")
    n = groups * beams
    args = BEAM_STATES.pack(states.data_ptr(), stride[0] * size, stride[1] * size, shape[2], inner // shape[2] * size,
                            _whole(parents, n, d, where, "parents"), 0 if held is None else _whole(held, n, d, where, "held"),
                            shape[1], groups, beams, 0)
    check(lib().stt_beam_reorder_device(d, args, stream), where)
