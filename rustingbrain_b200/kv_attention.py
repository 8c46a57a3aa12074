"""Host-side mirror of the reference's ``KvCache`` + ``MultiHeadAttention::forward_cached``
(attention.rs:19-78, 344-398) over the C ABI of include/kv_attention_b200.h, for many sequences.

The projections (query, key, value, output) stay with the caller; this object owns the caches and the
attention arithmetic between them.  There is no host implementation behind it.
"""
from __future__ import annotations

import ctypes as C
from typing import List, Optional

import numpy as np

from . import _lib
from ._torch import memory_of
from .moe import CudaError, InvalidConfig, InvalidInput, NetworkError

_ERRORS = {_lib.INVALID_CONFIG: InvalidConfig, _lib.INVALID_INPUT: InvalidInput, _lib.UNSUPPORTED: InvalidConfig}
_PRECISIONS = {"f32": _lib.PRECISION_F32, "bf16": _lib.PRECISION_BF16, "q4": _lib.PRECISION_Q4}


class KvCache:
    """``sequences`` caches of ``capacity`` positions (KvCache::with_capacity, attention.rs:39-48) and the
    RoPE tables for ``max_seq_len`` positions (Rope::new, rope.rs:71-97).

    ``precision`` is the type of the activations and of the cache, "f32" or "bf16"; "q4" keeps the cache in 4 bits with a step and a base
    per 32 channels of a head (bf16 activations, head_dim 32, 64, 128 or 256): a third of the bytes of a bf16 cache.

    Every call takes a ``stream`` (its number; None: the current one of the cache's device).  Calls on one cache follow one another, on one stream or
    ordered by the caller."""

    def __init__(self, sequences: int, num_heads: int, kv_heads: int, head_dim: int, capacity: int,
                 max_seq_len: Optional[int] = None, rope_base: float = 10000.0, rope: bool = True,
                 precision: str = "bf16", device: int = 0):
        if precision not in _PRECISIONS:
            raise InvalidConfig("precision is 'f32', 'bf16' or 'q4'")
        self.sequences, self.num_heads, self.kv_heads, self.head_dim = sequences, num_heads, kv_heads, head_dim
        self.capacity = capacity
        self.precision = precision
        self._h = C.c_void_p()
        cfg = _lib.KvCacheConfigC(sequences=sequences, num_heads=num_heads, kv_heads=kv_heads, head_dim=head_dim,
                                  capacity=capacity, max_seq_len=max_seq_len if max_seq_len is not None else capacity,
                                  rope_base=rope_base, rope=1 if rope else 0,
                                  precision=_PRECISIONS[precision], device=device)
        self.device = device
        self._dtype = self._raw_stream = self._f32 = None      # torch's, looked up with the first step
        self._forward = _lib.lib().kv_attention_forward_cached
        rc = _lib.lib().kv_cache_create(C.byref(cfg), C.byref(self._h))
        if rc != _lib.OK:
            text = _lib.lib().kv_cache_last_error(self._h).decode(errors="replace") if self._h else "kv_cache_create failed"
            if self._h:
                _lib.lib().kv_cache_destroy(self._h)
                self._h = C.c_void_p()
            raise _ERRORS.get(rc, CudaError)(text)

    def __del__(self):
        h = getattr(self, "_h", None)
        if h and _lib is not None and _lib.lib is not None:      # both are gone at the interpreter's own end
            _lib.lib().kv_cache_destroy(h)
            self._h = C.c_void_p()

    def _check(self, rc: int) -> None:
        if rc != _lib.OK:
            text = _lib.lib().kv_cache_last_error(self._h).decode(errors="replace")
            raise _ERRORS.get(rc, CudaError)(text)

    # -- KvCache ------------------------------------------------------------------------------------
    def lengths(self, stream=None) -> List[int]:
        """``KvCache::len`` of every sequence."""
        out = (C.c_int32 * self.sequences)()
        self._check(_lib.lib().kv_cache_lengths(self._h, out, self._on(stream)))
        return list(out)

    def clear(self, sequence: int = -1, stream=None) -> None:
        self._check(_lib.lib().kv_cache_clear(self._h, sequence, self._on(stream)))

    def truncate(self, length: int, sequence: int = -1, stream=None) -> None:
        self._check(_lib.lib().kv_cache_truncate(self._h, sequence, length, self._on(stream)))

    def keys_values(self, sequence: int, stream=None):
        """Cached (post-RoPE) keys and values of one sequence as f32 [len, kv_heads * head_dim]."""
        n = self.lengths(stream)[sequence]
        W = self.kv_heads * self.head_dim
        k = np.empty((n, W), np.float32)
        v = np.empty((n, W), np.float32)
        fp = C.POINTER(C.c_float)
        self._check(_lib.lib().kv_cache_read(self._h, sequence, k.ctypes.data_as(fp), v.ctypes.data_as(fp), self._on(stream)))
        return k, v

    # -- forward_cached -----------------------------------------------------------------------------
    def forward_cached(self, q, k, v, rows_per_sequence: int = 1, first_sequence: int = 0,
                       n_sequences: Optional[int] = None, out=None, stream=None):
        """Device tensors q [rows, num_heads * head_dim] (scratch: may be rotated in place), k and v
        [rows, kv_heads * head_dim], rows = n_sequences * rows_per_sequence; returns the merged heads, in ``out`` (of any shape with as many values, q itself too)
        where it is given."""
        n_seq = self.sequences - first_sequence if n_sequences is None else n_sequences
        rows = n_seq * rows_per_sequence
        W = self.kv_heads * self.head_dim
        self._rows(q, rows, self.num_heads * self.head_dim, "q")
        self._rows(k, rows, W, "k")
        self._rows(v, rows, W, "v")
        if out is None:
            with memory_of(stream, q.device):
                out = q.new_empty(q.shape)
        elif not (out.get_device() == self.device and out.is_contiguous() and out.dtype == self._dtype and out.numel() == q.numel()):
            raise InvalidInput("out must be a contiguous %s tensor of %d values on cuda:%d" % (self._dtype, q.numel(), self.device))
        self._check(self._forward(self._h, first_sequence, n_seq, q.data_ptr(), k.data_ptr(), v.data_ptr(), rows_per_sequence,
                                  out.data_ptr(), self._on(stream)))
        return out

    def _rows(self, t, rows, width, name) -> None:
        if self._dtype is None:
            import torch
            self._dtype = torch.float32 if self.precision == "f32" else torch.bfloat16
        if not (t.get_device() == self.device and t.is_contiguous() and t.dtype == self._dtype and t.shape == (rows, width)):
            raise InvalidInput("%s must be a contiguous %s tensor of shape %s on cuda:%d" % (name, self._dtype, (rows, width), self.device))

    def _on(self, stream):
        """The given stream, or the current one of the cache's device."""
        if self._raw_stream is None:
            import torch
            torch.cuda.init()                                  # a cache can be the first thing on the device
            self._raw_stream = torch._C._cuda_getCurrentRawStream
        return self._raw_stream(self.device) if stream is None else int(stream)

    def append(self, k, v, rows_per_sequence: int = 1, first_sequence: int = 0, n_sequences: Optional[int] = None, stream=None) -> None:
        """``KvCache::append`` (attention.rs:65-78): stores new keys (rotated here) and values without attending to anything."""
        n_seq = self.sequences - first_sequence if n_sequences is None else n_sequences
        W = self.kv_heads * self.head_dim
        self._rows(k, n_seq * rows_per_sequence, W, "k")
        self._rows(v, n_seq * rows_per_sequence, W, "v")
        self._check(_lib.lib().kv_cache_append(self._h, first_sequence, n_seq, k.data_ptr(), v.data_ptr(), rows_per_sequence, self._on(stream)))

    def rollback(self, rows_per_sequence: int, first_sequence: int = 0, n_sequences: Optional[int] = None, stream=None) -> None:
        """Takes back the newest rows of every sequence of the range, as after draft tokens that were not accepted."""
        n_seq = self.sequences - first_sequence if n_sequences is None else n_sequences
        self._check(_lib.lib().kv_cache_rollback(self._h, first_sequence, n_seq, rows_per_sequence, self._on(stream)))

    def newest(self, rows_per_sequence: int = 1, first_sequence: int = 0, n_sequences: Optional[int] = None, stream=None):
        """The newest rows of every sequence of the range as the cache holds them: f32 device tensors
        [n_sequences * rows_per_sequence, kv_heads * head_dim], keys (after the rotation) and values."""
        n_seq = self.sequences - first_sequence if n_sequences is None else n_sequences
        shape = (max(n_seq, 0) * max(rows_per_sequence, 0), self.kv_heads * self.head_dim)
        if self._f32 is None:
            import torch
            self._f32 = torch.empty(0, dtype=torch.float32, device=self.device)
        with memory_of(stream, self._f32.device):
            keys, values = self._f32.new_empty(shape), self._f32.new_empty(shape)
        self._check(_lib.lib().kv_cache_newest(self._h, first_sequence, n_seq, rows_per_sequence, keys.data_ptr(), values.data_ptr(), self._on(stream)))
        return keys, values


__all__ = ["KvCache", "NetworkError"]
