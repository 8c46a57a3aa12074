"""``Linear`` of a decode step with 4-bit weights and a bf16 scale per group of input channels, over the C ABI of
include/q4_linear_b200.h.  Device tensors in, device tensors out; no host implementation behind it.

``TransformerLm.new_kv_caches(..., precision="q4")`` keeps the cache in 4 bits; this layer does the same for the projections that a caller
puts around a ``KvCache`` and for an output head.
"""
from __future__ import annotations

from . import _lib
from ._torch import issue, memory_of
from .moe import CudaError, InvalidConfig, InvalidInput

_ERRORS = {_lib.INVALID_CONFIG: InvalidConfig, _lib.INVALID_INPUT: InvalidInput, _lib.UNSUPPORTED: InvalidConfig}


class Q4Linear:
    """``Linear::new(d_in, d_out)`` without a bias; weights start at zero and come from ``set_weight`` (quantised here) or ``set_codes``.

    Every call takes a ``stream`` (its number; None: the current one).  The caller orders calls that set weights against those that read them, and
    what a call reads against its stream."""

    def __init__(self, d_in: int, d_out: int, group_size: int = 32, device: int = 0):
        import torch
        self.d_in, self.d_out, self.group_size = int(d_in), int(d_out), int(group_size)
        size = int(_lib.lib().q4_linear_packed_bytes(self.d_out, self.d_in, self.group_size))
        if size == 0:
            raise InvalidConfig("d_in (%d) is a multiple of the group (%d), which is 32, 64 or 128, and d_out (%d) is positive"
                                % (d_in, group_size, d_out))
        self.packed = torch.zeros(size, dtype=torch.uint8, device="cuda:%d" % device)      # zero scales: a layer of zeros
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(device).synchronize()    # the zeros are there before weights of any stream
        self._dtypes = {torch.bfloat16: _lib.PRECISION_BF16, torch.float32: _lib.PRECISION_F32}
        self._fn = _lib.lib().q4_linear_forward
        self._at, self._index = self.packed.data_ptr(), self.packed.get_device()

    def _same_place(self, t, shape, dtype, name):
        if tuple(t.shape) != shape or t.dtype != dtype or t.device != self.packed.device or not t.is_contiguous():
            raise InvalidInput("%s must be a contiguous %s tensor of shape %s on %s" % (name, dtype, shape, self.packed.device))
        return t.data_ptr()

    def set_weight(self, weight, stream=None) -> None:
        """Quantises ``weight`` [d_out, d_in], a f32 device tensor: scale = bf16(max |w| / 7) of each group."""
        import torch
        at = self._same_place(weight, (self.d_out, self.d_in), torch.float32, "weight")
        issue(_lib.lib().q4_linear_quantize, self.packed, stream, _ERRORS, CudaError, at, self._at, self.d_out, self.d_in, self.group_size)

    def set_codes(self, codes, scales, stream=None) -> None:
        """``codes`` [d_out, d_in] int8 of -8 .. 7 and ``scales`` [d_out, d_in / group_size] bf16, device tensors."""
        import torch
        c = self._same_place(codes, (self.d_out, self.d_in), torch.int8, "codes")
        s = self._same_place(scales, (self.d_out, self.d_in // self.group_size), torch.bfloat16, "scales")
        issue(_lib.lib().q4_linear_pack, self.packed, stream, _ERRORS, CudaError, c, s, self._at, self.d_out, self.d_in, self.group_size)

    def weight(self, stream=None):
        """What the layer stands for: f32 [d_out, d_in]."""
        import torch
        with memory_of(stream, self.packed.device):
            w = torch.empty((self.d_out, self.d_in), dtype=torch.float32, device=self.packed.device)
        issue(_lib.lib().q4_linear_dequantize, self.packed, stream, _ERRORS, CudaError, self._at, w.data_ptr(), self.d_out, self.d_in, self.group_size)
        return w

    def forward(self, x, out=None, stream=None):
        """``x`` [rows, d_in], f32 or bf16, rows on 16-byte boundaries; returns [rows, d_out] of the same type."""
        precision, shape = self._dtypes.get(x.dtype), x.shape
        if precision is None or len(shape) != 2 or shape[1] != self.d_in or x.get_device() != self._index or (self.d_in > 1 and x.stride(1) != 1):
            raise InvalidInput("expected a f32 or bf16 tensor [rows, %d] on %s, the channels of a row adjacent" % (self.d_in, self.packed.device))
        rows = shape[0]
        if out is None:
            with memory_of(stream, x.device):
                out = x.new_empty((rows, self.d_out))
        elif tuple(out.shape) != (rows, self.d_out) or out.dtype != x.dtype or out.device != x.device or (self.d_out > 1 and out.stride(1) != 1):
            raise InvalidInput("out must be [%d, %d], of x's type and on its device" % (rows, self.d_out))
        issue(self._fn, x, stream, _ERRORS, CudaError, x.data_ptr(), x.stride(0) if rows > 1 else self.d_in, self._at, out.data_ptr(),
              out.stride(0) if rows > 1 else self.d_out, rows, self.d_in, self.d_out, self.group_size, precision)
        return out

    __call__ = forward


__all__ = ["Q4Linear"]
