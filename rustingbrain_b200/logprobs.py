"""Token log probabilities of device logits, with entropy and the most likely tokens, and their gradient: the C ABI of
include/logprobs_b200.h.  Device tensors in, device tensors out; no host implementation behind it.

``TransformerLm.score_batch`` gives the same numbers for the tokens of a batch without the logits leaving the device.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

from . import _lib
from ._torch import issue, memory_of
from .moe import CudaError, InvalidConfig, InvalidInput

MAX_TOP = 32

_ERRORS = {_lib.INVALID_CONFIG: InvalidConfig, _lib.INVALID_INPUT: InvalidInput, _lib.UNSUPPORTED: InvalidConfig}


class TokenLogProbs(NamedTuple):
    """What ``token_logprobs`` returns; every field is f32 [rows] but the alternatives, [rows, top] (None without them)."""
    logprob: "torch.Tensor"                    # log p of the given token; 0 where there is none
    entropy: "torch.Tensor"
    lse: "torch.Tensor"                        # log of the sum of the exponentials, which the gradient takes
    top_ids: Optional["torch.Tensor"]          # int32, the most likely first, the lower id first among equal logits
    top_logprobs: Optional["torch.Tensor"]


_precisions = {}                             # of torch's types


def _check_logits(t, name):
    if not _precisions:
        import torch
        _precisions.update({torch.float32: _lib.PRECISION_F32, torch.bfloat16: _lib.PRECISION_BF16})
    shape, precision = t.shape, _precisions.get(t.dtype)
    if len(shape) != 2 or not t.is_cuda or precision is None:
        raise InvalidInput("%s must be an f32 or bf16 device tensor [rows, vocab]" % name)
    rows, vocab = shape
    apart, step = t.stride()
    if vocab == 0 or (vocab > 1 and step != 1) or (rows > 1 and apart < vocab):
        raise InvalidInput("the logits of a row of %s are adjacent, and rows do not overlap" % name)
    return rows, vocab, apart if apart > vocab else vocab, precision


def _check_row(t, rows, dtype, like, name):
    if t is None:
        return None
    if t.dtype != dtype or t.shape != (rows,) or t.get_device() != like.get_device() or not t.is_contiguous():
        raise InvalidInput("%s must be a contiguous %s tensor of %d values on the logits' device" % (name, dtype, rows))
    return t.data_ptr()


def token_logprobs(logits, targets=None, top: int = 0, stream=None) -> TokenLogProbs:
    """``logits`` [rows, vocab], f32 or bf16, rows any distance apart; ``targets`` int32 [rows], negative for "no token" (None: no row
    has one); ``top`` alternatives per row, at most 32 and at most vocab."""
    import torch
    rows, vocab, stride, precision = _check_logits(logits, "logits")
    t = _check_row(targets, rows, torch.int32, logits, "targets")
    if not 0 <= top <= min(vocab, MAX_TOP):
        raise InvalidInput("top is 0 .. %d, got %d" % (min(vocab, MAX_TOP), top))
    ids = tlp = None
    with memory_of(stream, logits.device):
        lp = logits.new_empty(rows, dtype=torch.float32)
        h, lse = torch.empty_like(lp), torch.empty_like(lp)
        if top:
            ids = logits.new_empty((rows, top), dtype=torch.int32)
            tlp = lp.new_empty((rows, top))
    issue(_lib.lib().logprobs_forward, logits, stream, _ERRORS, CudaError, logits.data_ptr(), stride, t, rows, vocab, top, precision,
          lp.data_ptr(), h.data_ptr(), lse.data_ptr(), tlp.data_ptr() if top else None, ids.data_ptr() if top else None)
    return TokenLogProbs(lp, h, lse, ids, tlp)


def token_logprobs_backward(logits, targets, lse, entropy=None, grad_logprob=None, grad_entropy=None, out=None, stream=None):
    """dL/dlogits from dL/dlogprob and dL/dentropy [rows] (either may be None).  ``lse`` and ``entropy`` are the forward call's; ``out``
    (default: a new tensor) has the logits' shape and type and may be ``logits`` itself."""
    import torch
    rows, vocab, stride, precision = _check_logits(logits, "logits")
    if out is None:
        with memory_of(stream, logits.device):
            out, out_stride = logits.new_empty((rows, vocab)), vocab
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise InvalidInput("out must match the logits")
    else:
        _, _, out_stride, _ = _check_logits(out, "out")
    if lse is None or (grad_entropy is not None and entropy is None):
        raise InvalidInput("the gradient needs lse, and the entropy for a gradient of it")
    f32 = torch.float32
    issue(_lib.lib().logprobs_backward, logits, stream, _ERRORS, CudaError, logits.data_ptr(), stride,
          _check_row(targets, rows, torch.int32, logits, "targets"), _check_row(lse, rows, f32, logits, "lse"),
          _check_row(entropy, rows, f32, logits, "entropy"), _check_row(grad_logprob, rows, f32, logits, "grad_logprob"),
          _check_row(grad_entropy, rows, f32, logits, "grad_entropy"), rows, vocab, precision, out.data_ptr(), out_stride)
    return out


__all__ = ["TokenLogProbs", "token_logprobs", "token_logprobs_backward", "MAX_TOP"]
