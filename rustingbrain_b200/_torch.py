"""How the stateless calls of the C ABI are issued for torch tensors: on the tensors' device and, unless a stream is given, on
that device's current stream.

A stream is given by its number.  What the call reads has to be there for that stream, which is the caller's to see to; what the call returns
is that stream's memory, as if it had been the current one.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import threading

from . import _lib

class _Local(threading.local):
    def __init__(self):
        self.message = C.create_string_buffer(256)


_local = _Local()
_calls = None                                # torch's current device and current stream, looked up once


_no_change = contextlib.nullcontext()


def memory_of(stream, device):
    """Inside it, torch allocates for the given stream (None: for the current one, as always): memory that is let go before the stream has
    written it is then not given out elsewhere."""
    if stream is None:
        return _no_change
    import torch
    return torch.cuda.stream(torch.cuda.ExternalStream(int(stream), device=device))


def issue(fn, tensor, stream, errors, default_error, *args) -> None:
    """``fn(*args, stream, message, message_len)`` with ``tensor``'s device current; raises for a status other than OK."""
    global _calls
    if _calls is None:
        import torch
        _calls = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
    current, raw_stream = _calls
    index = tensor.get_device()
    st = raw_stream(index) if stream is None else int(stream)
    msg = _local.message
    if current() == index:
        rc = fn(*args, st, msg, 256)
    else:
        import torch
        with torch.cuda.device(index):
            rc = fn(*args, st, msg, 256)
    if rc != _lib.OK:
        raise errors.get(rc, default_error)(msg.value.decode(errors="replace"))
