"""How the stateless calls of the C ABI are issued for torch tensors: on the tensors' device and, unless a stream is given, on
that device's current stream."""
from __future__ import annotations

import ctypes as C
import threading

from . import _lib

class _Local(threading.local):
    def __init__(self):
        self.message = C.create_string_buffer(256)


_local = _Local()
_calls = None                                # torch's current device and current stream, looked up once


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
