"""How the stateless calls of the C ABI are issued for torch tensors: on the tensors' device and, unless a stream is given, on
that device's current stream."""
from __future__ import annotations

import ctypes as C
import threading

from . import _lib

_local = threading.local()


def _message():
    m = getattr(_local, "message", None)
    if m is None:
        m = _local.message = C.create_string_buffer(256)
    return m


def issue(fn, tensor, stream, errors, default_error, *args) -> None:
    """``fn(*args, stream, message, message_len)`` with ``tensor``'s device current; raises for a status other than OK."""
    import torch
    index = tensor.get_device()
    st = torch._C._cuda_getCurrentRawStream(index) if stream is None else int(stream)
    msg = _message()
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, st, msg, 256)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, st, msg, 256)
    if rc != _lib.OK:
        raise errors.get(rc, default_error)(msg.value.decode(errors="replace"))
