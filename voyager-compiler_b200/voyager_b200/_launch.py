"""Calling a kernel entry point with little host time: a decoding step's calls
take a few microseconds on the device, so the wrapper's own time is the call's."""

import torch

from voyager_b200 import _lib

# the current stream's handle as an integer, without a Stream object (0.1 us
# against 2 us)
raw_stream = torch._C._cuda_getCurrentRawStream
_device = torch._C._cuda_getDevice


def call(fn, index: int, what: str, *args) -> None:
    """``fn(*args, stream)`` on device ``index`` and its current stream; raises
    the status it returns."""
    if _device() == index:
        st = fn(*args, raw_stream(index))
    else:
        with torch.cuda.device(index):
            st = fn(*args, raw_stream(index))
    if st:
        _lib.check(st, what)
