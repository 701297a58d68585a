"""One entry point of the library as a Python callable with little host time per call.

A step of a small batch is bound by the host: building a ctypes record and a torch stream object costs more than the
kernel runs. `Launcher` packs the argument record of include/kvip_b200.h from plain values in field order (pointers as
integers, 0 = NULL) and passes it with the raw current stream of a device, which need not be the current device."""
import ctypes
import struct

import torch

from . import _lib

_CODES = {ctypes.c_void_p: "Q", ctypes.c_uint64: "Q", ctypes.c_int64: "q", ctypes.c_uint32: "I", ctypes.c_int32: "i", ctypes.c_float: "f"}


def _public_stream(index):
    return torch.cuda.current_stream(index).cuda_stream


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _public_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


class Launcher:
    def __init__(self, name):
        record = _lib._STAGES[name]
        layout = struct.Struct("".join(_CODES[kind] for _, kind in record._fields_))   # native alignment, as the C compiler's
        if not 0 <= ctypes.sizeof(record) - layout.size < 8:
            raise RuntimeError(f"{name}: the record's layout is not the compiler's")
        self.pack = struct.Struct(layout.format + "x" * (ctypes.sizeof(record) - layout.size)).pack
        self.function = _lib.load_library()[name]      # a function object of its own: the record comes as bytes here
        self.function.argtypes, self.function.restype = [ctypes.c_char_p, ctypes.c_void_p], ctypes.c_uint32
        self.what = name.replace("kvip_b200_", "")

    def __call__(self, index, *values):
        try:
            record = self.pack(*values)
        except struct.error as error:                  # a negative count, a number that its field does not hold
            raise ValueError(f"{self.what}: {error}") from None
        if _current_device() == index:
            code = self.function(record, _raw_stream(index))
        else:
            with torch.cuda.device(index):
                code = self.function(record, _raw_stream(index))
        if code:
            _lib.check(code, self.what)
