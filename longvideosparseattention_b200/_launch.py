"""Launching small kernels with little time on the host: arguments packed into
bytes in the C structures' layout rather than built as ctypes objects (a
structure of a dozen nested ones takes as long as several launches)."""

from __future__ import annotations

import struct

import torch

from . import _native as N

_ROWS, _VECTORS, _NORM = "Pqq", "Pqqii", "ifiiPP"
_FORWARD = _ROWS * 4 + _VECTORS * 3 + _NORM * 2 + "fiiiiiiPP"
BLOCK_NORM = struct.Struct("@" + _FORWARD)
BLOCK_NORM_GRAD = struct.Struct("@" + _FORWARD + _ROWS * 4 + _VECTORS * 3 + "PPPPPq")
W4_LINEAR = struct.Struct("@PPPPPqqiiiiiiiiii")  # the last: the structure's padding

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def launch(name: str, args, index: int) -> None:
    """Call the library's ``name`` on torch's current stream of device ``index``."""
    fn = getattr(N.load(), name)
    if index == torch.cuda.current_device():
        st = fn(args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            st = fn(args, _raw_stream(index))
    if st:
        N.check(st, name)
