"""Launching small kernels with little time on the host: arguments packed into
bytes in the C structures' layout rather than built as ctypes objects (a
structure of a dozen nested ones takes as long as several launches)."""

from __future__ import annotations

import struct

import torch
from torch.autograd import forward_ad

from . import _native as N

_ROWS, _VECTORS, _NORM = "Pqq", "Pqqii", "ifiiPP"
_FORWARD = _ROWS * 4 + _VECTORS * 3 + _NORM * 2 + "fiiiiiiPP"
BLOCK_NORM = struct.Struct("@" + _FORWARD)
BLOCK_NORM_GRAD = struct.Struct("@" + _FORWARD + _ROWS * 4 + _VECTORS * 3 + "PPPPPq")
W4_LINEAR = struct.Struct("@PPPPPqqiiiiiiiiii")  # the last: the structure's padding

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def dual_level() -> bool:
    """Whether a level of forward-mode differentiation is entered (without one no tensor is dual)."""
    return getattr(forward_ad, "_current_level", 0) >= 0


def refuse_tangents(where: str, tensors) -> None:
    """Raise for a dual tensor of forward-mode differentiation: a kernel called
    on its values would drop its tangent without a word."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{where} has no forward-mode derivative")


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
