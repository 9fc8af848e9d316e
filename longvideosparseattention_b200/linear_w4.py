"""Linear layers with 4-bit weights and a scale for each group of columns, for
few rows: the Linears whose time is that of reading their weights.

In a diffusion transformer these are the ones that the time embedding passes
through, with one row a sequence or a latent frame: the shift, scale and gate
vectors (``block_norm``) come from a Linear of SiLU(embedding), one in every
block of the HunyuanVideo and CogVideoX models, whose weights are a large part
of the model, one a step in Wan, whose blocks add a table of their own.  An
addition of this package: the reference leaves them to the model.

    w = quantize_w4(block.modulation.weight)               # once
    shift, scale, gate = linear_w4(temb, w, bias, "silu").chunk(3, dim=-1)

W[n, k] is approximated by scale[n, k // group] * code[n, k], codes -8 .. 7;
``pack_w4`` takes codes and scales of another quantiser; codes are signed, about
zero (a checkpoint with zero points has no form here).
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from . import _native as N
from ._launch import W4_LINEAR, dual_level, launch, refuse_tangents

_DT = {torch.bfloat16: N.LVSA_DTYPE_BF16, torch.float16: N.LVSA_DTYPE_F16, torch.float32: N.LVSA_DTYPE_F32}
_ACT = {None: N.LVSA_W4_ACT_NONE, "silu": N.LVSA_W4_ACT_SILU}
GROUPS = (32, 64, 128)


@dataclass(frozen=True)
class W4Weight:
    """A [n, k] weight laid out for ``linear_w4`` (made by ``pack_w4``): the
    kernel reads ``tiles`` and ``scales`` by n, k and group, which have to fit.
    Its tensors may be kept and moved like others and put together again."""

    n: int
    k: int
    group: int
    tiles: torch.Tensor   # uint8
    scales: torch.Tensor  # bf16 / fp16

    def __post_init__(self):
        if self.group not in GROUPS or self.n < 1 or self.k < 1:
            raise ValueError(f"W4Weight: [{self.n}, {self.k}] in groups of {self.group}: sizes from 1 and groups of {GROUPS} expected")
        if self.tiles.dtype != torch.uint8 or self.scales.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"W4Weight: uint8 tiles and bf16 / fp16 scales expected, got {self.tiles.dtype} and {self.scales.dtype}")
        tiles = -(-self.n // 16) * -(-self.k // 64)
        want = (tiles * 512, tiles * 16 * max(1, 64 // self.group))
        if (self.tiles.numel(), self.scales.numel()) != want or not (self.tiles.is_contiguous() and self.scales.is_contiguous()):
            raise ValueError(f"W4Weight: [{self.n}, {self.k}] in groups of {self.group} has {want[0]} bytes of tiles and "
                             f"{want[1]} scales, contiguous; got {self.tiles.numel()} and {self.scales.numel()}")
        if self.tiles.device != self.scales.device:
            raise ValueError(f"W4Weight: tiles on {self.tiles.device}, scales on {self.scales.device}")

    @property
    def device(self) -> torch.device:
        return self.tiles.device


def pack_w4(codes: torch.Tensor, scales: torch.Tensor, group: int) -> W4Weight:
    """Lay out codes [n, k] (int8, -8 .. 7) with scales [n, ceil(k / group)]
    (bf16 / fp16; group 32, 64 or 128).  Codes out of range are not looked
    for: their low four bits count."""
    if not codes.is_cuda:
        raise RuntimeError("pack_w4 needs CUDA tensors (no CPU fallback)")
    if codes.dtype != torch.int8 or scales.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"pack_w4: int8 codes and bf16 / fp16 scales expected, got {codes.dtype} and {scales.dtype}")
    if group not in GROUPS:
        raise ValueError(f"pack_w4: group must be one of {GROUPS}, got {group}")
    if codes.dim() != 2 or codes.shape[0] < 1 or codes.shape[1] < 1:
        raise ValueError(f"pack_w4: codes must be [n, k], got {tuple(codes.shape)}")
    n, k = codes.shape
    if scales.device != codes.device or tuple(scales.shape) != (n, -(-k // group)):
        raise ValueError(f"pack_w4: scales must be [{n}, {-(-k // group)}] on {codes.device}, got "
                         f"{tuple(scales.shape)} on {scales.device}")
    if (codes.stride(1) != 1 and k > 1) or (codes.stride(0) < k and n > 1):
        codes = codes.contiguous()
    lib, size = N.load(), ctypes.c_int64()
    N.check(lib.lvsa_w4_bytes(n, k, ctypes.byref(size)), "lvsa_w4_bytes")
    tiles = torch.empty(size.value, dtype=torch.uint8, device=codes.device)
    with torch.cuda.device(codes.device):
        st = lib.lvsa_w4_pack(codes.data_ptr(), codes.stride(0) if n > 1 else k, n, k, tiles.data_ptr(),
                              torch.cuda.current_stream().cuda_stream)
    N.check(st, "lvsa_w4_pack")
    # Two words a tile of 64 columns for group 32, one otherwise; a word has rows r and r + 8.
    rows, tile = -(-n // 16), max(1, 64 // group)
    s = scales.detach().repeat_interleave(2, dim=1) if group == 128 else scales.detach()
    s = s[:, :-(-k // 64) * tile]
    s = torch.nn.functional.pad(s, (0, -(-k // 64) * tile - s.shape[1], 0, rows * 16 - n))
    s = s.view(rows, 2, 8, -1, tile).permute(0, 3, 2, 4, 1)
    return W4Weight(n, k, group, tiles, s.contiguous())


def quantize_w4(weight: torch.Tensor, group: int = 64, scale_dtype: torch.dtype = torch.bfloat16) -> W4Weight:
    """Round a weight [n, k] to the nearest code -7 .. 7 of its group's scale,
    the largest size in the group over 7.  Refuses a weight with an infinity or
    NaN, or too large for ``scale_dtype`` (so it waits for the device once)."""
    if weight.dim() != 2:
        raise ValueError(f"quantize_w4: weight must be [n, k], got {tuple(weight.shape)}")
    if group not in GROUPS:
        raise ValueError(f"quantize_w4: group must be one of {GROUPS}, got {group}")
    if scale_dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"quantize_w4: scale_dtype must be bf16 or fp16, got {scale_dtype}")
    n, k = weight.shape
    w = torch.nn.functional.pad(weight.detach().float(), (0, -k % group)).unflatten(1, (-1, group))
    scales = (w.abs().amax(-1) / 7).to(scale_dtype)
    if not torch.isfinite(scales).all():  # NaN and infinities of the weight among them
        raise ValueError(f"quantize_w4: weight has values that are not finite, or whose scale passes {scale_dtype}")
    step = scales.float()[..., None]
    codes = torch.where(step > 0, w / step, 0.0).round_().clamp_(-7, 7).to(torch.int8).flatten(1)[:, :k]
    return pack_w4(codes, scales, group)


def linear_w4(x: torch.Tensor, weight: W4Weight, bias: Optional[torch.Tensor] = None,
              activation: Optional[str] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """act(x) W^T + bias: x [..., k] -> [..., n] in ``out_dtype`` (default x's).

    x, bias and output in bf16, fp16 or fp32; ``activation`` None or "silu",
    in fp32.  Values of act(x) count to 2^-22 of the largest of the 64 (32) in
    their group, whatever codes that one meets, or to 2^-128 where that is more;
    SiLU of values below -87 is zero; products with codes are exact
    and sums fp32, with one rounding of the result.  A row with an infinity or NaN
    gives NaN; x may have any finite size, scales any below 2^116.  Made for few
    rows (a row a sequence or a latent frame): each further 21 read the weights
    once more, and 65535 are the most.  Inference only: x must not require grad
    or be a dual tensor."""
    if dual_level():
        refuse_tangents("linear_w4", (x, bias))
    if not x.is_cuda:
        raise RuntimeError("linear_w4 needs CUDA tensors (no CPU fallback)")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if x.dtype not in _DT or out_dtype not in _DT or (bias is not None and bias.dtype not in _DT):
        raise TypeError("linear_w4: x, bias and output in bf16, fp16 or fp32")
    if activation not in _ACT:
        raise ValueError(f"linear_w4: activation must be None or 'silu', got {activation!r}")
    if x.dim() < 1 or x.shape[-1] != weight.k:
        raise ValueError(f"linear_w4: features of x {tuple(x.shape)} do not match weight [{weight.n}, {weight.k}]")
    if weight.tiles.get_device() != x.get_device() or (bias is not None and bias.get_device() != x.get_device()):
        raise ValueError("linear_w4: x, weight and bias must be on one device")
    if bias is not None and tuple(bias.shape) != (weight.n,):
        raise ValueError(f"linear_w4: bias must be [{weight.n}], got {tuple(bias.shape)}")
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
        raise RuntimeError("linear_w4 has no backward: call it under torch.no_grad() or on detached tensors")
    rows = x if x.dim() == 2 else x.reshape(-1, weight.k)
    m = rows.shape[0]
    if (rows.stride(1) != 1 and weight.k > 1) or (rows.stride(0) < weight.k and m > 1):
        rows = rows.contiguous()
    if bias is not None and bias.stride(0) != 1:
        bias = bias.contiguous()
    out = torch.empty(m, weight.n, dtype=out_dtype, device=x.device)
    if m:
        launch("lvsa_w4_linear", W4_LINEAR.pack(
            rows.data_ptr(), weight.tiles.data_ptr(), weight.scales.data_ptr(), 0 if bias is None else bias.data_ptr(),
            out.data_ptr(), rows.stride(0) if m > 1 else weight.k, weight.n, m, weight.n, weight.k, weight.group,
            _DT[x.dtype], _DT[out_dtype], 0 if bias is None else _DT[bias.dtype], _DT[weight.scales.dtype],
            _ACT[activation], 0), x.get_device())
    return out if x.dim() == 2 else out.view(*x.shape[:-1], weight.n)
