"""The elementwise steps of a transformer block around its attention or MLP:
the norm before the block with its modulation, and the join after it with
gate, residual scale and an optional norm of the branch, in one pass each.

    norm_modulate       n = norm(x) * (1 + scale) + shift
    gate_residual       h = residual_scale * x + gate * post_norm(y)
    gate_residual_norm  h as above and n = norm(h) * (1 + scale) + shift,
                        the join and the next block's norm in one pass

An addition of this package: the reference leaves these steps to the model.
The Wan, HunyuanVideo and CogVideoX blocks run ``norm_modulate`` before
attention and MLP and ``gate_residual`` after each; with sandwich norms the
branch is normalised first (``post_norm``).

Tensors: ``x`` (the residual stream) and ``h`` [B, S, C], C up to 8192, in bf16,
fp16 or fp32; ``y`` (the branch) and ``n`` of the same type, or bf16 / fp16 beside an
fp32 stream.  ``scale``, ``shift`` and ``gate`` are [C], [B, C] or [B, F, C]
(B or F may be 1) in any of the three types: with F frames, token s takes the
vector of frame s // (S / F).  Norms: ``"layer"`` (weight and bias optional) or
``"rms"`` (weight optional), over C.  Arithmetic and sums are fp32 with one
rounding of each output; ``n`` is of ``h`` before its rounding.

All three are differentiable in every tensor (once, in reverse mode; dual
tensors of forward mode are refused); gradients of vectors are fp32 sums in a
fixed order, so a step repeats bit for bit.  Calls run on the
current stream and can be captured into a CUDA graph, a backward pass with
them (``torch.autograd.grad``, after a first step outside the capture whose
autograd graph is gone: torch would have the capture wait for its stream).
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from ._launch import BLOCK_NORM, BLOCK_NORM_GRAD, dual_level, launch, refuse_tangents

_DT = {torch.bfloat16: N.LVSA_DTYPE_BF16, torch.float16: N.LVSA_DTYPE_F16, torch.float32: N.LVSA_DTYPE_F32}
_KINDS = {"layer": N.LVSA_BLOCK_NORM_LAYER, "rms": N.LVSA_BLOCK_NORM_RMS}


def norm_modulate(x: torch.Tensor, norm: str = "layer", weight: Optional[torch.Tensor] = None,
                  bias: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                  shift: Optional[torch.Tensor] = None, eps: float = 1e-6,
                  out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """norm(x) * (1 + scale) + shift, [B, S, C] in ``out_dtype`` (x's type, or
    bf16 / fp16 for an fp32 x)."""
    return _run("norm_modulate", x, None, None, 1.0, None, None, None, 0.0, norm, weight, bias, scale, shift, eps,
                out_dtype)[1]


def gate_residual(x: torch.Tensor, y: torch.Tensor, gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0,
                  post_norm: Optional[str] = None, post_weight: Optional[torch.Tensor] = None,
                  post_bias: Optional[torch.Tensor] = None, post_eps: float = 1e-6) -> torch.Tensor:
    """residual_scale * x + gate * post_norm(y), in x's type."""
    return _run("gate_residual", x, y, gate, residual_scale, post_norm, post_weight, post_bias, post_eps, None, None,
                None, None, None, 0.0, None)[0]


def gate_residual_norm(x: torch.Tensor, y: torch.Tensor, gate: Optional[torch.Tensor] = None,
                       residual_scale: float = 1.0, post_norm: Optional[str] = None,
                       post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                       post_eps: float = 1e-6, norm: str = "layer", weight: Optional[torch.Tensor] = None,
                       bias: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                       shift: Optional[torch.Tensor] = None, eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """(h, n): ``gate_residual`` and ``norm_modulate`` of its result, h in
    x's type and n in y's."""
    return _run("gate_residual_norm", x, y, gate, residual_scale, post_norm, post_weight, post_bias, post_eps, norm,
                weight, bias, scale, shift, eps, None)


# ------------------------------------------------------------------ arguments
class _Form:
    """What a call does, apart from its tensors."""
    __slots__ = ("join", "next", "post_kind", "post_eps", "kind", "eps", "alpha", "branch", "frames")


_ABSENT = (0, 0, 0, 0, 0)
_NO_ROWS = (0, 0, 0)


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _typed(where: str, name: str, t: torch.Tensor, device: int) -> int:
    if t.get_device() != device:
        raise ValueError(f"{where}: {name} is on {t.device}, x on cuda:{device}")
    code = _DT.get(t.dtype)
    if code is None:
        raise TypeError(f"{where}: {name} must be bf16, fp16 or fp32, got {t.dtype}")
    return code


def _vectors(where: str, name: str, t: torch.Tensor, B: int, C: int, device: int) -> torch.Tensor:
    """A modulation tensor, its channels contiguous, checked."""
    _typed(where, name, t, device)
    shape = t.shape
    n = len(shape)
    if not 1 <= n <= 3 or shape[-1] != C or (n > 1 and shape[0] != B and shape[0] != 1):
        raise ValueError(f"{where}: {name} must be [C], [B, C] or [B, F, C] with B = {B} and C = {C}, got {tuple(shape)}")
    return t if t.stride(-1) == 1 or C == 1 else t.contiguous()


def _channel(where: str, name: str, t: torch.Tensor, C: int, device: int) -> torch.Tensor:
    _typed(where, name, t, device)
    if t.dim() != 1 or t.shape[0] != C:
        raise ValueError(f"{where}: {name} must be [{C}], got {tuple(t.shape)}")
    return t if C == 1 or t.stride(0) == 1 else t.contiguous()


def _run(where, x, y, gate, alpha, post_norm, post_weight, post_bias, post_eps, norm, weight, bias, scale, shift, eps,
         out_dtype):
    if dual_level():
        refuse_tangents(where, (x, y, gate, scale, shift, weight, bias, post_weight, post_bias))
    if not x.is_cuda:
        raise RuntimeError(f"{where} needs CUDA tensors (no CPU fallback)")
    dtype, shape, device = x.dtype, x.shape, x.get_device()
    if dtype not in _DT:
        raise TypeError(f"{where}: x must be bf16, fp16 or fp32, got {dtype}")
    if len(shape) != 3 or not 1 <= shape[2] <= N.LVSA_BLOCK_NORM_MAX_WIDTH:
        raise ValueError(f"{where}: x must be [B, S, C] with C of 1 to {N.LVSA_BLOCK_NORM_MAX_WIDTH}, got {tuple(shape)}")
    B, S, C = shape
    form = _Form()
    form.join, form.next = y is not None, where != "gate_residual"
    form.alpha, form.eps, form.post_eps = float(alpha), float(eps), float(post_eps)
    if not (form.eps >= 0 and form.post_eps >= 0):
        raise ValueError(f"{where}: eps must not be negative")
    form.kind = _KINDS.get(norm, 0)
    form.post_kind = _KINDS.get(post_norm, 0)
    if form.next and not form.kind:
        raise ValueError(f"{where}: norm must be 'layer' or 'rms', got {norm!r}")
    if post_norm is not None and not form.post_kind:
        raise ValueError(f"{where}: post_norm must be None, 'layer' or 'rms', got {post_norm!r}")
    if form.join:
        _typed(where, "y", y, device)
        if y.shape != shape:
            raise ValueError(f"{where}: y {tuple(y.shape)} and x {tuple(shape)} differ")
        y = _rows(y)
        form.branch = y.dtype
    elif where == "norm_modulate":
        form.branch = dtype if out_dtype is None else out_dtype
    else:
        raise ValueError(f"{where}: y is missing")
    if form.branch != dtype and not (dtype == torch.float32 and form.branch in _DT):
        raise TypeError(f"{where}: a {dtype} stream goes with {dtype} branches"
                        f"{' or bf16 / fp16 ones' if dtype == torch.float32 else ''}, got {form.branch}")
    x = _rows(x)
    frames = None
    if gate is not None:
        gate = _vectors(where, "gate", gate, B, C, device)
        frames = gate.shape[1] if gate.dim() == 3 else 1
    if scale is not None:
        scale = _vectors(where, "scale", scale, B, C, device)
        frames = _frames(where, "scale", scale, frames)
    if shift is not None:
        shift = _vectors(where, "shift", shift, B, C, device)
        frames = _frames(where, "shift", shift, frames)
    form.frames = 1 if frames is None else frames
    if form.frames < 1 or S % form.frames:
        raise ValueError(f"{where}: {S} tokens do not divide into {form.frames} frames")
    if weight is not None:
        weight = _channel(where, "weight", weight, C, device)
    if bias is not None:
        if norm != "layer":
            raise ValueError(f"{where}: only a layer norm has a bias")
        bias = _channel(where, "bias", bias, C, device)
    if post_weight is not None:
        if not form.post_kind:
            raise ValueError(f"{where}: post_weight without post_norm")
        post_weight = _channel(where, "post_weight", post_weight, C, device)
    if post_bias is not None:
        if post_norm != "layer":
            raise ValueError(f"{where}: only a layer norm has a bias")
        post_bias = _channel(where, "post_bias", post_bias, C, device)
    tensors = (x, y, gate, scale, shift, weight, bias, post_weight, post_bias)
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                full = (B, form.frames, C)
                gate, scale, shift = (_full(v, full) for v in (gate, scale, shift))
                return _BlockNorm.apply(form, x, y, gate, scale, shift, weight, bias, post_weight, post_bias)
    return _forward(form, tensors, False)[:2]


def _frames(where: str, name: str, v: torch.Tensor, frames: Optional[int]) -> int:
    """The frames of v and of the vectors before it: those of any that has several."""
    n = v.shape[1] if v.dim() == 3 else 1
    if frames is None or frames == n or frames == 1:
        return n
    if n != 1:
        raise ValueError(f"{where}: {name} has {n} frames, another vector {frames}")
    return frames


def _full(v: Optional[torch.Tensor], full: Tuple[int, int, int]) -> Optional[torch.Tensor]:
    """A vector that needs a gradient as [B, F, C]: one that sequences or
    frames share gets its gradient summed over them in fp32, rounded once."""
    if v is None or not v.requires_grad or tuple(v.shape) == full:
        return v
    v = v[None, None] if v.dim() == 1 else v[:, None] if v.dim() == 2 else v
    return v if tuple(v.shape) == full else v.float().expand(full)


# ------------------------------------------------------------------- launches
def _row_args(t: Optional[torch.Tensor]) -> Tuple[int, int, int]:
    if t is None:
        return _NO_ROWS
    B, S, _ = t.shape
    stride_b, stride_t, _ = t.stride()
    return t.data_ptr(), stride_b if B > 1 else 0, stride_t if S > 1 else 0


def _vector_args(t: Optional[torch.Tensor]) -> Tuple[int, int, int, int, int]:
    if t is None:
        return _ABSENT
    n = t.dim()
    if n == 1:
        return t.data_ptr(), 0, 0, _DT[t.dtype], 0
    shape, stride = t.shape, t.stride()
    return (t.data_ptr(), stride[0] if shape[0] > 1 else 0, stride[1] if n == 3 and shape[1] > 1 else 0,
            _DT[t.dtype], 0)


def _norm_args(kind: int, eps: float, w: Optional[torch.Tensor], b: Optional[torch.Tensor]):
    if w is None and b is None:
        return kind, eps, 0, 0, 0, 0
    return (kind, eps, 0 if w is None else _DT[w.dtype], 0 if b is None else _DT[b.dtype],
            0 if w is None else w.data_ptr(), 0 if b is None else b.data_ptr())


def _args(form: _Form, tensors, h: int, n: int, stats, post_stats) -> tuple:
    """LvsaBlockNorm's fields; h, n: addresses of contiguous outputs."""
    x, y, gate, scale, shift, weight, bias, post_weight, post_bias = tensors
    B, S, C = x.shape
    return (*_row_args(x), *_row_args(y), h, S * C, C, n, S * C, C, *_vector_args(gate), *_vector_args(scale),
            *_vector_args(shift), *_norm_args(form.post_kind, form.post_eps, post_weight, post_bias),
            *_norm_args(form.kind, form.eps, weight, bias), form.alpha, _DT[x.dtype], _DT[form.branch], B, S,
            form.frames, C, 0 if stats is None else stats.data_ptr(), 0 if post_stats is None else post_stats.data_ptr())


def _forward(form: _Form, tensors, keep: bool):
    """(h or None, n or None, stats, post_stats); the statistics only where ``keep``."""
    x = tensors[0]
    shape = x.shape
    h = x.new_empty(shape) if form.join else None
    n = x.new_empty(shape, dtype=form.branch) if form.next else None
    rows = shape[0] * shape[1]
    stats = x.new_empty((rows, 2), dtype=torch.float32) if keep and form.next else None
    post_stats = x.new_empty((rows, 2), dtype=torch.float32) if keep and form.post_kind else None
    if rows:
        launch("lvsa_block_norm_fwd", BLOCK_NORM.pack(*_args(
            form, tensors, 0 if h is None else h.data_ptr(), 0 if n is None else n.data_ptr(), stats, post_stats)),
            x.get_device())
    return h, n, stats, post_stats


@lru_cache(maxsize=256)
def _workspace(stream: torch.dtype, branch: torch.dtype, B: int, S: int, frames: int, C: int, post: bool, join: bool,
               totals: bool, device: int) -> int:
    """Bytes that the backward of such a call needs, whatever its tensors."""
    mark = N.LvsaRows(16, 0, 0)  # not read
    g = N.LvsaBlockNormGrad()
    g.f.x = g.f.n = mark
    g.f.stats = g.f.post_stats = 16
    g.f.next.kind = N.LVSA_BLOCK_NORM_LAYER
    if join:
        g.f.y = mark
        g.f.post.kind = N.LVSA_BLOCK_NORM_LAYER if post else N.LVSA_BLOCK_NORM_NONE
    g.f.stream_dtype, g.f.branch_dtype = _DT[stream], _DT[branch]
    g.f.batch, g.f.seq, g.f.frames, g.f.width = B, S, frames, C
    if totals:
        g.f.next.weight = g.dweight = 16
    size = ctypes.c_int64()
    with torch.cuda.device(device):
        N.check(N.load().lvsa_block_norm_workspace(ctypes.byref(g), ctypes.byref(size)), "lvsa_block_norm_workspace")
    return size.value


def _backward(ctx, dh, dn):
    if dh is None and dn is None:
        return (None,) * 10
    if dual_level():
        refuse_tangents("the block norms' backward", (dh, dn))
    form = ctx.form
    saved = ctx.saved_tensors
    tensors, stats, post_stats = saved[:9], saved[9], saved[10]
    x = tensors[0]
    B, S, C = x.shape
    make = torch.empty_like if B * S else torch.zeros_like
    grads = [make(t, memory_format=torch.contiguous_format) if wanted and t is not None else None
             for t, wanted in zip(tensors, ctx.needs_input_grad[1:])]
    if B * S:
        dx, dy, dgate, dscale, dshift, dw, db, dpw, dpb = grads
        totals = [0 if t is None else t.data_ptr() for t in (dw, db, dpw, dpb)]
        device = x.get_device()
        size = _workspace(x.dtype, form.branch, B, S, form.frames, C, form.post_kind != 0, form.join, any(totals), device)
        space = x.new_empty((size,), dtype=torch.uint8)
        # n is set where there is a next norm, and not read.
        args = BLOCK_NORM_GRAD.pack(
            *_args(form, tensors, 0, x.data_ptr() if form.next else 0, stats, post_stats),
            *_row_args(None if dh is None else _rows(dh)), *_row_args(None if dn is None else _rows(dn)),
            *_row_args(dx), *_row_args(dy), *_vector_args(dgate), *_vector_args(dscale), *_vector_args(dshift), *totals,
            space.data_ptr(), size)
        launch("lvsa_block_norm_bwd", args, device)
    return (None, *grads)


_backward_once = once_differentiable(_backward)


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, form, *tensors):
        h, n, stats, post_stats = _forward(form, tensors, True)
        ctx.form = form
        ctx.save_for_backward(*tensors, stats, post_stats)
        ctx.set_materialize_grads(False)
        return h, n

    @staticmethod
    def backward(ctx, dh, dn):
        # Under create_graph a second differentiation has to be refused.
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, dh, dn)
