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

Tensors: ``x`` (the residual stream) and ``h`` [B, S, C] in bf16, fp16 or
fp32; ``y`` (the branch) and ``n`` of the same type, or bf16 / fp16 beside an
fp32 stream.  ``scale``, ``shift`` and ``gate`` are [C], [B, C] or [B, F, C]
(B or F may be 1) in any of the three types: with F frames, token s takes the
vector of frame s // (S / F).  Norms: ``"layer"`` (weight and bias optional) or
``"rms"`` (weight optional), over C.  Arithmetic and sums are fp32 with one
rounding of each output; ``n`` is of ``h`` before its rounding.

All three are differentiable in every tensor (once); gradients of vectors are
fp32 sums in a fixed order, so a step repeats bit for bit.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from .block_sparse import _stream_ptr

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
def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _vectors(where: str, name: str, t: Optional[torch.Tensor], x: torch.Tensor) -> Optional[torch.Tensor]:
    """A modulation tensor as [B or 1, F or 1, C]."""
    if t is None:
        return None
    _same_device(where, name, t, x)
    B, S, C = x.shape
    v = t[None, None] if t.dim() == 1 else t[:, None] if t.dim() == 2 else t
    if v.dim() != 3 or v.shape[2] != C or v.shape[0] not in (1, B):
        raise ValueError(f"{where}: {name} must be [C], [B, C] or [B, F, C] for x {tuple(x.shape)}, got {tuple(t.shape)}")
    return v if v.stride(2) == 1 or C == 1 else v.contiguous()


def _channel(where: str, name: str, t: Optional[torch.Tensor], x: torch.Tensor) -> Optional[torch.Tensor]:
    if t is None:
        return None
    _same_device(where, name, t, x)
    if t.dim() != 1 or t.shape[0] != x.shape[2]:
        raise ValueError(f"{where}: {name} must be [{x.shape[2]}], got {tuple(t.shape)}")
    return t if t.stride(0) == 1 or t.shape[0] == 1 else t.contiguous()


def _same_device(where: str, name: str, t: torch.Tensor, x: torch.Tensor) -> None:
    if t.device != x.device:
        raise ValueError(f"{where}: {name} is on {t.device}, x on {x.device}")
    if t.dtype not in _DT:
        raise TypeError(f"{where}: {name} must be bf16, fp16 or fp32, got {t.dtype}")


def _kind(where: str, name: str, kind: Optional[str]) -> int:
    if kind is None:
        return N.LVSA_BLOCK_NORM_NONE
    try:
        return _KINDS[kind]
    except KeyError:
        raise ValueError(f"{where}: {name} must be 'layer' or 'rms', got {kind!r}") from None


class _Form:
    """What a call does, apart from its tensors."""
    __slots__ = ("where", "join", "next", "post_kind", "post_eps", "kind", "eps", "alpha", "branch", "frames")


def _run(where, x, y, gate, alpha, post_norm, post_weight, post_bias, post_eps, norm, weight, bias, scale, shift, eps,
         out_dtype):
    if not x.is_cuda:
        raise RuntimeError(f"{where} needs CUDA tensors (no CPU fallback)")
    if x.dtype not in _DT:
        raise TypeError(f"{where}: x must be bf16, fp16 or fp32, got {x.dtype}")
    if x.dim() != 3 or not 1 <= x.shape[2] <= N.LVSA_BLOCK_NORM_MAX_WIDTH:
        raise ValueError(f"{where}: x must be [B, S, C] with C of 1 to {N.LVSA_BLOCK_NORM_MAX_WIDTH}, got {tuple(x.shape)}")
    form = _Form()
    form.where, form.join, form.next = where, y is not None, where != "gate_residual"
    form.alpha, form.eps, form.post_eps = float(alpha), float(eps), float(post_eps)
    if not (form.eps >= 0 and form.post_eps >= 0):
        raise ValueError(f"{where}: eps must not be negative")
    form.kind, form.post_kind = _kind(where, "norm", norm), _kind(where, "post_norm", post_norm)
    if form.next and not form.kind:
        raise ValueError(f"{where}: norm must be 'layer' or 'rms'")
    if (bias is not None and norm != "layer") or (post_bias is not None and post_norm != "layer"):
        raise ValueError(f"{where}: only a layer norm has a bias")
    if post_weight is not None and not form.post_kind:
        raise ValueError(f"{where}: post_weight without post_norm")
    if form.join:
        _same_device(where, "y", y, x)
        if y.shape != x.shape:
            raise ValueError(f"{where}: y {tuple(y.shape)} and x {tuple(x.shape)} differ")
        y = _rows(y)
        form.branch = y.dtype
    else:
        if where != "norm_modulate":
            raise ValueError(f"{where}: y is missing")
        form.branch = out_dtype if out_dtype is not None else x.dtype
    if form.branch != x.dtype and not (x.dtype == torch.float32 and form.branch in _DT):
        raise TypeError(f"{where}: a {x.dtype} stream goes with {x.dtype} branches"
                        f"{' or bf16 / fp16 ones' if x.dtype == torch.float32 else ''}, got {form.branch}")
    x = _rows(x)
    gate, scale, shift = (_vectors(where, n, t, x) for n, t in (("gate", gate), ("scale", scale), ("shift", shift)))
    weight, bias, post_weight, post_bias = (
        _channel(where, n, t, x) for n, t in (("weight", weight), ("bias", bias), ("post_weight", post_weight),
                                              ("post_bias", post_bias)))
    form.frames = max([v.shape[1] for v in (gate, scale, shift) if v is not None], default=1)
    if form.frames < 1 or x.shape[1] % form.frames:
        raise ValueError(f"{where}: {x.shape[1]} tokens do not divide into {form.frames} frames")
    for name, v in (("gate", gate), ("scale", scale), ("shift", shift)):
        if v is not None and v.shape[1] not in (1, form.frames):
            raise ValueError(f"{where}: {name} has {v.shape[1]} frames, another vector {form.frames}")
    tensors = (x, y, gate, scale, shift, weight, bias, post_weight, post_bias)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        # A vector shared by sequences or frames: its gradient is summed in fp32 over them, then rounded once.
        full = (x.shape[0], form.frames, x.shape[2])
        gate, scale, shift = (v if v is None or not v.requires_grad or v.shape == full else v.float().expand(full)
                              for v in (gate, scale, shift))
        return _BlockNorm.apply(form, x, y, gate, scale, shift, weight, bias, post_weight, post_bias)
    return _forward(form, tensors, False)[:2]


# ------------------------------------------------------------------- launches
def _row_view(t: Optional[torch.Tensor]) -> N.LvsaRows:
    if t is None:
        return N.LvsaRows()
    B, S, _ = t.shape
    return N.LvsaRows(t.data_ptr(), t.stride(0) if B > 1 else 0, t.stride(1) if S > 1 else 0)


def _vector_view(t: Optional[torch.Tensor]) -> N.LvsaVectors:
    if t is None:
        return N.LvsaVectors()
    return N.LvsaVectors(t.data_ptr(), t.stride(0) if t.shape[0] > 1 else 0, t.stride(1) if t.shape[1] > 1 else 0,
                         _DT[t.dtype], 0)


def _norm_view(kind: int, eps: float, w: Optional[torch.Tensor], b: Optional[torch.Tensor]) -> N.LvsaRowNorm:
    return N.LvsaRowNorm(kind, eps, _DT[w.dtype] if w is not None else 0, _DT[b.dtype] if b is not None else 0,
                         w.data_ptr() if w is not None else None, b.data_ptr() if b is not None else None)


def _args(form: _Form, tensors, h, n, stats, post_stats) -> N.LvsaBlockNorm:
    x, y, gate, scale, shift, weight, bias, post_weight, post_bias = tensors
    B, S, C = x.shape
    return N.LvsaBlockNorm(_row_view(x), _row_view(y), _row_view(h), _row_view(n), _vector_view(gate),
                           _vector_view(scale), _vector_view(shift),
                           _norm_view(form.post_kind, form.post_eps, post_weight, post_bias),
                           _norm_view(form.kind, form.eps, weight, bias), form.alpha, _DT[x.dtype], _DT[form.branch],
                           B, S, form.frames, C, stats.data_ptr() if stats is not None else None,
                           post_stats.data_ptr() if post_stats is not None else None)


def _forward(form: _Form, tensors, keep: bool):
    """(h or None, n or None, stats, post_stats); the statistics only where ``keep``."""
    x = tensors[0]
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device) if form.join else None
    n = torch.empty(x.shape, dtype=form.branch, device=x.device) if form.next else None
    rows = x.shape[0] * x.shape[1]
    stats = torch.empty(rows, 2, dtype=torch.float32, device=x.device) if keep and form.next else None
    post_stats = torch.empty(rows, 2, dtype=torch.float32, device=x.device) if keep and form.post_kind else None
    if rows:
        args = _args(form, tensors, h, n, stats, post_stats)
        with torch.cuda.device(x.device):
            st = N.load().lvsa_block_norm_fwd(ctypes.byref(args), _stream_ptr(x.device))
        N.check(st, "lvsa_block_norm_fwd")
    return h, n, stats, post_stats


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, form, *tensors):
        h, n, stats, post_stats = _forward(form, tensors, True)
        ctx.form = form
        ctx.save_for_backward(*tensors, stats, post_stats)
        ctx.set_materialize_grads(False)
        return h, n

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dn):
        form = ctx.form
        *tensors, stats, post_stats = ctx.saved_tensors
        x, y, gate, scale, shift, weight, bias, post_weight, post_bias = tensors
        need = ctx.needs_input_grad[1:]
        if dh is None and dn is None:
            return (None,) * 10
        dh, dn = (None if d is None else _rows(d) for d in (dh, dn))
        make = torch.empty if x.shape[0] * x.shape[1] else torch.zeros
        grads = [make(t.shape, dtype=t.dtype, device=t.device) if wanted and t is not None else None
                 for t, wanted in zip(tensors, need)]
        dx, dy, dgate, dscale, dshift, dw, db, dpw, dpb = grads
        if x.shape[0] * x.shape[1]:
            ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
            f = _args(form, tensors, None, None, stats, post_stats)
            if form.next:  # says that there is a next norm; not read
                f.n = _row_view(x)
            args = N.LvsaBlockNormGrad(f, _row_view(dh), _row_view(dn), _row_view(dx), _row_view(dy),
                                       _vector_view(dgate), _vector_view(dscale), _vector_view(dshift),
                                       ptr(dw), ptr(db), ptr(dpw), ptr(dpb), None, 0)
            lib, size = N.load(), ctypes.c_int64()
            with torch.cuda.device(x.device):
                N.check(lib.lvsa_block_norm_workspace(ctypes.byref(args), ctypes.byref(size)),
                        "lvsa_block_norm_workspace")
                space = torch.empty(size.value, dtype=torch.uint8, device=x.device)
                args.workspace, args.workspace_bytes = space.data_ptr(), size.value
                st = lib.lvsa_block_norm_bwd(ctypes.byref(args), _stream_ptr(x.device))
            N.check(st, "lvsa_block_norm_bwd")
        return (None, *grads)
