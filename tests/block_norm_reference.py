"""The block norms' definition in 64 bits, and how far fp32 arithmetic with
one rounding of each output may be from it."""

import torch

U32 = 2.0 ** -24  # one fp32 rounding, relative


def _norm(z, kind, w, b, eps):
    zc = z - z.mean(-1, keepdim=True) if kind == "layer" else z
    zh = zc / torch.sqrt((zc * zc).mean(-1, keepdim=True) + eps)
    out = zh if w is None else zh * w
    return out if b is None else out + b


def _rows_of(v, x):
    """[C], [B, C] or [B, F, C] -> broadcastable over [B, S, C]."""
    v = v[None, None] if v.dim() == 1 else v[:, None] if v.dim() == 2 else v
    return v.repeat_interleave(x.shape[1] // v.shape[1], dim=1) if v.shape[1] else v


def definition(x, y=None, gate=None, alpha=1.0, post=None, post_weight=None, post_bias=None, norm=None, weight=None,
               bias=None, scale=None, shift=None, eps=1e-6, post_eps=1e-6):
    """(h, n) of 64-bit tensors; h = x without a join, n = None without a norm."""
    h = x
    if y is not None:
        branch = y if post is None else _norm(y, post, post_weight, post_bias, post_eps)
        h = alpha * x + (branch if gate is None else _rows_of(gate, x) * branch)
    n = None
    if norm is not None:
        n = _norm(h, norm, weight, bias, eps)
        n = n if scale is None else n * (1 + _rows_of(scale, x))
        n = n if shift is None else n + _rows_of(shift, x)
    return h, n


def check(what, got, want, size):
    """got within half a step of its type of want, plus ``size`` (a bound of
    the fp32 arithmetic's error, as a tensor or a number)."""
    half = torch.finfo(got.dtype).eps / 2
    # A value below the normal range is rounded on the smallest step there.
    floor = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    bound = half * want.abs() * (1 + half) + size * (1 + half) + floor
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, the worst by " \
        f"{float(((got.double() - want).abs() / bound).nan_to_num(float('inf')).max()):.2f} of what is allowed"
