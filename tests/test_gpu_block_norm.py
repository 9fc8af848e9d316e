"""Block norms (norm, modulation, gate, residual scale) against their
definition in 64 bits, forward and backward.

Bounds.  u = 2^-24.  A normalised value zh = (z - m) r takes a rounding each for
z - m, the product and r's few operations, and m and r carry the error of sums
of C terms added in a tree of at most 8 + 5 + 5 levels a thread, warp and CTA:
below 24 u (|z| + mean|z|) r + 24 u |zh| together, doubled for the second norm.
Sums over R rows are added row by row in a thread: below (R + 40) u of the sum
of the terms' sizes, plus the terms' own error."""

import pytest
import torch

from tests.block_norm_reference import U32, check, definition

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _make(shape, dtype, g, scale=1.0, at=0.0):
    return (torch.randn(*shape, generator=g) * scale + at).to(dtype).cuda()


def _inputs(B, S, F, C, stream, branch, mod, norm, affine, post, seed, join):
    g = torch.Generator().manual_seed(seed)
    t = dict(x=_make((B, S, C), stream, g, 2.0, 0.5))
    if join:
        t["y"] = _make((B, S, C), branch, g, 0.7)
        t["gate"] = _make((B, F, C), mod, g, 0.5)
        if post:
            t["post_weight"] = _make((C,), mod, g, 0.2, 1.0)
        if post == "layer":
            t["post_bias"] = _make((C,), mod, g, 0.2)
    if norm:
        t["scale"], t["shift"] = _make((B, F, C), mod, g, 0.3), _make((B, F, C), mod, g, 0.3)
        if affine:
            t["weight"] = _make((C,), mod, g, 0.2, 1.0)
            if norm == "layer":
                t["bias"] = _make((C,), mod, g, 0.2)
    return t


def _call(t, norm, post, alpha, branch, eps=1e-6):
    from longvideosparseattention_b200.block_norm import gate_residual, gate_residual_norm, norm_modulate
    get = t.get
    if "y" not in t:
        return None, norm_modulate(t["x"], norm, get("weight"), get("bias"), get("scale"), get("shift"), eps, out_dtype=branch)
    if not norm:
        return gate_residual(t["x"], t["y"], get("gate"), alpha, post, get("post_weight"), get("post_bias"), eps), None
    return gate_residual_norm(t["x"], t["y"], get("gate"), alpha, post, get("post_weight"), get("post_bias"), eps, norm,
                              get("weight"), get("bias"), get("scale"), get("shift"), eps)


def _define(t, norm, post, alpha, eps=1e-6):
    return definition(t["x"], t.get("y"), t.get("gate"), alpha, post, t.get("post_weight"), t.get("post_bias"), norm,
                      t.get("weight"), t.get("bias"), t.get("scale"), t.get("shift"), eps, eps)


def _rows_of(v, x):
    v = v[None, None] if v.dim() == 1 else v[:, None] if v.dim() == 2 else v
    return v.repeat_interleave(x.shape[1] // v.shape[1], dim=1)


def _sizes(t, norm, post, alpha, eps=1e-6):
    """Bounds of the fp32 error of h and of n before their rounding."""
    def of_norm(z, dz, kind, w, b):
        zc = z - z.mean(-1, keepdim=True) if kind == "layer" else z
        r = 1 / torch.sqrt((zc * zc).mean(-1, keepdim=True) + eps)
        zh = (zc * r).abs()
        far = 24 * U32 * ((z.abs() + z.abs().mean(-1, keepdim=True)) * r + zh) + 2 * (dz + dz.mean(-1, keepdim=True)) * r * (1 + zh)
        out, val = (far, zh) if w is None else (far * w.abs(), zh * w.abs())
        val = val if b is None else val + b.abs()
        return out + 4 * U32 * val, val
    x = t["x"].double()
    z, dz = x, torch.zeros_like(x)
    if "y" in t:
        d, val = torch.zeros_like(x), t["y"].double().abs()
        if post:
            w, b = t.get("post_weight"), t.get("post_bias")
            d, val = of_norm(t["y"].double(), d, post, None if w is None else w.double(), None if b is None else b.double())
        g = _rows_of(t["gate"].double(), x).abs() if "gate" in t else 1.0
        dz = g * d + 6 * U32 * (g * val + (alpha * x).abs())
        z = _define({k: v.double() for k, v in t.items()}, None, post, alpha, eps)[0]
    if not norm:
        return dz, None
    w, b = t.get("weight"), t.get("bias")
    d, val = of_norm(z, dz, norm, None if w is None else w.double(), None if b is None else b.double())
    up = (1 + _rows_of(t["scale"].double(), x)).abs() if "scale" in t else 1.0
    sh = _rows_of(t["shift"].double(), x).abs() if "shift" in t else 0.0
    return dz, up * d + 6 * U32 * (up * val + sh)


SHAPES = [  # B, S, F, C
    (1, 1, 1, 8), (1, 3, 3, 1), (2, 77, 1, 2048), (1, 35, 5, 1155), (2, 12, 4, 264), (1, 300, 1, 5120), (1, 9, 3, 6144),
    (1, 4, 1, 8192), (1, 3, 1, 8191), (2, 5000, 5, 64), (1, 40, 40, 128), (1, 2600, 2, 1536), (3, 7, 7, 9)]
TYPES = [(BF, BF, BF), (HF, HF, F32), (F32, BF, F32), (F32, HF, HF), (F32, F32, F32), (BF, BF, F32)]
FORMS = [  # norm, affine, post, alpha, join
    ("layer", False, None, 1.0, False), ("rms", True, None, 1.0, False), ("layer", True, None, 0.5, True),
    ("rms", False, "rms", 1.0, True), ("layer", True, "layer", -0.7, True), (None, False, "rms", 2.0, True),
    (None, False, None, 1.0, True)]


def _cases():
    """Every shape with every form, the types in turn."""
    return [(s, TYPES[(i + 2 * j) % len(TYPES)], f) for i, s in enumerate(SHAPES) for j, f in enumerate(FORMS)]


@pytest.mark.parametrize("shape,types,form", _cases())
def test_forward(shape, types, form):
    (B, S, F, C), (stream, branch, mod), (norm, affine, post, alpha, join) = shape, types, form
    t = _inputs(B, S, F, C, stream, branch, mod, norm, affine, post, S + C, join)
    h, n = _call(t, norm, post, alpha, branch)
    wh, wn = _define({k: v.double() for k, v in t.items()}, norm, post, alpha)
    dh, dn = _sizes(t, norm, post, alpha)
    if join:
        assert h.dtype == stream and h.shape == (B, S, C)
        check("h", h, wh, dh)
    if norm:
        assert n.dtype == branch and n.shape == (B, S, C)
        check("n", n, wn, dn)


@pytest.mark.parametrize("shape,types,form", _cases())
def test_backward(shape, types, form):
    (B, S, F, C), (stream, branch, mod), (norm, affine, post, alpha, join) = shape, types, form
    t = _inputs(B, S, F, C, stream, branch, mod, norm, affine, post, S + C + 1, join)
    g = torch.Generator().manual_seed(5)
    seeds = [_make((B, S, C), ty, g) for ty, there in ((stream, join), (branch, norm)) if there]
    leaves = {k: v.requires_grad_(True) for k, v in t.items()}
    outs = [o for o in _call(leaves, norm, post, alpha, branch) if o is not None]
    got = torch.autograd.grad(outs, list(leaves.values()), seeds)
    again = torch.autograd.grad([o for o in _call(leaves, norm, post, alpha, branch) if o is not None],
                                list(leaves.values()), seeds)
    wide = {k: v.detach().double().requires_grad_(True) for k, v in t.items()}
    wh, wn = _define(wide, norm, post, alpha)
    wouts = [o for o, there in ((wh, join), (wn, norm)) if there]
    want = torch.autograd.grad(wouts, list(wide.values()), [s.double() for s in seeds])
    # Sizes of the terms: the same gradients with every term at its absolute value would be the sharpest; a row's
    # statistics, r and |zh| and |yh|, bound them all.
    with torch.no_grad():
        size = _gradient_sizes({k: v.detach() for k, v in wide.items()}, norm, post, alpha, seeds, join)
    for k, a, b, w in zip(leaves, got, again, want):
        assert a.dtype == t[k].dtype and torch.equal(a, b), k
        check("d" + k, a, w, size[k])


def _gradient_sizes(t, norm, post, alpha, seeds, join, eps=1e-6):
    """Bounds of the fp32 error of each gradient before its rounding."""
    x = t["x"]
    B, S, C = x.shape
    seeds = [s.double() for s in seeds]
    dh = seeds[0] if join else torch.zeros_like(x)
    dn = seeds[-1] if norm else None
    out = {}

    def stats(z, kind):
        zc = z - z.mean(-1, keepdim=True) if kind == "layer" else z
        r = 1 / torch.sqrt((zc * zc).mean(-1, keepdim=True) + eps)
        return zc * r, r

    def through(v, zh, r, ez, ev):
        """Size of an error of r (v - mean v - zh mean(v zh)) with zh off by ez and v by ev."""
        v, zh = v.abs(), zh.abs()
        m = lambda q: q.mean(-1, keepdim=True)  # noqa: E731
        rel = 48 * U32 * r * (v + m(v) + zh * m(v * zh))
        return rel + r * (ev + m(ev) + zh * m(ev * zh) + ez * m(v * zh) + zh * m(v * ez))

    def sums(terms, errors):
        """Of a sum over the rows of each frame, and over all of them."""
        F = max(t[k].shape[1] for k in ("gate", "scale", "shift") if k in t)
        fold = lambda q: q.view(B, F, S // F, C).sum(2)  # noqa: E731
        return (S // F + 40) * U32 * fold(terms) + fold(errors), fold

    yh = ey = None
    if join:
        yh, yr = stats(t["y"], post) if post else (t["y"], torch.ones_like(x[..., :1]))
        ey = 24 * U32 * ((t["y"].abs() + t["y"].abs().mean(-1, keepdim=True)) * yr + yh.abs()) if post else torch.zeros_like(x)
    e, d = torch.zeros_like(x), dh
    if norm:
        h = _define(t, None, post, alpha)[0]
        zh, r = stats(h, norm)
        eh = _sizes({k: v for k, v in t.items()}, None, post, alpha)[0]
        ez = 24 * U32 * ((h.abs() + h.abs().mean(-1, keepdim=True)) * r + zh.abs()) + 2 * (eh + eh.mean(-1, keepdim=True)) * r * (1 + zh.abs())
        w, b = t.get("weight"), t.get("bias")
        up = 1 + _rows_of(t["scale"], x)
        s0, fold = sums(dn.abs() * zh.abs(), dn.abs() * ez)
        q0, _ = sums(dn.abs(), torch.zeros_like(x))
        wa, ba = (1.0 if w is None else w.abs()), (0.0 if b is None else b.abs())
        out["shift"] = q0
        out["scale"] = s0 * wa + q0 * ba + 4 * U32 * (wa * fold((dn * zh).abs()) + ba * fold(dn.abs()))
        upf = (1 + t["scale"]).abs()
        many = (B * t["scale"].shape[1] + 40) * U32
        if w is not None:
            out["weight"] = (upf * s0).sum((0, 1)) + many * (upf * fold((dn * zh).abs())).sum((0, 1))
        if b is not None:
            out["bias"] = (upf * q0).sum((0, 1)) + many * (upf * fold(dn.abs())).sum((0, 1))
        v = dn * up * (1.0 if w is None else w)
        e = through(v, zh, r, ez, 4 * U32 * v.abs())
        m = lambda q: q.mean(-1, keepdim=True)  # noqa: E731
        d = dh + r * (v - (m(v) if norm == "layer" else 0) - zh * m(v * zh))
        e = e + 4 * U32 * (dh.abs() + d.abs())
    out["x"] = abs(alpha) * (e + 2 * U32 * d.abs()) if join else e
    if join:
        w, b = t.get("post_weight"), t.get("post_bias")
        wa, ba = (1.0 if w is None else w.abs()), (0.0 if b is None else b.abs())
        s2, fold = sums((d * yh).abs(), e * yh.abs() + d.abs() * ey)
        q2, _ = sums(d.abs(), e)
        out["gate"] = s2 * wa + q2 * ba + 4 * U32 * (wa * fold((d * yh).abs()) + ba * fold(d.abs()))
        gt = t["gate"].abs()
        many = (B * t["gate"].shape[1] + 40) * U32
        if w is not None:
            out["post_weight"] = (gt * s2).sum((0, 1)) + many * (gt * fold((d * yh).abs())).sum((0, 1))
        if b is not None:
            out["post_bias"] = (gt * q2).sum((0, 1)) + many * (gt * fold(d.abs())).sum((0, 1))
        g1 = _rows_of(t["gate"], x) * (1.0 if w is None else w)
        u, eu = d * g1, e * g1.abs() + 4 * U32 * (d * g1).abs()
        out["y"] = through(u, yh, yr, ey, eu) if post else eu
    return out


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("shape", [(1, 592, 4, 45), (1, 595, 5, 1155), (2, 310, 2, 2047), (2, 21, 3, 1539), (1, 10, 2, 2049),
                                   (1, 600, 600, 33), (1, 37, 1, 4097)])
def test_widths_of_no_vector(shape, form):
    """On both sides of 592 rows (four an SM) and of 4 values a thread."""
    types = TYPES[(shape[3] + FORMS.index(form)) % len(TYPES)]
    test_forward(shape, types, form)
    test_backward(shape, types, form)


def test_gradient_against_differences():
    """Along a direction, central differences of the fp32 kernels themselves:
    off by the step's square (1e-4) and by the outputs' rounding over it."""
    t = _inputs(1, 24, 3, 136, F32, F32, F32, "layer", True, "rms", 3, True)
    g = torch.Generator().manual_seed(9)
    ah, an = _make((1, 24, 136), F32, g), _make((1, 24, 136), F32, g)
    def loss(at):
        h, n = _call(at, "layer", "rms", 0.8, F32)
        return (h.double() * ah).sum() + (n.double() * an).sum()
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    h, n = _call(leaves, "layer", "rms", 0.8, F32)
    grads = dict(zip(leaves, torch.autograd.grad([h, n], list(leaves.values()), [ah, an])))
    for k, v in t.items():
        direction = _make(v.shape, F32, g)
        step = 1e-2
        up = loss({**t, k: v + step * direction})
        down = loss({**t, k: v - step * direction})
        want = float((up - down) / (2 * step))
        got = float((grads[k].double() * direction).sum())
        # third derivatives of a normalised value are of the order of the values: step^2 of sqrt(terms) x 10, and
        # 2^-24 of them each over the step.
        size = float((grads[k].double() * direction).square().sum().sqrt()) + 10 * (24 * 136) ** 0.5 ** 1
        assert abs(got - want) <= size * (step * step * 10 + 2 ** -24 / step * 4), k


@pytest.mark.parametrize("shape", [(2, 6, 3, 40), (2, 6, 1, 40)])
def test_shared_vectors(shape):
    """[C], [B, C], [1, F, C] and [B, 1, C] vectors: values, and gradients summed over what shares them."""
    B, S, F, C = shape
    g = torch.Generator().manual_seed(1)
    forms = [(C,), (B, C), (1, F, C), (B, 1, C), (B, F, C)]
    for i, sg in enumerate(forms):
        t = _inputs(B, S, F, C, F32, F32, F32, "layer", False, None, i, True)
        t["gate"], t["scale"] = _make(sg, F32, g), _make(forms[(i + 1) % 5], F32, g)
        t["shift"] = _make(forms[(i + 2) % 5], BF, g)
        leaves = {k: v.requires_grad_(True) for k, v in t.items()}
        h, n = _call(leaves, "layer", None, 1.0, F32)
        got = torch.autograd.grad([h, n], list(leaves.values()), [h.detach(), n.detach()])
        wide = {k: v.detach().double().requires_grad_(True) for k, v in t.items()}
        wh, wn = _define(wide, "layer", None, 1.0)
        want = torch.autograd.grad([wh, wn], list(wide.values()), [h.detach().double(), n.detach().double()])
        for k, a, w in zip(leaves, got, want):
            assert a.dtype == t[k].dtype
            check(k, a, w, 400 * U32 * (w.abs().max() + 10))  # 12 rows of values below 10, each off by < 24 u of them


def test_absent_vectors_and_partial_gradients():
    """No gate, scale, shift; gradients of some tensors only, or of one output only."""
    from longvideosparseattention_b200.block_norm import gate_residual_norm, norm_modulate
    g = torch.Generator().manual_seed(2)
    x, y = _make((2, 9, 72), F32, g).requires_grad_(True), _make((2, 9, 72), F32, g)
    gate = _make((72,), F32, g).requires_grad_(True)
    h, n = gate_residual_norm(x, y, gate, norm="rms")
    wx, wg = x.detach().double().requires_grad_(True), gate.detach().double().requires_grad_(True)
    wh, wn = definition(wx, y.double(), wg, norm="rms")
    for outs, wouts in (([h], [wh]), ([n], [wn]), ([h, n], [wh, wn])):
        a = torch.autograd.grad(outs, [x, gate], [torch.ones_like(o) for o in outs], retain_graph=True)
        b = torch.autograd.grad(wouts, [wx, wg], [torch.ones_like(o) for o in wouts], retain_graph=True)
        for p, q in zip(a, b):
            check("gradient", p, q, 2000 * U32 * (1 + q.abs().max()))  # 18 rows of values below 5
    check("plain", norm_modulate(x.detach()), definition(x.detach().double(), norm="layer")[1], 100 * U32 * 5)
    z = norm_modulate(x, "rms").sum()  # an expanded gradient (stride 0)
    z.backward()
    assert torch.isfinite(x.grad).all()


def test_strides_and_alignment():
    """Slices of a joint sequence, chunks of one modulation tensor, an odd offset, a transposed tensor."""
    from longvideosparseattention_b200.block_norm import gate_residual_norm, norm_modulate
    g = torch.Generator().manual_seed(4)
    B, C = 2, 192
    joint = _make((B, 50, C), BF, g)
    mod = _make((B, 6, C), F32, g, 0.3)
    shift, scale, gate = mod[:, 0], mod[:, 1], mod[:, 2]
    for x in (joint[:, 7:40], joint[:, ::2], joint[1:], joint.transpose(1, 2)[:, :50, :48].transpose(1, 2)[:, :48]):
        c = x.shape[2]
        s, t = scale[:x.shape[0], :c], shift[:x.shape[0], :c]
        got = norm_modulate(x, "layer", scale=s, shift=t)
        d = dict(x=x, scale=s, shift=t)
        check("slice", got, _define({k: v.double() for k, v in d.items()}, "layer", None, 1.0)[1], _sizes(d, "layer", None, 1.0)[1])
    flat = _make((1, 10 * C + 1,), BF, g)
    x = flat[0, 1:].view(1, 10, C)  # 2 bytes past a vector
    y = joint[:1, :10]
    d = dict(x=x, y=y, gate=gate[:1], scale=scale[:1], shift=mod[:1, 0])
    h, n = gate_residual_norm(x, y, gate[:1], scale=scale[:1], shift=mod[:1, 0])
    wh, wn = _define({k: v.double() for k, v in d.items()}, "layer", None, 1.0)
    dh, dn = _sizes(d, "layer", None, 1.0)
    check("h", h, wh, dh)
    check("n", n, wn, dn)
    shifted = torch.zeros(C + 3, device="cuda")[3:].copy_(scale[0])  # 12 bytes past a vector
    assert torch.equal(norm_modulate(joint, scale=shifted), norm_modulate(joint, scale=scale[0]))


def test_values_out_of_range_stay_in_their_row():
    from longvideosparseattention_b200.block_norm import gate_residual_norm, norm_modulate
    g = torch.Generator().manual_seed(6)
    x, y = _make((1, 8, 320), F32, g), _make((1, 8, 320), F32, g)
    h0, n0 = gate_residual_norm(x, y)
    x[0, 2, 5], x[0, 4, 0], y[0, 6, 319] = float("nan"), float("inf"), float("-inf")
    h, n = gate_residual_norm(x, y)
    good = [0, 1, 3, 5, 7]
    assert torch.equal(h[:, good], h0[:, good]) and torch.equal(n[:, good], n0[:, good])
    assert n[0, [2, 4, 6]].isnan().all()
    assert torch.equal(h[0, 2, :5], h0[0, 2, :5]) and h[0, 4, 0] == float("inf") and h[0, 6, 319] == float("-inf")
    # A constant row has no deviation: n = shift; a large offset does not cost the deviation its digits.
    shift = _make((320,), F32, g)
    assert torch.equal(norm_modulate(torch.full((1, 2, 320), 3.0, device="cuda"), shift=shift)[0, 0], shift)
    z = 4096.0 + torch.randn(1, 5, 320, generator=g).cuda().mul_(64).round_().div_(64)
    check("offset", norm_modulate(z), definition(z.double(), norm="layer")[1],
          _sizes(dict(x=z), "layer", None, 1.0)[1])


@pytest.mark.parametrize("shape", [(0, 5, 16), (2, 0, 16)])
def test_empty(shape):
    from longvideosparseattention_b200.block_norm import gate_residual_norm
    x = torch.zeros(shape, device="cuda", requires_grad=True)
    gate = torch.ones(16, device="cuda", requires_grad=True)
    h, n = gate_residual_norm(x, torch.zeros(shape, device="cuda"), gate)
    assert h.shape == n.shape == shape
    (h.sum() + n.sum()).backward()
    assert torch.equal(gate.grad, torch.zeros(16, device="cuda")) and x.grad.shape == shape


def test_other_stream_and_graph():
    """On a side stream, and a training step captured once and replayed on new values."""
    t = _inputs(1, 600, 3, 512, BF, BF, BF, "layer", True, "rms", 8, True)
    g = torch.Generator().manual_seed(8)
    ah, an = _make((1, 600, 512), BF, g), _make((1, 600, 512), BF, g)
    leaves = {k: v.requires_grad_(True) for k, v in t.items()}

    def step():
        h, n = _call(leaves, "layer", "rms", 1.0, BF)
        return (h, n, *torch.autograd.grad([h, n], list(leaves.values()), [ah, an]))
    want = [v.detach().clone() for v in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [v.detach() for v in step()]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same leaves, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([v.detach() for v in step()])
        graphs.append(graph)
    with torch.no_grad():
        for v in leaves.values():
            v.mul_(0.5)
    want = [v.detach().clone() for v in step()]
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_second_derivative_is_refused():
    """create_graph gives first derivatives; differentiating those raises rather than giving zeros."""
    from longvideosparseattention_b200.block_norm import gate_residual_norm
    g = torch.Generator().manual_seed(3)
    x, y = _make((1, 4, 64), F32, g).requires_grad_(True), _make((1, 4, 64), F32, g)
    h, n = gate_residual_norm(x, y)
    first, = torch.autograd.grad(h.sum() + (n * n).sum(), x, create_graph=True)
    h, n = gate_residual_norm(x, y)
    again, = torch.autograd.grad(h.sum() + (n * n).sum(), x)
    assert torch.equal(first.detach(), again)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), x)


def test_saved_tensors():
    """Saved tensors that a hook keeps elsewhere and brings back to other places; and one changed in place."""
    t = _inputs(1, 30, 3, 264, BF, BF, F32, "layer", True, "rms", 5, True)
    leaves = {k: v.requires_grad_(True) for k, v in t.items()}
    h, n = _call(leaves, "layer", "rms", 1.0, BF)
    want = torch.autograd.grad([h, n], list(leaves.values()), [h.detach(), n.detach()])
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v.cpu(), lambda v: v.cuda()):
        h, n = _call(leaves, "layer", "rms", 1.0, BF)
    got = torch.autograd.grad([h, n], list(leaves.values()), [h.detach(), n.detach()])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    h, n = _call(leaves, "layer", "rms", 1.0, BF)
    with torch.no_grad():
        t["scale"].add_(1)
    with pytest.raises(RuntimeError):
        n.sum().backward()


def test_offsets_past_32_bits():
    """More than 2^31 values: the last rows, forward and backward."""
    from longvideosparseattention_b200.block_norm import gate_residual_norm
    C, S = 8192, 2 ** 18 + 5
    g = torch.Generator().manual_seed(12)
    x, y = (torch.zeros(1, S, C, dtype=BF, device="cuda") for _ in range(2))
    last = 3
    x[:, -last:], y[:, -last:] = _make((1, last, C), BF, g), _make((1, last, C), BF, g)
    gate, shift = _make((C,), F32, g), _make((C,), F32, g)
    short = [v[:, -last:].clone() for v in (x, y)]
    for v in (x, y, gate):
        v.requires_grad_(True)
    h, n = gate_residual_norm(x, y, gate, shift=shift)
    dn = torch.zeros_like(n)
    dn[:, -last:] = _make((1, last, C), BF, g)
    dx, dy, dgate = torch.autograd.grad(n, (x, y, gate), dn)
    assert torch.equal(n[0, 0], shift.bfloat16()) and torch.equal(n[0, 2 ** 17], shift.bfloat16())
    sx, sy, sg = short[0].requires_grad_(True), short[1].requires_grad_(True), gate.detach().requires_grad_(True)
    sh, sn = gate_residual_norm(sx, sy, sg, shift=shift)
    ex, ey, eg = torch.autograd.grad(sn, (sx, sy, sg), dn[:, -last:])
    # The same rows by the same kernels, in another order of the sums of a row: a step of bf16, and fp32's.
    for a, b in ((h[:, -last:], sh), (n[:, -last:], sn), (dx[:, -last:], ex), (dy[:, -last:], ey)):
        assert ((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 1e-4).all()
    assert ((dgate - eg).abs() <= 1e-4 * (1 + eg.abs())).all()
    assert not dx[:, : -last].any() and not dy[:, : -last].any()


def test_refusals_on_cuda_tensors():
    from longvideosparseattention_b200.block_norm import gate_residual, gate_residual_norm, norm_modulate
    x = torch.zeros(2, 6, 16, device="cuda")
    v = torch.zeros(16, device="cuda")
    bad = [
        lambda: norm_modulate(x[0]), lambda: norm_modulate(x, "batch"), lambda: norm_modulate(x, None),
        lambda: norm_modulate(x, "rms", bias=v), lambda: norm_modulate(x, weight=v[:8]),
        lambda: norm_modulate(x, scale=torch.zeros(3, 16, device="cuda")),
        lambda: norm_modulate(x, scale=torch.zeros(2, 4, 16, device="cuda")),
        lambda: norm_modulate(x, scale=torch.zeros(2, 2, 16, device="cuda"), shift=torch.zeros(2, 3, 16, device="cuda")),
        lambda: norm_modulate(x, scale=torch.zeros(16)), lambda: norm_modulate(x, eps=-1.0),
        lambda: norm_modulate(torch.zeros(1, 1, 8193, device="cuda")),
        lambda: gate_residual(x, x[:, :3]), lambda: gate_residual(x, x, post_weight=v),
        lambda: gate_residual(x, x, post_norm="rms", post_bias=v), lambda: gate_residual_norm(x, x, norm=None),
        lambda: gate_residual(x, x, gate=torch.zeros(2, 0, 16, device="cuda")), lambda: gate_residual(x, None)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    for call in (lambda: norm_modulate(x.bfloat16(), out_dtype=F32), lambda: norm_modulate(x.double()),
                 lambda: gate_residual(x.bfloat16(), x), lambda: norm_modulate(x, scale=v.double()),
                 lambda: gate_residual(x.bfloat16(), x.half()), lambda: norm_modulate(x, out_dtype=torch.int8)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(RuntimeError):
        norm_modulate(x.cpu())


WIDE = [2932, 4096, 4252, 5120, 5124, 6144, 7172, 8192]  # ends of ranges in which fewer teams than threads allow have room


@pytest.mark.parametrize("types", [(F32, F32, F32), (F32, BF, F32), (F32, HF, HF), (BF, BF, F32)])
@pytest.mark.parametrize("width", WIDE)
def test_many_wide_rows(width, types):
    """Rows that fill the device with every team a CTA has room for: joins with and without a norm of the branch.
    A row's sums take 16 additions of pairs a thread and at most 1 + 5 + 4 more; their errors have either sign."""
    for form in ((None, False, None, 1.0, True), ("layer", True, None, 0.5, True), ("rms", False, "rms", 1.0, True),
                 ("layer", True, "layer", -0.7, True)):
        test_forward((1, 1500, 1, width), types, form)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("width", [4096, 5124, 8192])
def test_steps_of_many_wide_rows(width, form):
    test_backward((1, 1200, 2, width), (F32, F32, F32), form)


def test_forward_mode_derivatives_are_refused():
    """A dual tensor raises rather than losing its tangent, with and without gradients; so does a transform."""
    from torch.autograd import forward_ad

    from longvideosparseattention_b200.block_norm import gate_residual, gate_residual_norm, norm_modulate
    g = torch.Generator().manual_seed(3)
    x, y, v = _make((1, 4, 64), F32, g), _make((1, 4, 64), F32, g), _make((64,), F32, g)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: norm_modulate(dual(x)), lambda: norm_modulate(x, scale=dual(v)),
                     lambda: gate_residual(x, dual(y)), lambda: gate_residual(x, y, dual(v)),
                     lambda: gate_residual_norm(x, y, weight=dual(v)), lambda: gate_residual_norm(x, y, shift=dual(v)),
                     lambda: gate_residual(x, y, post_norm="layer", post_weight=v, post_bias=dual(v)),
                     lambda: norm_modulate(x.clone().requires_grad_(True), weight=dual(v))):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError):
                    call()
        norm_modulate(x, scale=v)  # none of its tensors is dual
        z = x.clone().requires_grad_(True)
        n = norm_modulate(z)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(n, z, dual(y))
    z = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(norm_modulate(z), z, y[None], is_grads_batched=True)
    with pytest.raises(RuntimeError):
        torch.func.jvp(norm_modulate, (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(norm_modulate)(x[None])
