"""Linear with 4-bit weights against its definition in 64 bits.

Bounds.  u = 2^-24.  Values of act(x) are rounded to whole numbers, 2^21 at
least for the largest of 64 (32): off by 2^-22 of it at most; sums of products
are exact.  A group's three sums (one a digit, sizes up to 2^0, 2^-7 and 2^-15 of
64 times the largest) take three roundings each and are added over groups in
fp32, in at most 320 steps of a warp and 28 more, most in less than 100: below
(3 + 24) u of the sum of |q| s max|x|, as it grows with its root.
SiLU is off by 8 u of its value."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _make(n, k, group, sdt, seed):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8)
    scales = ((torch.rand(n, -(-k // group), generator=g) + 0.1) / math.sqrt(k)).to(sdt)
    return codes.cuda(), scales.cuda()


def _want(x, codes, scales, group, bias, act):
    """(result in 64 bits, bound of the error before the last rounding)."""
    k = codes.shape[1]
    s = scales.double().repeat_interleave(group, dim=1)[:, :k]
    xd = x.double()
    v = xd * torch.sigmoid(xd) if act else xd
    q = codes.double().abs() * s
    y = v @ (codes.double() * s).t()
    block = min(group, 64)
    most = torch.nn.functional.pad(v.abs(), (0, -k % block)).unflatten(1, (-1, block)).amax(-1)
    most = most.repeat_interleave(block, dim=1)[:, :k]
    size = 2.0 ** -22 * (most @ q.t()) + 27 * U * (most @ q.t())
    if act:
        size = size + 8 * U * (v.abs() @ q.t())
    if bias is not None:
        y = y + bias.double()
        size = size + U * y.abs()
    return y, size


def _check(got, want, size):
    half = torch.finfo(got.dtype).eps / 2
    floor = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    bound = half * want.abs() + size * (1 + half) + floor
    worst = ((got.double() - want).abs() / bound).max()
    assert worst <= 1, f"{float(worst):.2f} of what is allowed"


CASES = [  # m, n, k, group, x, out, scales, act, bias
    (1, 16, 64, 64, BF, BF, BF, None, None), (1, 1, 1, 32, F32, F32, BF, None, F32), (1, 17, 65, 32, BF, F32, HF, "silu", BF),
    (2, 48, 200, 128, HF, HF, HF, None, HF), (3, 1000, 2000, 64, F32, F32, BF, "silu", F32), (8, 256, 1536, 64, BF, F32, BF, None, F32),
    (1, 9216, 1536, 64, BF, BF, BF, "silu", BF), (4, 640, 5120, 32, F32, F32, HF, None, None), (5, 333, 777, 128, HF, F32, BF, "silu", F32),
    (9, 512, 1024, 64, BF, F32, BF, None, BF), (16, 130, 96, 32, HF, HF, BF, "silu", HF), (21, 768, 1536, 128, F32, F32, BF, "silu", None),
    (33, 100, 320, 64, BF, BF, BF, None, BF), (64, 400, 512, 32, HF, F32, BF, "silu", None), (1, 40, 20000, 64, F32, F32, BF, None, None),
    (40, 64, 9000, 128, F32, F32, HF, "silu", F32), (2, 30720, 128, 128, BF, BF, BF, None, BF), (130, 64, 128, 64, BF, BF, BF, None, None)]


@pytest.mark.parametrize("case", CASES)
def test_against_definition(case):
    from longvideosparseattention_b200.linear_w4 import linear_w4, pack_w4
    m, n, k, group, xt, ot, st, act, bt = case
    codes, scales = _make(n, k, group, st, n + k)
    g = torch.Generator().manual_seed(m)
    x = (torch.randn(m, k, generator=g) * 1.5).to(xt).cuda()
    bias = None if bt is None else torch.randn(n, generator=g).to(bt).cuda()
    w = pack_w4(codes, scales, group)
    got = linear_w4(x, w, bias, act, ot)
    assert got.dtype == ot and got.shape == (m, n)
    want, size = _want(x, codes, scales, group, bias, act)
    _check(got, want, size)
    assert torch.equal(got, linear_w4(x, w, bias, act, ot))


def test_every_code_in_every_place():
    """x a unit vector picks a column of W out exactly."""
    from longvideosparseattention_b200.linear_w4 import linear_w4, pack_w4
    n, k = 32, 128
    codes = ((torch.arange(n)[:, None] * 5 + torch.arange(k)[None] * 3) % 16 - 8).to(torch.int8).cuda()
    for group in (32, 64, 128):
        scales = (2.0 ** (torch.arange(n)[:, None] % 4 - torch.arange(k // group)[None] % 3)).bfloat16().cuda()
        w = pack_w4(codes, scales, group)
        want = codes.float() * scales.float().repeat_interleave(group, dim=1)
        for first in range(0, k, 8):
            x = torch.zeros(8, k, device="cuda", dtype=BF)
            x[torch.arange(8), first + torch.arange(8)] = 1
            assert torch.equal(linear_w4(x, w, out_dtype=F32), want[:, first:first + 8].t())


def test_shapes_and_strides():
    from longvideosparseattention_b200.linear_w4 import linear_w4, pack_w4
    codes, scales = _make(96, 192, 64, BF, 3)
    w = pack_w4(codes, scales, 64)
    x = torch.randn(2, 3, 192, device="cuda", dtype=BF)
    y = linear_w4(x, w)
    assert y.shape == (2, 3, 96)
    assert torch.equal(y.view(6, 96), linear_w4(x.view(6, 192), w))
    assert torch.equal(linear_w4(x[0, 0], w), linear_w4(x[0, :1], w)[0])
    wide = torch.randn(5, 400, device="cuda", dtype=BF)
    assert torch.equal(linear_w4(wide[:, 1:193], w), linear_w4(wide[:, 1:193].contiguous(), w))
    assert torch.equal(linear_w4(wide[::2, 3:195], w), linear_w4(wide[::2, 3:195].contiguous(), w))
    assert torch.equal(linear_w4(x[:1, :1].expand(4, 3, 192), w)[3, 2], y[0, 0])
    t = torch.randn(192, 4, device="cuda", dtype=BF).t()
    assert torch.equal(linear_w4(t, w), linear_w4(t.contiguous(), w))
    assert linear_w4(x[:0], w).shape == (0, 3, 96)
    padded = torch.zeros(96, 200, dtype=torch.int8, device="cuda")
    padded[:, :192] = codes
    assert torch.equal(pack_w4(padded[:, :192], scales, 64).tiles, w.tiles)
    assert torch.equal(pack_w4(codes.t().contiguous().t(), scales, 64).tiles, w.tiles)


def test_one_row_with_any_stride():
    """A dimension of one element counts as contiguous whatever its stride is."""
    from longvideosparseattention_b200.linear_w4 import linear_w4, pack_w4
    codes, scales = _make(1, 192, 64, BF, 4)
    w = pack_w4(codes, scales, 64)
    assert torch.equal(pack_w4(codes.clone().as_strided((1, 192), (1, 1)), scales, 64).tiles, w.tiles)
    x = torch.randn(1, 192, device="cuda", dtype=BF)
    want = linear_w4(x, w)
    assert torch.equal(linear_w4(x.view(192, 1).t(), w), want)
    assert torch.equal(linear_w4(x.as_strided((1, 192), (0, 1)), w), want)
    one = pack_w4(codes[:, :1], scales[:, :1], 64)
    assert torch.equal(linear_w4(x.view(192, 1).as_strided((192, 1), (1, 7)), one), linear_w4(x.view(192, 1), one))


def test_quantize():
    """The nearest code: off by at most half a step, and exactly the codes back from what they stand for."""
    from longvideosparseattention_b200.linear_w4 import linear_w4, quantize_w4
    g = torch.Generator().manual_seed(0)
    weight = torch.randn(40, 150, generator=g).cuda()
    weight[3] = 0
    for group in (32, 64, 128):
        w = quantize_w4(weight, group)
        eye = torch.eye(150, device="cuda", dtype=BF)
        back = linear_w4(eye, w, out_dtype=F32).t()
        steps = torch.nn.functional.pad(weight, (0, -150 % group)).unflatten(1, (-1, group)).abs().amax(-1) / 7
        steps = steps.bfloat16().float().repeat_interleave(group, dim=1)[:, :150]
        # half a step, and what clamping at 7 costs where the scale was rounded down (7 x 2^-9 of a step)
        assert ((back - weight).abs() <= steps * (0.5 + 7 * 2.0 ** -8) + 1e-7).all()
        assert (back[3] == 0).all()


def test_offsets_past_32_bits():
    """Weights of more than 2^31 bytes of tiles: the first and the last outputs."""
    from longvideosparseattention_b200.linear_w4 import linear_w4, pack_w4
    n, k, group = 2 ** 18 + 20, 16448, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    codes = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8, device="cuda")
    scales = (torch.rand(n, -(-k // group), generator=g, device="cuda") / 128).bfloat16()
    x = torch.randn(2, k, generator=g, device="cuda")
    y = linear_w4(x, pack_w4(codes, scales, group))
    for part in (slice(0, 40), slice(n - 40, n)):
        want, size = _want(x, codes[part], scales[part], group, None, None)
        _check(y[:, part], want, size)


def test_a_row_of_millions():
    """Bytes of x as digits pass 32 bits.  Values are powers of two and scales 1:
    every sum is a whole number below 2^24, and so exact in any order."""
    from longvideosparseattention_b200.linear_w4 import linear_w4, pack_w4
    m, k = 21, 36_000_065
    codes = torch.randint(-7, 8, (1, k), device="cuda", dtype=torch.int8)
    sums = torch.cumsum(codes[0].long(), 0)
    assert 8 * int(sums.max() - sums.min()) < 2 ** 24
    w = pack_w4(codes, torch.ones(1, -(-k // 128), device="cuda", dtype=BF), 128)
    size = torch.tensor([(-1.0) ** i * 2.0 ** (i % 3) for i in range(m)], device="cuda")
    x = size.to(BF)[:, None].expand(m, k).contiguous()
    assert torch.equal(linear_w4(x, w, out_dtype=F32)[:, 0], size * sums[-1])


def test_infinities_and_large_rows():
    from longvideosparseattention_b200.linear_w4 import linear_w4, pack_w4
    codes, scales = _make(64, 256, 64, BF, 5)
    w = pack_w4(codes, scales, 64)
    x = torch.randn(4, 256, device="cuda")
    clean = linear_w4(x, w)
    x[1, 7], x[3, 9] = float("inf"), float("nan")
    y = linear_w4(x, w)
    assert torch.equal(y[[0, 2]], clean[[0, 2]]) and y[[1, 3]].isnan().all()
    big = torch.full((1, 256), 1e30, device="cuda")
    want, size = _want(big, codes, scales, 64, None, None)
    _check(linear_w4(big, w), want, size)
    low = torch.full((1, 256), -200.0, device="cuda")  # SiLU underflows to zero
    assert (linear_w4(low, w, activation="silu") == 0).all()


def test_streams_graph_and_refusals():
    from longvideosparseattention_b200.linear_w4 import linear_w4, pack_w4, quantize_w4
    codes, scales = _make(512, 640, 64, BF, 6)
    w = pack_w4(codes, scales, 64)
    x, bias = torch.randn(3, 640, device="cuda"), torch.randn(512, device="cuda")
    want = linear_w4(x, w, bias, "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = linear_w4(x, w, bias, "silu")
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = linear_w4(x, w, bias, "silu")
    x.mul_(0.5)
    want = linear_w4(x, w, bias, "silu")
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    for call in (lambda: linear_w4(x[:, :600], w), lambda: linear_w4(x, w, bias[:5]), lambda: linear_w4(x, w, bias.cpu()),
                 lambda: linear_w4(x, w, activation="gelu"), lambda: pack_w4(codes, scales, 16),
                 lambda: pack_w4(codes, scales[:, :3], 64), lambda: pack_w4(codes[0], scales, 64),
                 lambda: pack_w4(codes, scales.cpu(), 64), lambda: quantize_w4(x[0]), lambda: quantize_w4(x, 48)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: linear_w4(x.double(), w), lambda: linear_w4(x, w, out_dtype=torch.float64),
                 lambda: pack_w4(codes.int(), scales, 64), lambda: pack_w4(codes, scales.float(), 64),
                 lambda: quantize_w4(x, scale_dtype=torch.float32)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(RuntimeError):
        linear_w4(x.requires_grad_(True), w)
    with torch.no_grad():
        linear_w4(x, w)
    with pytest.raises(RuntimeError):
        linear_w4(torch.zeros(1, 640), w)


def test_block_of_a_layer():
    """The operators as a layer runs them: time embedding -> vectors, norm, attention, projection, join with the
    norm before the MLP, MLP, join; against the same steps in 64 bits from the same quantised weights, attention and
    projection taken from the framework on both sides (they have tests of their own)."""
    from longvideosparseattention_b200 import block_sparse_attention, build_block_mask
    from longvideosparseattention_b200.block_norm import gate_residual, gate_residual_norm, norm_modulate
    from longvideosparseattention_b200.linear_w4 import linear_w4, quantize_w4
    from longvideosparseattention_b200.out_proj import out_projection
    from longvideosparseattention_b200.prologue import qk_norm_rope
    from tests.block_norm_reference import definition
    T, P, H, D = 5, 160, 4, 128
    C, S = H * D, T * P
    g = torch.Generator().manual_seed(1)
    def mk(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(BF).cuda()
    x, temb = mk(1, S, C), mk(1, T, C)  # a noise level for every frame
    wmod, bmod = quantize_w4(mk(6 * C, C, scale=C ** -0.5)), mk(6 * C, scale=0.1)
    wq, wk, wv, wo = (mk(C, C, scale=C ** -0.5) for _ in range(4))
    w1, w2 = mk(2 * C, C, scale=C ** -0.5), mk(C, 2 * C, scale=C ** -0.5)
    mask = build_block_mask(T, P, 1, 1, 3, 0, True, 0, device=x.device)

    def attention(n):
        q, k, v = (torch.nn.functional.linear(n, w).view(1, S, H, D) for w in (wq, wk, wv))
        qk_norm_rope(q, "rms_head")
        qk_norm_rope(k, "rms_head")
        return out_projection(block_sparse_attention(q, k, v, mask)[0], wo)

    def mlp(n):
        return torch.nn.functional.linear(torch.nn.functional.gelu(torch.nn.functional.linear(n, w1)), w2)

    vectors = linear_w4(temb, wmod, bmod, "silu")
    sh1, sc1, g1, sh2, sc2, g2 = vectors.chunk(6, dim=-1)
    n1 = norm_modulate(x, scale=sc1, shift=sh1)
    y1 = attention(n1)
    h, n2 = gate_residual_norm(x, y1, g1, scale=sc2, shift=sh2)
    y2 = mlp(n2)
    out = gate_residual(h, y2, g2)
    torch.cuda.synchronize()
    # Each step's own inputs, in 64 bits: half a step of bf16 and the fp32 steps' 2^-18 of values below 30.
    for got, want in ((n1, definition(x.double(), norm="layer", scale=sc1.double(), shift=sh1.double())[1]),
                      (h, definition(x.double(), y1.double(), g1.double())[0]),
                      (n2, definition(x.double(), y1.double(), g1.double(), norm="layer", scale=sc2.double(), shift=sh2.double())[1]),
                      (out, definition(h.double(), y2.double(), g2.double())[0])):
        assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * 30).all()
    assert out.shape == x.shape and torch.isfinite(out).all()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 5, 9, 30])
def test_large_values_of_x(m, group):
    """Results in fp32's range though x times the codes alone is not; groups that cancel; and large scales."""
    from longvideosparseattention_b200.linear_w4 import linear_w4, pack_w4
    g = torch.Generator().manual_seed(7)
    n, k = 48, 256
    codes = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8)
    codes[0], codes[1] = 7, -8
    codes[2, :128], codes[2, 128:] = 7, -7
    codes[3, 1::2] = 0
    codes = codes.cuda()
    for xt, size, scale in ((BF, 2.0 ** 120, 2.0 ** -9), (F32, 3e37, 2.0 ** -8), (F32, 3e38, 2.0 ** -12), (F32, 1.0, 2.0 ** 100)):
        scales = torch.full((n, k // group), scale).to(BF).cuda()
        w = pack_w4(codes, scales, group)
        x = (size * (1 - torch.rand(m, k, generator=g) / 8)).to(xt).cuda()
        for act in (None, "silu"):
            want, bound = _want(x, codes, scales, group, None, act)
            assert want.abs().max() < 3.3e38
            _check(linear_w4(x, w, activation=act, out_dtype=F32), want, bound)
        same = linear_w4(torch.full((m, k), size, device="cuda").to(xt), w, out_dtype=F32)
        assert (same[:, 2] == 0).all()


def test_small_values_of_x():
    """Near the low end of fp32's range a value counts to 2^-128 where that is more than 2^-22 of the largest."""
    from longvideosparseattention_b200.linear_w4 import linear_w4, pack_w4
    codes, _ = _make(32, 128, 64, BF, 8)
    scales = torch.full((32, 2), 8.0, device="cuda", dtype=BF)
    w = pack_w4(codes, scales, 64)
    g = torch.Generator().manual_seed(9)
    for power in (-100, -106, -110, -116, -120):
        x = (torch.randn(3, 128, generator=g) * 2.0 ** power).to(BF).cuda()
        want, bound = _want(x, codes, scales, 64, None, None)
        _check(linear_w4(x, w, out_dtype=F32), want, bound + 2.0 ** -128 * 8 * codes.double().abs().sum(-1))


def test_forward_mode_derivatives_are_refused():
    """A dual tensor raises rather than losing its tangent, also without gradients; so does a transform."""
    from torch.autograd import forward_ad

    from longvideosparseattention_b200.linear_w4 import linear_w4, pack_w4
    codes, scales = _make(32, 64, 64, BF, 6)
    w = pack_w4(codes, scales, 64)
    x, bias = torch.randn(2, 64, device="cuda"), torch.randn(32, device="cuda")
    with forward_ad.dual_level():
        for args in ((forward_ad.make_dual(x, torch.ones_like(x)), w), (x, w, forward_ad.make_dual(bias, bias))):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError):
                    linear_w4(*args)
        linear_w4(x, w, bias)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda v: linear_w4(v, w), (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda v: linear_w4(v, w))(x)
