"""The operators around a video transformer's attention block, as they are measured.

A layer of such a model takes its shift, scale and gate vectors from a Linear of the time embedding (one row a sequence,
or one a latent frame), normalises and modulates the residual stream before the block, and joins the block's output to
the stream with a gate, a residual scale and, in sandwich layouts, a norm after the block; the norm before the next
block follows at once.  Cases of four kinds:

  prenorm  n = norm(x) (1 + scale) + shift
  join     h = a x + gate post(y), and n = norm(h) (1 + scale) + shift
  train    one of the two, forward and backward
  w4       the modulation Linear with 4-bit weights and a scale for each group of columns

``run`` computes them from elementary torch operations, or with the framework's kernels where ``own`` is set.
"""

import math

import torch

own = False

EPS = 1e-6
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def _block(name, kind, batch, frames, tokens, width, stream, branch, mod, norm="layer", affine=False, post="none",
           alpha=1.0):
    """``tokens`` a frame; shift, scale and gate [batch, frames, width] of type ``mod``."""
    return dict(name=name, kind=kind, batch=batch, frames=frames, tokens=tokens, width=width, stream=stream,
                branch=branch, mod=mod, norm=norm, affine=affine, post=post, alpha=alpha)


def _linear(name, rows, n, k, group, x, silu, bias, out):
    return dict(name=name, kind="w4", rows=rows, n=n, k=k, group=group, x=x, silu=silu, bias=bias, out=out)


def listed():
    return [
        # The text tokens of a dual-stream layer, two prompts: latency counts.
        _block("prenorm_text", "prenorm", 2, 1, 77, 2048, "bf16", "bf16", "bf16"),
        # One sequence of 81 latent frames x 1560 tokens, vectors of the sequence in fp32.
        _block("prenorm_long", "prenorm", 1, 1, 126360, 1536, "bf16", "bf16", "f32"),
        # The stream kept in fp32, a noise level for every latent frame, the widest model.
        _block("prenorm_frames_f32", "prenorm", 1, 21, 1560, 5120, "f32", "bf16", "f32"),
        # Joint attention, 49 latent frames x 1590 tokens: the join after a block with the next block's norm.
        _block("join_long", "join", 1, 1, 77910, 2048, "bf16", "bf16", "bf16"),
        # Sandwich norms with weights, a prime count of tokens.
        _block("join_sandwich", "join", 2, 1, 4099, 1920, "f16", "f16", "f16", "rms", True, "rms", 0.5),
        # A width that no vector load fits, few tokens.
        _block("join_odd", "join", 1, 5, 67, 1155, "f32", "f32", "f32", "layer", True, "layer"),
        # Fine-tuning step of a join on the training length, 21 latent frames x 1560 tokens, a noise level each.
        _block("train_join", "train_join", 1, 21, 1560, 1536, "bf16", "bf16", "bf16"),
        # Norm with its own weight and bias, all in fp32, two sequences.
        _block("train_prenorm_f32", "train_prenorm", 2, 1, 1001, 1280, "f32", "f32", "f32", "layer", True),
        # The largest step: fp32 stream, sandwich norms.
        _block("train_sandwich", "train_join", 1, 13, 1350, 5120, "f32", "bf16", "f32", "rms", True, "rms"),
        # The modulation of one sequence in the small model: six vectors of 1536.
        _linear("w4_one", 1, 9216, 1536, 64, "bf16", False, True, "bf16"),
        # The widest model, conditional and unconditional row, time embedding in fp32.
        _linear("w4_pair", 2, 30720, 5120, 64, "f32", True, True, "f32"),
        # A row for every latent frame.
        _linear("w4_frames", 49, 12288, 2048, 128, "f16", True, True, "f16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prenorm", "join", "train_prenorm", "train_join", "w4", "w4"])
    if kind == "w4":
        n, k = _log_int(rng, 48, 30720), _log_int(rng, 96, 5120)
        if rng.random() < 0.6:  # most models' widths are multiples of 64
            n, k = (n + 63) // 64 * 64, (k + 63) // 64 * 64
        x = rng.choice(["bf16", "bf16", "f16", "f32"])
        case = _linear("", rng.choice([1, 1, 2, 3, 4, rng.randint(5, 16), rng.randint(17, 64)]), n, k,
                       rng.choice([32, 64, 128]), x, rng.random() < 0.5, rng.random() < 0.5, x)
    else:
        width = _log_int(rng, 256, 5120)
        if rng.random() < 0.8:
            width = (width + 63) // 64 * 64
        elements = _log_int(rng, width, 60_000_000 if kind.startswith("train") else 120_000_000)
        rows = max(1, elements // width)
        frames = rng.choice([1, 1, rng.randint(2, 21)])
        batch = rng.choice([1, 1, 2])
        stream, branch = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"),
                                     ("f32", "f32")])
        joins = kind.endswith("join")
        case = _block("", kind, batch, frames, max(1, rows // (frames * batch)), width, stream, branch,
                      rng.choice(["f32", branch]), rng.choice(["layer", "layer", "rms"]), rng.random() < 0.4,
                      rng.choice(["none", "none", "rms", "layer"]) if joins else "none",
                      rng.choice([1.0, 1.0, 0.7071]) if joins else 1.0)
    del case["name"]
    return case


def _joins(case):
    return case["kind"] in ("join", "train_join")


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "w4":
        codes = s.pop("codes")
        if own:  # the handle that a program makes once from its checkpoint
            from longvideosparseattention_b200.linear_w4 import pack_w4
            s["weight"] = pack_w4(codes, s["scales"], case["group"])
        else:  # two codes a byte, as a checkpoint holds them
            u = torch.nn.functional.pad(codes, (0, case["k"] % 2)).to(torch.uint8) & 15
            s["nibbles"] = u[:, 0::2] | (u[:, 1::2] << 4)
    return s


def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, scale=1.0, at=0.0, dtype="f32"):
        return torch.randn(*shape, generator=gen, device=dev).mul_(scale).add_(at).to(DTYPES[dtype])

    if case["kind"] == "w4":
        n, k, group = case["n"], case["k"], case["group"]
        codes = torch.randn(n, k, generator=gen, device=dev).mul_(2.5).round_().clamp_(-8, 7).to(torch.int8)
        scales = (torch.rand(n, -(-k // group), generator=gen, device=dev) + 0.5) * (0.4 / math.sqrt(k))
        return dict(case=case, codes=codes, scales=scales.to(torch.bfloat16),
                    x=normal(case["rows"], k, dtype=case["x"]),
                    bias=normal(n, scale=0.1, dtype=case["x"]) if case["bias"] else None)

    b, f, p, c = case["batch"], case["frames"], case["tokens"], case["width"]
    train = case["kind"].startswith("train")
    # A residual stream: channels of different size, a few of them large, an offset.
    spread = torch.exp(normal(c, scale=0.5))
    spread[:: max(1, c // 3)] *= 8.0
    s = dict(case=case)
    s["x"] = normal(b, f * p, c).mul_(spread).add_(0.3).to(DTYPES[case["stream"]])
    if _joins(case):
        s["y"] = normal(b, f * p, c, scale=0.7, dtype=case["branch"])
        s["gate"] = normal(b, f, c, scale=0.5, dtype=case["mod"])
        if case["post"] != "none":
            s["post_weight"] = normal(c, scale=0.2, at=1.0, dtype=case["mod"])
        if case["post"] == "layer":
            s["post_bias"] = normal(c, scale=0.1, dtype=case["mod"])
    s["scale"] = normal(b, f, c, scale=0.3, dtype=case["mod"])
    s["shift"] = normal(b, f, c, scale=0.3, dtype=case["mod"])
    if case["affine"]:
        s["weight"] = normal(c, scale=0.2, at=1.0, dtype=case["mod"])
        if case["norm"] == "layer":
            s["bias"] = normal(c, scale=0.1, dtype=case["mod"])
    s["leaves"] = [name for name in ("x", "y", "gate", "post_weight", "post_bias", "scale", "shift", "weight", "bias")
                   if name in s]
    if train:
        s["dn"] = normal(b, f * p, c, dtype=case["branch"])
        if _joins(case):
            s["dh"] = normal(b, f * p, c, dtype=case["stream"])
        for name in s["leaves"]:
            s[name].requires_grad_(True)
    return s


def run(state):
    case = state["case"]
    if case["kind"] == "w4":
        return _own_w4(state) if own else _plain_w4(state)
    return _own_block(state) if own else _plain_block(state)


def _own_w4(s):
    from longvideosparseattention_b200.linear_w4 import linear_w4
    return linear_w4(s["x"], s["weight"], s["bias"], activation="silu" if s["case"]["silu"] else None)


def _own_block(s):
    from longvideosparseattention_b200.block_norm import gate_residual_norm, norm_modulate
    case = s["case"]
    branch = DTYPES[case["branch"]]
    if _joins(case):
        outs = gate_residual_norm(s["x"], s["y"], s["gate"], residual_scale=case["alpha"],
                                  post_norm=None if case["post"] == "none" else case["post"],
                                  post_weight=s.get("post_weight"), post_bias=s.get("post_bias"), post_eps=EPS,
                                  norm=case["norm"], weight=s.get("weight"), bias=s.get("bias"), scale=s["scale"],
                                  shift=s["shift"], eps=EPS)
    else:
        outs = (norm_modulate(s["x"], case["norm"], s.get("weight"), s.get("bias"), s["scale"], s["shift"], EPS,
                              out_dtype=branch),)
    if "dn" not in s:
        return outs
    grads = torch.autograd.grad(outs, [s[name] for name in s["leaves"]], (s["dh"], s["dn"]) if _joins(case) else s["dn"])
    return list(outs) + list(grads)


def _plain_w4(s):
    case = s["case"]
    k, group = case["k"], case["group"]
    u = torch.stack((s["nibbles"] & 15, s["nibbles"] >> 4), dim=-1).flatten(1)[:, :k]
    q = ((u ^ 8).to(torch.float32) - 8.0)
    w = q * s["scales"].float().repeat_interleave(group, dim=1)[:, :k]
    x = s["x"].float()
    if case["silu"]:
        x = x / (1.0 + torch.exp(-x))
    y = x @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(DTYPES[case["out"]])


def _normed(z, kind):
    """(z hat, 1 / deviation) of each row."""
    if kind == "layer":
        z = z - z.mean(-1, keepdim=True)
    r = torch.rsqrt((z * z).mean(-1, keepdim=True) + EPS)
    return z * r, r


def _normed_back(v, zh, r, kind):
    d = v - zh * (v * zh).mean(-1, keepdim=True)
    return r * (d - v.mean(-1, keepdim=True) if kind == "layer" else d)


def _affine(zh, w, b):
    if w is not None:
        zh = zh * w
    return zh if b is None else zh + b


def _plain_block(s):
    case = s["case"]
    with torch.no_grad():
        fwd, saved = _plain_forward(s, case)
        if "dn" not in s:
            return tuple(fwd)
        return fwd + _plain_backward(s, case, saved)


def _vector(s, name):
    """A vector of the channels in 32 bits; [B, F, 1, C] where it is one of each frame."""
    t = s.get(name)
    if t is None:
        return None
    return t.float()[:, :, None] if t.dim() == 3 else t.float()


def _plain_forward(s, case):
    b, f, p, c = case["batch"], case["frames"], case["tokens"], case["width"]
    stream, branch = DTYPES[case["stream"]], DTYPES[case["branch"]]
    z = s["x"].float().view(b, f, p, c)
    outs, yh, yr = [], None, None
    if _joins(case):
        yh = s["y"].float().view(b, f, p, c)
        if case["post"] != "none":
            yh, yr = _normed(yh, case["post"])
        z = case["alpha"] * z + _vector(s, "gate") * _affine(yh, _vector(s, "post_weight"), _vector(s, "post_bias"))
        outs.append(z.view(b, f * p, c).to(stream))
    zh, zr = _normed(z, case["norm"])
    n = _affine(zh, _vector(s, "weight"), _vector(s, "bias")) * (1.0 + _vector(s, "scale")) + _vector(s, "shift")
    outs.append(n.view(b, f * p, c).to(branch))
    return outs, (zh, zr, yh, yr)


def _plain_backward(s, case, saved):
    zh, zr, yh, yr = saved
    shape = zh.shape
    grads = {}
    dn = s["dn"].float().view(shape)
    w, up = _vector(s, "weight"), 1.0 + _vector(s, "scale")
    grads["shift"] = dn.sum(2)
    grads["scale"] = (dn * _affine(zh, w, _vector(s, "bias"))).sum(2)
    u = dn * up
    if case["affine"]:
        grads["weight"] = (u * zh).sum((0, 1, 2))
        if case["norm"] == "layer":
            grads["bias"] = u.sum((0, 1, 2))
        u = u * w
    d = _normed_back(u, zh, zr, case["norm"])
    if _joins(case):
        d = d + s["dh"].float().view(shape)
        w2, g = _vector(s, "post_weight"), _vector(s, "gate")
        grads["gate"] = (d * _affine(yh, w2, _vector(s, "post_bias"))).sum(2)
        e = d * g
        if case["post"] != "none":
            grads["post_weight"] = (e * yh).sum((0, 1, 2))
            if case["post"] == "layer":
                grads["post_bias"] = e.sum((0, 1, 2))
            e = _normed_back(e * w2, yh, yr, case["post"])
        grads["y"] = e
        d = case["alpha"] * d
    grads["x"] = d
    return [grads[name].view(s[name].shape).to(s[name].dtype) for name in s["leaves"]]


def exact(case, seed):
    """The definition in 64 bits, its gradients by differentiation."""
    s = _inputs(case, seed)
    if case["kind"] == "w4":
        w = s["codes"].double()
        w *= s["scales"].double()[:, torch.arange(case["k"], device="cuda") // case["group"]]
        x = s["x"].double()
        if case["silu"]:
            x = x * torch.sigmoid(x)
        y = torch.matmul(x, w.transpose(0, 1))
        return y if s["bias"] is None else y + s["bias"].double()

    b, f, p, c = case["batch"], case["frames"], case["tokens"], case["width"]
    if b * f * p * c > 200_000_000:
        return None
    train = case["kind"].startswith("train")
    v = {name: s[name].detach().double().requires_grad_(train) for name in s["leaves"]}

    def a_row(name):
        return v[name].repeat_interleave(p, dim=1)

    def norm(z, kind, w, bias):
        mean = z.mean(-1, keepdim=True) if kind == "layer" else 0.0
        out = (z - mean) / torch.sqrt(((z - mean) ** 2).mean(-1, keepdim=True) + EPS)
        out = out if w is None else out * w
        return out if bias is None else out + bias

    with torch.set_grad_enabled(train):
        h, outs = v["x"], []
        if _joins(case):
            y = v["y"]
            if case["post"] != "none":
                y = norm(y, case["post"], v["post_weight"], v.get("post_bias"))
            h = h * case["alpha"] + a_row("gate") * y
            outs.append(h)
        n = norm(h, case["norm"], v.get("weight"), v.get("bias"))
        outs.append(n + n * a_row("scale") + a_row("shift"))
        if not train:
            return tuple(outs)
        grads = torch.autograd.grad(outs, list(v.values()), [s[d].double() for d in ("dh", "dn") if d in s])
    return [o.detach() for o in outs] + list(grads)


def work(case):
    if case["kind"] == "w4":
        m, n, k = case["rows"], case["n"], case["k"]
        e = SIZES[case["x"]]
        return {"bytes": n * k / 2 + 2 * n * -(-k // case["group"]) + m * k * e + m * n * SIZES[case["out"]] +
                (n * e if case["bias"] else 0), "flops": 2 * m * n * k}
    e, o, m = SIZES[case["stream"]], SIZES[case["branch"]], SIZES[case["mod"]]
    groups, c = case["batch"] * case["frames"], case["width"]
    elements = groups * case["tokens"] * c
    join, train = _joins(case), case["kind"].startswith("train")
    vectors = groups * c * m * (3 if join else 2) + c * m * (
        (case["affine"] * (2 if case["norm"] == "layer" else 1)) + {"none": 0, "rms": 1, "layer": 2}[case["post"]])
    tensors = (2 * e + 2 * o) if join else (e + o)  # the forward's inputs and outputs
    if train:  # the gradients that come in and go out
        tensors += (2 * e + 2 * o) if join else (e + o)
        vectors *= 2
    return {"bytes": elements * tensors + vectors, "flops": elements * (12 if join else 8) * (3 if train else 1)}
