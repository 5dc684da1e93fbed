"""Performance cases of the feature-image decoder's operators.

A splatting model that carries learned features renders them as channel-last
images (..., H, W, D); a small per-pixel network decodes those images into the
space it is trained in.  ``kind`` names the operator:

  linear    activation(x W^T + b) + residual over the pixels of an image
  norm      group normalisation of channel-last images, then an activation
  quantize  activations written in 8 bits for the backward pass and read back

``train`` is a forward and the backward from the output's gradient, otherwise
the call runs without gradients.  ``checkpoint`` keeps the input for the
backward pass in 8 bits: the gradients then see the value that was kept.

The 8-bit form: 32 neighbouring channels of a pixel share a power of two 2^e,
the smallest with max |x| <= 127 * 2^e and e >= -126; a value is stored as the
nearest integer (ties to even) to x / 2^e and stands for that integer times 2^e.
"""

import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_EPS = 1e-5


def _linear(rows, inner, outer, dtype, **options):
    return dict(dict(kind="linear", rows=rows, inner=inner, outer=outer, dtype=dtype, activation="none",
                     residual=False, train=False, checkpoint=False), **options)


def _norm(images, height, width, channels, groups, dtype, **options):
    return dict(dict(kind="norm", images=images, height=height, width=width, channels=channels, groups=groups,
                     dtype=dtype, activation="silu", train=False, checkpoint=False), **options)


def _quantize(rows, channels, dtype):
    return dict(kind="quantize", rows=rows, channels=channels, dtype=dtype)


def listed():
    return [
        # A viewer asks for the decoded feature of the one pixel under the cursor.
        dict(_linear(1, 32, 512, "float32"), name="linear_pick_1_32_512_f32"),
        # The first layer on a thumbnail-sized view, no gradients.
        dict(_linear(256 * 256, 32, 64, "float32", activation="silu"), name="linear_256x256_32_64_f32"),
        # Training: the layer that widens the rendered 32 channels.
        dict(_linear(1600 * 1200, 32, 128, "bfloat16", activation="gelu", train=True),
             name="linear_train_1600x1200_32_128_bf16"),
        # Training: a residual block's product, its input kept in 8 bits.
        dict(_linear(1600 * 1200, 128, 128, "bfloat16", activation="silu", residual=True, train=True,
                     checkpoint=True), name="linear_train_8bit_1600x1200_128_128_bf16"),
        # The head that fills a teacher's 512 channels, full HD, no gradients.
        dict(_linear(1920 * 1080, 64, 512, "float16"), name="linear_1080p_64_512_f16"),
        # Training on three ragged views: 32 channels and the depth, an odd class count.
        dict(_linear(3 * 801 * 601, 33, 97, "float32", activation="silu", train=True),
             name="linear_train_3x801x601_33_97_f32"),
        # Training: a wide hidden layer, where the products count more than the bytes.
        dict(_linear(637 * 421, 256, 512, "bfloat16", activation="gelu", train=True),
             name="linear_train_637x421_256_512_bf16"),
        # A batch of small scenes seen by two cameras each, no gradients.
        dict(_norm(8, 128, 128, 48, 6, "float16"), name="norm_8x128x128_48_f16"),
        # Training on four full-HD views: the largest images.
        dict(_norm(4, 1080, 1920, 64, 8, "float32", train=True), name="norm_train_4x1080p_64_f32"),
        # Training: the norm of a residual block, its input kept in 8 bits.
        dict(_norm(1, 1200, 1600, 128, 32, "bfloat16", train=True, checkpoint=True),
             name="norm_train_8bit_1600x1200_128_bf16"),
        # Keeping rendered features and the depth of ragged views in 8 bits.
        dict(_quantize(3 * 801 * 601, 33, "float32"), name="quantize_3x801x601_33_f32"),
        # Keeping a hidden layer of a full view in 8 bits.
        dict(_quantize(1600 * 1200, 128, "bfloat16"), name="quantize_1600x1200_128_bf16"),
    ]


def _log_int(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, max(lo, v + rng.randint(-2, 2)))


def _channels(rng, hi):
    """Half the widths are round, half are any."""
    if rng.random() < 0.5:
        return rng.choice([c for c in (8, 16, 32, 48, 64, 96, 128, 192, 256, 384, 512) if c <= hi])
    return _log_int(rng, 3, hi)


def draw(rng):
    kind = rng.choice(("linear", "linear", "linear", "norm", "norm", "quantize"))
    dtype = rng.choice(("float32", "bfloat16", "bfloat16", "float16"))
    train = rng.random() < 0.6
    checkpoint = train and rng.random() < 0.4
    if kind == "linear":
        inner, outer = _channels(rng, 512), _channels(rng, 512)
        most = min(2.5e8 / (inner + outer), (1.5e10 if dtype == "float32" else 3.2e10) / (inner * outer), 2e6)
        rows = _log_int(rng, 1, int(most)) if rng.random() < 0.3 else _log_int(rng, int(most / 64) + 1, int(most))
        return _linear(rows, inner, outer, dtype, activation=rng.choice(("none", "silu", "gelu")),
                       residual=rng.random() < 0.4, train=train, checkpoint=checkpoint)
    channels = _channels(rng, 512)
    if kind == "quantize":
        return _quantize(_log_int(rng, 1000, int(2.4e8 / channels)), channels, dtype)
    groups = rng.choice([g for g in range(1, min(channels, 64) + 1) if channels % g == 0])
    images = rng.choice((1, 1, 2, 3, 4, 8))
    width = _log_int(rng, 64, min(1920, int(math.sqrt(4e8 / images / channels))))
    height = max(32, int(width * rng.uniform(0.5, 0.8)))
    return _norm(images, height, width, channels, groups, dtype, activation=rng.choice(("none", "silu", "gelu")),
                 train=train, checkpoint=checkpoint)


# --------------------------------------------------------------------------
# Inputs


def _image(g, rows, channels, dtype):
    """Feature rows of an image: every channel with a mean and a width of its
    own, faded by the pixel's coverage; one pixel in ten shows nothing."""
    x = torch.randn((rows, channels), generator=g, device="cuda")
    spread = torch.rand((channels,), generator=g, device="cuda") + 0.5
    centre = torch.randn((channels,), generator=g, device="cuda") * 0.5
    cover = (torch.rand((rows, 1), generator=g, device="cuda") * 1.1 - 0.1).clamp_(0, 1)
    return x.mul_(spread).add_(centre).mul_(cover).to(dtype)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)

    state = dict(case)
    if case["kind"] == "quantize":
        state["x"] = _image(g, case["rows"], case["channels"], dtype)
        return state
    train = case["train"]
    if case["kind"] == "linear":
        state["x"] = _image(g, case["rows"], case["inner"], dtype)
        state["weight"] = normal(case["outer"], case["inner"], scale=case["inner"] ** -0.5)
        state["bias"] = normal(case["outer"], scale=0.2)
        shape = (case["rows"], case["outer"])
        if case["residual"]:
            state["residual"] = _image(g, *shape, dtype)
    else:
        shape = (case["images"], case["height"], case["width"], case["channels"])
        state["x"] = _image(g, math.prod(shape[:3]), shape[3], dtype).view(shape)
        state["weight"] = normal(case["channels"], scale=0.2, shift=1.0)
        state["bias"] = normal(case["channels"], scale=0.2)
    if train:
        state["upstream"] = normal(*shape)
        for name in ("x", "weight", "bias", "residual"):
            if name in state and torch.is_tensor(state[name]):
                state[name].requires_grad_(True)
    return state


# --------------------------------------------------------------------------
# One pass


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        if state["kind"] == "linear":
            return _plain_linear(state)
        if state["kind"] == "norm":
            return _plain_norm(state)
        return _plain_quantized(state["x"])


def _run_own(state):
    from dsl_splat_amd import decoding

    if state["kind"] == "quantize":
        return decoding.quantize_activations(state["x"]).dequantize()
    checkpoint = "int8" if state["checkpoint"] else None
    leaves = [state[n] for n in ("x", "weight", "bias")]
    if state["kind"] == "linear":
        residual = state["residual"] if torch.is_tensor(state["residual"]) else None
        y = decoding.linear(*leaves, activation=state["activation"], residual=residual, checkpoint=checkpoint)
        leaves += [residual] if residual is not None else []
    else:
        y = decoding.group_norm(leaves[0], state["groups"], *leaves[1:], eps=_EPS, activation=state["activation"],
                                checkpoint=checkpoint)
    if not state["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, leaves, state["upstream"])]


# --------------------------------------------------------------------------
# The plain form: elementary operations in 32 bits, rounded once at the end


def _activate(z, activation):
    if activation == "silu":
        return z * torch.sigmoid(z)
    if activation == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z


def _slope(z, activation):
    if activation == "silu":
        s = torch.sigmoid(z)
        return s * (1.0 + z * (1.0 - s))
    if activation == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    return torch.ones_like(z)


def _plain_quantized(x):
    rows, channels = x.reshape(-1, x.shape[-1]).shape
    blocks = -(-channels // 32)
    v = torch.zeros((rows, blocks * 32), device=x.device)
    v[:, :channels] = x.reshape(rows, channels)
    v = v.view(rows, blocks, 32)
    mantissa, exponent = torch.frexp(v.abs().amax(-1, keepdim=True))
    # max = mantissa * 2^exponent with mantissa in [0.5, 1): 127 * 2^(exponent-7) covers mantissas up to 127/128.
    e = torch.where(mantissa > 127.0 / 128.0, exponent - 6, exponent - 7).clamp_min(-126)
    e = torch.where(mantissa == 0, -126, e)
    step, inverse = (((n + 127) << 23).to(torch.int32).view(torch.float32) for n in (e, -e))  # 2^e and 2^-e, exactly
    kept = torch.round(v * inverse) * step
    return kept.view(rows, blocks * 32)[:, :channels].reshape(x.shape).to(x.dtype)


def _plain_linear(state):
    dtype = state["x"].dtype
    x, weight, bias = (state[n].float() for n in ("x", "weight", "bias"))
    y = _activate(x @ weight.T + bias, state["activation"])
    if torch.is_tensor(state["residual"]):
        y = y + state["residual"].float()
    if not state["train"]:
        return [y.to(dtype)]
    kept = _plain_quantized(state["x"]).float() if state["checkpoint"] else x
    grad = state["upstream"].float()
    if state["activation"] != "none":
        grad = grad * _slope(kept @ weight.T + bias, state["activation"])
    out = [y.to(dtype), (grad @ weight).to(dtype), (grad.T @ kept).to(dtype), grad.sum(0).to(dtype)]
    return out + ([state["upstream"]] if torch.is_tensor(state["residual"]) else [])


def _plain_norm(state):
    dtype, shape = state["x"].dtype, state["x"].shape
    images, channels, groups = shape[0], shape[3], state["groups"]
    grouped = (images, shape[1] * shape[2], groups, channels // groups)
    x, upstream = state["x"].float().view(grouped), None
    weight, bias = (state[n].float().view(groups, -1) for n in ("weight", "bias"))
    mean = x.mean((1, 3), keepdim=True)
    rstd = torch.rsqrt((x - mean).square().mean((1, 3), keepdim=True) + _EPS)
    y = _activate((x - mean) * rstd * weight + bias, state["activation"]).view(shape).to(dtype)
    if not state["train"]:
        return [y]
    if state["checkpoint"]:
        x = _plain_quantized(state["x"]).float().view(grouped)
    unit = (x - mean) * rstd
    upstream = state["upstream"].float().view(grouped)
    grad = upstream * _slope(unit * weight + bias, state["activation"])
    inner = grad * weight
    dx = rstd * (inner - inner.mean((1, 3), keepdim=True) - unit * (inner * unit).mean((1, 3), keepdim=True))
    return [y, dx.view(shape).to(dtype), (grad * unit).sum((0, 1)).view(-1).to(dtype),
            grad.sum((0, 1)).view(-1).to(dtype)]


# --------------------------------------------------------------------------
# The definition in 64 bits, written apart from the plain form


def _exact_activation(z, activation):
    """Value and derivative of the activation."""
    if activation == "silu":
        gate = 1.0 / (1.0 + torch.exp(-z))
        return z * gate, gate + z * gate * (1.0 - gate)
    if activation == "gelu":
        below = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        return z * below, below + z * torch.exp(-z * z / 2.0) * (2.0 * math.pi) ** -0.5
    return z, torch.ones((), dtype=z.dtype, device=z.device)


def _exact_kept(x):
    """What the 8-bit form of x stands for: block by block of 32 channels."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for c in range(0, x.shape[-1], 32):
        part = x[..., c:c + 32].detach().double()
        largest = part.abs().amax(-1, keepdim=True)
        # The exponent field of the largest magnitude, one step up where 127 steps fall short of it.
        power = ((largest.view(torch.int64) >> 52) - 6).clamp_min(1023 - 126)
        power = torch.where(largest > 127.0 * (power << 52).view(torch.float64), power + 1, power)
        step = (power << 52).view(torch.float64)
        out[..., c:c + 32] = torch.round(part / step) * step
    return out


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "quantize":
            return _exact_kept(state["x"])
        x, weight, bias = (state[n].double() for n in ("x", "weight", "bias"))
        kept = _exact_kept(state["x"]) if case["checkpoint"] else x
        if case["kind"] == "linear":
            y = _exact_activation(torch.addmm(bias, x, weight.T), case["activation"])[0]
            if case["residual"]:
                y += state["residual"].double()
            if not case["train"]:
                return [y]
            slope = _exact_activation(torch.addmm(bias, kept, weight.T), case["activation"])[1]
            grad = state["upstream"].double() * slope
            out = [y, torch.mm(grad, weight), torch.mm(grad.T, kept), torch.sum(grad, 0)]
            return out + ([state["upstream"].double()] if case["residual"] else [])
        n, c, g = case["images"], case["channels"], case["groups"]
        # Groups first: (images, groups, pixels, channels of the group).
        split = lambda t: t.reshape(n, -1, g, c // g).transpose(1, 2)  # noqa: E731
        join = lambda t: t.transpose(1, 2).reshape(state["x"].shape)  # noqa: E731
        gamma, beta = (t.view(1, g, 1, c // g) for t in (weight, bias))
        x = split(x)
        count = x.shape[2] * x.shape[3]
        centre = x.sum((2, 3), keepdim=True) / count
        scale = 1.0 / torch.sqrt(((x - centre) ** 2).sum((2, 3), keepdim=True) / count + _EPS)
        y = join(_exact_activation(gamma * ((x - centre) * scale) + beta, case["activation"])[0])
        if not case["train"]:
            return [y]
        unit = (split(kept) - centre) * scale
        grad = split(state["upstream"].double()) * _exact_activation(gamma * unit + beta, case["activation"])[1]
        pulled = gamma * grad
        along = (pulled * unit).sum((2, 3), keepdim=True) / count
        level = pulled.sum((2, 3), keepdim=True) / count
        return [y, join((pulled - level - unit * along) * scale), (grad * unit).sum((0, 2)).reshape(c),
                grad.sum((0, 2)).reshape(c)]


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "quantize":
        rows, c = case["rows"], case["channels"]
        # Read the activations, write codes and scales, read them, write the values.
        return {"bytes": 2 * size * rows * c + 2 * (rows * c + rows * -(-c // 32)), "flops": 4 * rows * c}
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["inner"], case["outer"]
        values = m * k + n * k + n + m * n * (2 if case["residual"] else 1)
        if case["train"]:
            values += m * n + m * k + n * k + n  # upstream in; the gradients of input, weight and bias out
        return {"bytes": size * values, "flops": 2 * m * k * n * (3 if case["train"] else 1)}
    values = case["images"] * case["height"] * case["width"] * case["channels"]
    return {"bytes": size * (values * (4 if case["train"] else 2) + case["channels"] * (4 if case["train"] else 2)),
            "flops": values * (30 if case["train"] else 10)}
