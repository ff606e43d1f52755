"""The neural shading operators, as cases to measure: group normalisation with an activation over
channels-last images, and dropout whose mask is drawn from a counter and never stored.

A case names the operator, the direction ("forward": the call without gradients; "training": the
call and its gradients), the type, and the image: ``batch`` views of ``height`` x ``width`` pixels
with ``channels`` features. ``extra`` more channels in the buffer make the features a channel slice
of it, as ``interpolate`` returns them beside texture coordinates. The features have the look of
rendered ones: a scale and an offset for each channel, and a background of zeros around the object.

``run`` computes the plain form (elementary torch operations in 32 bits, rounded once at the end)
or, with ``own``, makes the calls of ``diffrast_b200``.
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5
# Elements of the largest image a case may have (the largest listed ones have as many).
LIMIT = 1 << 27


def _norm(name, direction, dtype, batch, height, width, channels, groups, activation="silu",
          dropout=0.0, per_view=False, extra=0):
    return {"name": name, "op": "group_norm", "direction": direction, "dtype": dtype,
            "batch": batch, "height": height, "width": width, "channels": channels,
            "groups": groups, "activation": activation, "dropout": dropout,
            "per_view": per_view, "extra": extra}


def _drop(name, direction, dtype, batch, height, width, channels, dropout, residual):
    return {"name": name, "op": "dropout", "direction": direction, "dtype": dtype,
            "batch": batch, "height": height, "width": width, "channels": channels,
            "dropout": dropout, "residual": residual}


def listed():
    return [
        # A preview tile of an interactive viewer: one small launch, its latency is all.
        _norm("norm tile", "forward", "bf16", 1, 16, 16, 64, 16),
        # The coarsest level of a small network being fitted to two views.
        _norm("norm tile training", "training", "fp32", 2, 24, 24, 48, 6),
        # Four frames of a deferred shader, two channels to a group.
        _norm("norm frames", "forward", "bf16", 4, 512, 512, 64, 32),
        # Features read in place beside texture coordinates, a scale and shift for each view.
        _norm("norm slice per view", "forward", "fp32", 2, 512, 512, 32, 8, "relu",
              per_view=True, extra=8),
        # One megapixel view with wide features: a single view is larger than the L2 cache.
        _norm("norm large view", "forward", "bf16", 1, 1024, 1024, 128, 32),
        # Cropped views of an odd size, six channels to a group.
        _norm("norm ragged training", "training", "fp16", 3, 237, 311, 30, 5),
        # A deep level of the network, with its dropout fused.
        _norm("norm level training", "training", "bf16", 8, 128, 128, 256, 32, dropout=0.1),
        # A training step's full-resolution level over eight views.
        _norm("norm views training", "training", "bf16", 8, 512, 512, 64, 16),
        # The preview tile again, for dropout on its own.
        _drop("dropout tile", "forward", "bf16", 1, 16, 16, 64, 0.1, False),
        # Odd crops with an odd number of channels, added to the skip connection.
        _drop("dropout odd residual", "forward", "fp32", 5, 333, 257, 7, 0.25, True),
        # Sampled neural texture features, regularised while they are fitted.
        _drop("dropout features training", "training", "fp16", 2, 200, 200, 96, 0.5, False),
        # The residual join of a full-resolution level over eight views.
        _drop("dropout views training", "training", "bf16", 8, 512, 512, 64, 0.1, True),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["group_norm", "group_norm", "dropout"])
    direction = rng.choice(["forward", "training"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    batch = _log_uniform(rng, 1, 16)
    height, width = _log_uniform(rng, 8, 1024), _log_uniform(rng, 8, 1024)
    groups = rng.choice([1, 2, 3, 4, 5, 6, 8, 12, 16, 32])
    channels = groups * max(1, min(256 // groups, _log_uniform(rng, 1, 32)))
    if op == "dropout":
        channels = _log_uniform(rng, 1, 256)
    most = LIMIT if dtype != "fp32" else LIMIT // 2
    while batch * height * width * channels > most:
        batch, height, width = max(1, batch // 2), max(1, height * 3 // 4), max(1, width * 3 // 4)
    dropout = rng.choice([0.05, 0.1, 0.25, 0.5])
    if op == "dropout":
        case = _drop("", direction, dtype, batch, height, width, channels, dropout,
                     rng.random() < 0.5)
    else:
        # relu's gradient jumps where a value rounds to the other side of zero, so it is drawn
        # for the forward direction alone.
        activation = rng.choice(["none", "silu", "silu"] + ["relu"] * (direction == "forward"))
        case = _norm("", direction, dtype, batch, height, width, channels, groups, activation,
                     rng.choice([0.0, dropout]), rng.random() < 0.3,
                     rng.choice([0, 0, 0, 8, 4, 1]))
    del case["name"]
    return case


def _features(case, gen):
    """Feature images ``[batch, height, width, channels]``, a slice of a wider buffer with
    ``extra``; the rim of each view, as wide as an eighth of it, is background."""
    b, h, w, c = (case[k] for k in ("batch", "height", "width", "channels"))
    extra = case.get("extra", 0)
    buffer = torch.randn((b, h, w, c + extra), generator=gen, device="cuda",
                         dtype=torch.float32)
    buffer *= torch.rand((c + extra,), generator=gen, device="cuda") + 0.5
    buffer += 0.5 * torch.randn((b, 1, 1, c + extra), generator=gen, device="cuda")
    buffer[:, : h // 8] = 0
    buffer[:, :, : w // 8] = 0
    return buffer.to(DTYPES[case["dtype"]])[..., extra:]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    training = case["direction"] == "training"
    dtype = DTYPES[case["dtype"]]
    x = _features(case, gen)
    state = {"case": case, "x": x.detach().requires_grad_(training)}
    state["seed"] = torch.randint(0, 1 << 62, (1,), generator=gen, device="cuda")
    if training:
        grad = torch.randn(x.shape, generator=gen, device="cuda", dtype=torch.float32)
        state["grad"] = grad.to(dtype)
    if case["op"] == "group_norm":
        c = case["channels"]
        shape = (case["batch"], c) if case["per_view"] else (c,)
        weight = 1 + 0.2 * torch.randn(shape, generator=gen, device="cuda")
        bias = 0.2 * torch.randn(shape, generator=gen, device="cuda")
        state["weight"] = weight.requires_grad_(training)
        state["bias"] = bias.requires_grad_(training)
    elif case["residual"]:
        residual = torch.randn(x.shape, generator=gen, device="cuda", dtype=torch.float32)
        state["residual"] = residual.to(dtype).requires_grad_(training)
    return state


# ---- the framework's calls -----------------------------------------------------------------


def _run_own(state):
    import diffrast_b200 as dr

    case, x = state["case"], state["x"]
    inputs = [x]
    if case["op"] == "group_norm":
        dropout = case["dropout"]
        y = dr.group_norm(x, case["groups"], state["weight"], state["bias"], eps=EPS,
                          activation=case["activation"], dropout=dropout,
                          seed=state["seed"] if dropout else None)
        inputs += [state["weight"], state["bias"]]
    else:
        residual = state.get("residual")
        y = dr.dropout(x, case["dropout"], state["seed"], residual=residual)
        inputs += [residual] if residual is not None else []
    if case["direction"] == "forward":
        return [y]
    return [y.detach(), *torch.autograd.grad(y, inputs, state["grad"])]


# ---- the plain form ------------------------------------------------------------------------

# Philox4x32 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011):
# multipliers and key increments.
PHILOX_M = (0xD2511F53, 0xCD9E8D57)
PHILOX_W = (0x9E3779B9, 0xBB67AE85)
WORD = 0xFFFFFFFF


def threshold(p):
    """Elements whose 16 random bits are below this are dropped."""
    return min(65535, int(math.floor(p * 65536 + 0.5)))


def _keep(count, p, seed):
    """Which of ``count`` elements are kept: the counter of eight elements in a row is their index
    over eight, its four random words give 16 bits to each, low half first."""
    index = torch.arange((count + 7) // 8, device="cuda")
    c0, c1 = index & WORD, index >> 32
    c2, c3 = torch.zeros_like(index), torch.zeros_like(index)
    k0, k1 = seed & WORD, (seed >> 32) & WORD
    for _ in range(10):
        # Products of 32-bit words wrap in signed 64 bits, but keep all their bits.
        p0, p1 = PHILOX_M[0] * c0, PHILOX_M[1] * c2
        c0, c1, c2, c3 = (((p1 >> 32) & WORD) ^ c1 ^ k0, p1 & WORD,
                          ((p0 >> 32) & WORD) ^ c3 ^ k1, p0 & WORD)
        k0, k1 = (k0 + PHILOX_W[0]) & WORD, (k1 + PHILOX_W[1]) & WORD
    words = torch.stack([c0, c1, c2, c3], 1)
    halves = torch.stack([words & 0xFFFF, words >> 16], 2)
    return halves.reshape(-1)[:count] >= threshold(p)


def _kept_scale(p):
    return 65536.0 / (65536 - threshold(p))


def _plain_dropout(state):
    case, x = state["case"], state["x"].detach()
    keep = _keep(x.numel(), case["dropout"], state["seed"]).view(x.shape)
    scale = torch.tensor(_kept_scale(case["dropout"]), device="cuda")
    y = torch.where(keep, x.float() * scale, 0.0)
    residual = state.get("residual")
    if residual is not None:
        y = y + residual.detach().float()
    out = [y.to(x.dtype)]
    if case["direction"] == "training":
        grad = state["grad"]
        out.append(torch.where(keep, grad.float() * scale, 0.0).to(x.dtype))
        if residual is not None:
            out.append(grad)
    return out


def _plain_norm(state):
    case, x = state["case"], state["x"].detach()
    b, c, g = case["batch"], case["channels"], case["groups"]
    pixels = case["height"] * case["width"]
    weight = state["weight"].detach().view(-1, 1, g, c // g)
    bias = state["bias"].detach().view(-1, 1, g, c // g)
    xf = x.float().reshape(b, pixels, g, c // g)
    centred = xf - xf.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt((centred * centred).mean((1, 3), keepdim=True) + EPS)
    normed = centred * rstd
    z = normed * weight + bias
    activation = case["activation"]
    sigmoid = 1 / (1 + torch.exp(-z)) if activation == "silu" else None
    if activation == "silu":
        y = z * sigmoid
    else:
        y = torch.where(z > 0, z, 0.0) if activation == "relu" else z
    keep = None
    if case["dropout"]:
        keep = _keep(x.numel(), case["dropout"], state["seed"]).view(y.shape)
        scale = torch.tensor(_kept_scale(case["dropout"]), device="cuda")
        y = torch.where(keep, y * scale, 0.0)
    out = [y.to(x.dtype).view(x.shape)]
    if case["direction"] == "forward":
        return out
    dz = state["grad"].float().view(y.shape)
    if keep is not None:
        dz = torch.where(keep, dz * scale, 0.0)
    if activation == "silu":
        dz = dz * sigmoid * (1 + z * (1 - sigmoid))
    elif activation == "relu":
        dz = torch.where(z > 0, dz, 0.0)
    dn = dz * weight
    mean_dn = dn.mean((1, 3), keepdim=True)
    mean_dnn = (dn * normed).mean((1, 3), keepdim=True)
    dx = rstd * (dn - mean_dn - normed * mean_dnn)
    dims = (1,) if case["per_view"] else (0, 1)
    return out + [dx.to(x.dtype).view(x.shape),
                  (dz * normed).sum(dims).reshape(state["weight"].shape),
                  dz.sum(dims).reshape(state["bias"].shape)]


def run(state):
    if own:
        return _run_own(state)
    return _plain_norm(state) if state["case"]["op"] == "group_norm" else _plain_dropout(state)


# ---- the definition in 64 bits -------------------------------------------------------------


def _mask64(count, p, seed):
    """The kept elements again, with the 64-bit products built from 16-bit limbs."""
    state = [torch.arange((count + 7) // 8, device="cuda"), 0, 0, 0]
    state[1] = torch.div(state[0], 1 << 32, rounding_mode="floor")
    state[0] = torch.remainder(state[0], 1 << 32)
    state[2:] = [state[0] * 0, state[0] * 0]
    seed = int(seed.item())
    key = [seed % (1 << 32), seed // (1 << 32)]

    def product(word, factor):
        high, low = (word >> 16) * factor, (word & 0xFFFF) * factor
        carry = high + (low >> 16)
        return carry >> 16, ((carry & 0xFFFF) << 16) | (low & 0xFFFF)

    for n in range(10):
        h0, l0 = product(state[0], PHILOX_M[0])
        h1, l1 = product(state[2], PHILOX_M[1])
        round_key = [(k + n * step) % (1 << 32) for k, step in zip(key, PHILOX_W)]
        state = [h1 ^ state[1] ^ round_key[0], l1, h0 ^ state[3] ^ round_key[1], l0]
    bits = torch.empty((state[0].numel(), 8), dtype=torch.int32, device="cuda")
    for n, word in enumerate(state):
        bits[:, 2 * n] = word.remainder(65536)
        bits[:, 2 * n + 1] = torch.div(word, 65536, rounding_mode="floor")
    return bits.flatten()[:count] >= threshold(p)


def exact(case, seed):
    state = prepare(case, seed)
    training = case["direction"] == "training"
    shape = state["x"].shape
    leaves = [state["x"].detach().double().requires_grad_(training)]
    p = case["dropout"]
    mask = None
    if p:
        mask = _mask64(state["x"].numel(), p, state["seed"]).view(shape)
        mask = mask.double().mul_(65536 / (65536 - threshold(p)))
    if case["op"] == "group_norm":
        leaves += [state[k].detach().double().requires_grad_(training) for k in ("weight", "bias")]
        x, weight, bias = leaves
        grouped = x.unflatten(-1, (case["groups"], -1))
        variance, mean = torch.var_mean(grouped, (1, 2, 4), correction=0, keepdim=True)
        z = ((grouped - mean) * (variance + EPS) ** -0.5).flatten(-2)
        views = (-1, 1, 1, case["channels"])
        z = z * weight.view(views) + bias.view(views)
        if case["activation"] == "silu":
            z = z * torch.sigmoid(z)
        elif case["activation"] == "relu":
            z = z.clamp_min(0)
        y = z if mask is None else z * mask
    else:
        y = leaves[0] * mask
        if "residual" in state:
            leaves.append(state["residual"].detach().double().requires_grad_(training))
            y = y + leaves[1]
    if not training:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, leaves, state["grad"].double())]


def work(case):
    elements = case["batch"] * case["height"] * case["width"] * case["channels"]
    size = 4 if case["dtype"] == "fp32" else 2
    training = case["direction"] == "training"
    # Forward reads the image and writes the result; training also reads the result's gradient
    # and writes the image's. The residual is read once more, and its gradient is the result's.
    images = 4 if training else 2
    params, flops = 0, 2
    if case["op"] == "group_norm":
        rows = case["batch"] if case["per_view"] else 1
        params = 2 * rows * case["channels"] * 4 * (2 if training else 1)
        # Statistics 3, normalise and scale 3, silu 4; backward: those again, the derivative and
        # the two sums 8, the result 4.
        flops = 7 + 4 * (case["activation"] == "silu")
        flops = flops + 22 if training else flops
    elif case["residual"]:
        images += 1
    return {"bytes": images * elements * size + params, "flops": flops * elements}
