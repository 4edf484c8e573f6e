"""The operators of a training step, as cases: what each computes in plain torch operations, the calls of
this package that compute the same, and what a pass has to read, write and compute.

  adam        one optimiser step over every tensor of a policy/value network: global gradient norm, clipping,
              Adam (weight decay in the gradient) or AdamW (weight decay on the weights), with moments in
              32 bits or in 8
  norm_act    batch normalisation with the batch's statistics and ReLU, forward and backward
  norm_gate   the end of a squeeze-excitation residual block: batch normalisation, gate and bias computed from
              the board means, residual, ReLU, forward and backward
  loss        soft-target policy cross-entropy + outcome cross-entropy with their gradients

`own` False: elementary torch operations in 32 bits.  `own` True: the package's entry points.
"""
import math

import torch

own = False

DEVICE = "cuda"
PAD = 256                      # every parameter tensor starts at a multiple of this many elements
BETA1, BETA2, ADAM_EPS = 0.9, 0.999, 1e-8
NORM_EPS, MOMENTUM = 1e-5, 0.1
MASK32 = 0xFFFFFFFF

LARGEST_PARAMETERS = 28_000_000
LARGEST_ACTIVATIONS = 4096 * 256 * 64
LARGEST_LOGITS = 8192 * 4001


# ---------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # the network of the trainer's own tests: a step over a few hundred thousand weights is launches and little else
        {"name": "adam 2x32 32-bit", "op": "adam", "blocks": 2, "filters": 32, "ratio": 8, "bits": 32, "decoupled": False, "clip": 1.0},
        # the default network and the trainer's own optimiser settings
        {"name": "adam 20x128 32-bit", "op": "adam", "blocks": 20, "filters": 128, "ratio": 8, "bits": 32, "decoupled": False, "clip": 1.0},
        # the default network with decoupled decay and moments in 8 bits
        {"name": "adamw 20x128 8-bit", "op": "adam", "blocks": 20, "filters": 128, "ratio": 8, "bits": 8, "decoupled": True, "clip": 1.0},
        # the widest network that the inference kernels take, no clipping
        {"name": "adamw 20x256 8-bit", "op": "adam", "blocks": 20, "filters": 256, "ratio": 8, "bits": 8, "decoupled": True, "clip": 0.0},
        # a last, ragged batch on an odd board
        {"name": "norm_act 37x48 9x9 fp16", "op": "norm_act", "n": 37, "c": 48, "h": 9, "w": 9, "hidden": 0, "dtype": "float16", "layout": "nchw"},
        # the first norm of a block at the default batch under autocast
        {"name": "norm_act 1024x128 bf16", "op": "norm_act", "n": 1024, "c": 128, "h": 8, "w": 8, "hidden": 0, "dtype": "bfloat16", "layout": "nchw"},
        # a block's end at the batch and width of the trainer's own tests
        {"name": "norm_gate 32x32 fp32", "op": "norm_gate", "n": 32, "c": 32, "h": 8, "w": 8, "hidden": 4, "dtype": "float32", "layout": "nchw"},
        # the default batch and network, in the default precision
        {"name": "norm_gate 1024x128 fp32", "op": "norm_gate", "n": 1024, "c": 128, "h": 8, "w": 8, "hidden": 16, "dtype": "float32", "layout": "nchw"},
        # the same under autocast, with channels-last activations
        {"name": "norm_gate 1024x128 bf16 nhwc", "op": "norm_gate", "n": 1024, "c": 128, "h": 8, "w": 8, "hidden": 16, "dtype": "bfloat16", "layout": "nhwc"},
        # the widest network at a large batch
        {"name": "norm_gate 4096x256 bf16", "op": "norm_gate", "n": 4096, "c": 256, "h": 8, "w": 8, "hidden": 32, "dtype": "bfloat16", "layout": "nchw"},
        # the loss of the default batch
        {"name": "loss 1024x192 fp32", "op": "loss", "n": 1024, "actions": 192, "dtype": "float32", "masked": False},
        # a game with a large action space (an odd number of actions), legal moves only, some positions without any
        {"name": "loss 8192x4001 bf16 masked", "op": "loss", "n": 8192, "actions": 4001, "dtype": "bfloat16", "masked": True},
    ]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["adam", "norm_act", "norm_gate", "loss"])
    if op == "adam":
        case = {"op": op, "blocks": spread(1, 20), "filters": spread(8, 256), "ratio": rng.choice([1, 2, 4, 8]),
                "bits": rng.choice([32, 8]), "decoupled": rng.choice([False, True]), "clip": rng.choice([0.0, 1.0, 100.0])}
        while sum(math.prod(s) for s in network_shapes(case)) > LARGEST_PARAMETERS:
            case["blocks"] -= 1
        return case
    if op == "loss":
        actions = spread(2, 8000)
        return {"op": op, "n": min(spread(1, 16384), LARGEST_LOGITS // actions), "actions": actions,
                "dtype": rng.choice(["float32", "bfloat16", "float16"]), "masked": rng.choice([False, True])}
    c, h, w = spread(4, 256), rng.randint(3, 19), rng.randint(3, 19)
    if rng.random() < 0.5:
        h = w = 8
    return {"op": op, "n": min(spread(2, 4096), LARGEST_ACTIVATIONS // (c * h * w)), "c": c, "h": h, "w": w,
            "hidden": max(1, c // rng.choice([1, 4, 8])) if op == "norm_gate" else 0,
            "dtype": rng.choice(["float32", "bfloat16", "float16"]), "layout": rng.choice(["nchw", "nhwc"])}


def network_shapes(case):
    """The parameter tensors of a squeeze-excitation residual network for 8 x 8 boards, in order."""
    c, hidden = case["filters"], max(1, case["filters"] // case["ratio"])
    block = [(c, c, 3, 3), (c,), (c,), (c, c, 3, 3), (c,), (c,), (hidden, c), (hidden,), (2 * c, hidden), (2 * c,)]
    return ([(c, 3, 3, 3), (c,), (c,)] + block * case["blocks"] + [(c, c, 3, 3), (c,), (c,), (192, 64 * c), (192,)]
            + [(32, c, 1, 1), (32,), (32,), (128, 2048), (128,), (2, 128), (2,)])


def work(case):
    if case["op"] == "adam":
        p = sum(math.prod(s) for s in network_shapes(case))
        # weight, both moments: read and written; gradient: read.  In 8 bits a moment is a byte and, per 256, a scale
        moment = 8 if case["bits"] == 32 else 2 + 8 / 256
        return {"bytes": p * (12 + 2 * moment), "flops": p * (15 if case["bits"] == 32 else 45)}
    if case["op"] == "loss":
        cells, size = case["n"] * case["actions"], torch.finfo(getattr(torch, case["dtype"])).bits // 8
        # logits and gradients, targets, mask; the outcome's two columns beside them
        return {"bytes": cells * (2 * size + 4 + (1 if case["masked"] else 0)) + case["n"] * 2 * (2 * size + 4), "flops": 8 * cells}
    cells, size = case["n"] * case["c"] * case["h"] * case["w"], torch.finfo(getattr(torch, case["dtype"])).bits // 8
    weights = 3 * case["c"] * case["hidden"]
    # x, gradient of the output, output, gradient of x; with a gate the residual and its gradient too
    return {"bytes": cells * size * (6 if case["op"] == "norm_gate" else 4) + 4 * 2 * weights,
            "flops": (24 if case["op"] == "norm_gate" else 16) * cells + 6 * case["n"] * weights}


# ------------------------------------------------------------------------------------------------ prepare
def prepare(case, seed):
    gen = torch.Generator(DEVICE).manual_seed(seed)
    return {"adam": prepare_adam, "loss": prepare_loss}.get(case["op"], prepare_norm)(case, gen)


def normal(gen, *shape):
    return torch.randn(shape, device=DEVICE, generator=gen)


def uniform(gen, *shape):
    return torch.rand(shape, device=DEVICE, generator=gen)


def prepare_adam(case, gen):
    """Weights, gradients and moments of an optimiser that has run for a while.  A user's tensors are separate
    allocations; here they are views of one buffer, each at a multiple of PAD elements, so that they can be
    compared as one output.  The gaps are zeros and stay zeros."""
    shapes = network_shapes(case)
    sizes = [math.prod(s) for s in shapes]
    starts, total = [], 0
    for k in sizes:
        starts.append(total)
        total += -(-k // PAD) * PAD
    # gradients of one tensor have one magnitude, those of different tensors lie decades apart; some are exactly zero
    scale = 10.0 ** (-5 + 3 * uniform(gen, len(shapes)))
    lengths = torch.tensor([x for k in sizes for x in (k, -(-k // PAD) * PAD - k)], device=DEVICE)
    both = torch.stack((scale, torch.zeros_like(scale)), 1).reshape(-1)
    scale = torch.repeat_interleave(both, lengths, output_size=total)
    p = normal(gen, total) * 0.03 * (scale > 0)
    g = normal(gen, total) * scale * (uniform(gen, total) > 0.05)
    m = normal(gen, total) * scale * 0.3
    v = (scale * (0.3 + uniform(gen, total))) ** 2
    params = []
    for s, k, at in zip(shapes, sizes, starts):
        q = p[at:at + k].view(s).requires_grad_(True)
        q.grad = g[at:at + k].view(s)
        params.append(q)
    state = {"case": case, "params": params, "p": p, "g": g, "t": 400, "lr": 1e-3, "wd": 1e-4, "seed": 17}
    if case["bits"] == 32:
        return {**state, "m": m, "v": v}
    half = torch.full((total,), 0.5, device=DEVICE)
    (state["m"], state["m_scale"]), (state["r"], state["r_scale"]) = to_8_bits(m, half, False), to_8_bits(v.sqrt(), half, True)
    return state


def prepare_norm(case, gen):
    """What autograd holds of a block when its end runs: the convolution's output, the block's input, the
    gradient that arrives, parameters and running statistics."""
    dtype = getattr(torch, case["dtype"])
    n, c, h, w, hidden = (case[k] for k in ("n", "c", "h", "w", "hidden"))
    layout = torch.channels_last if case["layout"] == "nhwc" else torch.contiguous_format

    def laid_out(t):
        return t.to(dtype).contiguous(memory_format=layout)

    spread, centre = 0.5 + uniform(gen, 1, c, 1, 1), normal(gen, 1, c, 1, 1)
    x = laid_out(normal(gen, n, c, h, w) * spread + centre + 0.5 * spread * normal(gen, n, c, 1, 1))
    state = {"case": case, "x": x, "weight": 1 + 0.2 * normal(gen, c), "bias": 0.2 * normal(gen, c),
             "running_mean": 0.1 * normal(gen, c), "running_var": 0.5 + uniform(gen, c)}
    if hidden:
        k1, k2 = c ** -0.5, hidden ** -0.5
        state |= {"residual": laid_out(torch.relu(normal(gen, n, c, h, w))),
                  "fc1_weight": k1 * (2 * uniform(gen, hidden, c) - 1), "fc1_bias": k1 * (2 * uniform(gen, hidden) - 1),
                  "fc2_weight": k2 * (2 * uniform(gen, 2 * c, hidden) - 1), "fc2_bias": k2 * (2 * uniform(gen, 2 * c) - 1)}
    grad = normal(gen, n, c, h, w) * 1e-2
    # No gradient arrives where a ReLU's argument lies within rounding of zero: there both of its slopes are right,
    # and which one a sum of 32-bit terms takes is chance.  About one value in ten thousand, one board in a few hundred.
    y, _, _ = normalised(x.double(), state["weight"].double(), state["bias"].double())
    if hidden:
        inner = y.mean((2, 3)) @ state["fc1_weight"].double().t() + state["fc1_bias"].double()
        e = torch.relu(inner) @ state["fc2_weight"].double().t() + state["fc2_bias"].double()
        y = y * torch.sigmoid(e[:, :c, None, None]) + e[:, c:, None, None] + state["residual"].double()
        grad = grad * (inner.abs() > 1e-5).all(1)[:, None, None, None]
    state["grad"] = laid_out(grad * (y.abs() > 1e-4))
    names = ["x", "weight", "bias"] + (["residual", "fc1_weight", "fc1_bias", "fc2_weight", "fc2_bias"] if hidden else [])
    state["leaves"] = [state[k].requires_grad_(True) for k in names]
    return state


def prepare_loss(case, gen):
    """Logits of a policy and an outcome head; visit distributions over a position's legal moves; who won.  With a
    mask the illegal moves' logits are whatever a program leaves there, and one position in 64 has no legal move."""
    n, a, dtype = case["n"], case["actions"], getattr(torch, case["dtype"])
    policy = normal(gen, n, a) * 2
    legal = uniform(gen, n, a) < max(0.15, 1.5 / a)
    legal[torch.arange(n, device=DEVICE), torch.randint(0, a, (n,), device=DEVICE, generator=gen)] = True
    visits = uniform(gen, n, a) ** 4 * legal + 1e-6 * legal
    if case["masked"]:
        legal[torch.arange(n, device=DEVICE) % 64 == 37] = False
        junk = torch.tensor([math.inf, -math.inf, math.nan, torch.finfo(dtype).min], device=DEVICE)
        policy = torch.where(legal, policy, junk[torch.randint(0, 4, (n, a), device=DEVICE, generator=gen)])
        visits = visits * legal
    targets = visits / visits.sum(1, keepdim=True).clamp(min=1e-12)
    won = torch.randint(0, 2, (n,), device=DEVICE, generator=gen)
    outcome = torch.stack((won, 1 - won), 1).float()
    return {"case": case, "policy": policy.to(dtype).requires_grad_(True), "wl": normal(gen, n, 2).to(dtype).requires_grad_(True),
            "targets": targets, "outcome": outcome, "mask": legal if case["masked"] else None}


# ---------------------------------------------------------------------------------------------------- run
def run(state):
    op = state["case"]["op"]
    if own:
        return {"adam": own_adam, "loss": own_loss}.get(op, own_norm)(state)
    return {"adam": plain_adam, "loss": plain_loss}.get(op, plain_norm)(state)


def own_adam(state):
    case = state["case"]
    if "optimizer" not in state:                    # built once, as a training program does
        from alphazero_amd.optim import FusedAdam
        optimizer = FusedAdam(state["params"], lr=state["lr"], betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=state["wd"],
                              decoupled=case["decoupled"], state_bits=case["bits"], seed=state["seed"])
        held = optimizer.flat_state()
        for name, key in own_names(case):
            held[name].copy_(state[key])
        held["step"].fill_(state["t"])
        state["optimizer"], state["held"] = optimizer, held
    optimizer = state["optimizer"]
    optimizer.step(max_norm=case["clip"] or None)
    got = {key: state["held"][name] for name, key in own_names(case)}
    got["p"] = state["p"]
    if case["clip"]:
        got["norm"] = optimizer.grad_norm
    return got


def own_names(case):
    if case["bits"] == 32:
        return (("exp_avg", "m"), ("exp_avg_sq", "v"))
    return (("exp_avg", "m"), ("exp_avg_scale", "m_scale"), ("exp_rms", "r"), ("exp_rms_scale", "r_scale"))


def own_norm(state):
    from alphazero_amd import ops
    if state["case"]["op"] == "norm_act":
        out = ops.norm_act(state["x"], state["weight"], state["bias"], state["running_mean"], state["running_var"],
                           training=True, momentum=MOMENTUM, eps=NORM_EPS)
    else:
        out = ops.norm_gate_residual(state["x"], state["residual"], state["weight"], state["bias"], state["running_mean"],
                                     state["running_var"], state["fc1_weight"], state["fc1_bias"], state["fc2_weight"],
                                     state["fc2_bias"], training=True, momentum=MOMENTUM, eps=NORM_EPS)
    grads = torch.autograd.grad(out, state["leaves"], state["grad"])
    return {"out": out, "grads": grads, "running_mean": state["running_mean"], "running_var": state["running_var"]}


def own_loss(state):
    from alphazero_amd import ops
    losses = ops.policy_value_loss(state["policy"], state["wl"], state["targets"], state["outcome"], mask=state["mask"])
    return {"losses": losses, "grads": torch.autograd.grad(losses[0], (state["policy"], state["wl"]))}


# ------------------------------------------------------------------------------------------- plain forms
def random_16(state, t, total):
    """Two numbers of 16 bits for every element of this step: an integer mix of seed, step and place."""
    z = (torch.arange(total, device=DEVICE) + (state["seed"] * 0x9E3779B9 + t * 0x85EBCA6B)) & MASK32
    z = ((z ^ (z >> 16)) * 0x7FEB352D) & MASK32
    z = ((z ^ (z >> 15)) * 0x846CA68B) & MASK32
    z = z ^ (z >> 16)
    return (z & 0xFFFF).float() / 65536, (z >> 16).float() / 65536


def to_8_bits(x, u, keep):
    """e4m3 codes and a power of two for each 256 values: the largest of them lands in (224, 448].  A value between
    two codes goes up where `u` (0 to 1) is over the rest of the way: with a random u it is right on average.
    keep: what is not zero does not become zero."""
    top = x.reshape(-1, PAD).abs().amax(1)
    mantissa, exponent = torch.frexp(top)
    exponent = exponent - 9 + (mantissa > 0.875)
    exponent = torch.where(top > 0, exponent.clamp(min=-108), torch.full_like(exponent, -108))
    scale = torch.ldexp(torch.ones_like(top), exponent)
    y = (x.reshape(-1, PAD).abs() / scale[:, None]).reshape(-1)
    place = (torch.frexp(y)[1] - 1).clamp(min=-6) - 3              # the exponent of a code's last place
    q = torch.floor(torch.ldexp(y, -place) + u)
    if keep:
        q = torch.where((y > 0) & (q < 1), torch.ones_like(q), q)
    code = torch.copysign(torch.ldexp(q, place), x)
    return code.to(torch.float8_e4m3fn), scale


def from_8_bits(code, scale):
    return (code.float().reshape(-1, PAD) * scale[:, None]).reshape(-1)


def plain_adam(state):
    case, p, g, lr, wd = state["case"], state["p"], state["g"], state["lr"], state["wd"]
    state["t"] += 1
    t, got = state["t"], {"p": p}
    if case["clip"]:
        got["norm"] = g.double().square().sum().sqrt()
        g = g * (case["clip"] / (got["norm"] + 1e-6)).clamp(max=1.0).float()
        got["norm"] = got["norm"].float()
    if case["decoupled"]:
        new = p * (1 - lr * wd)
    else:
        new = p
        g = g + p * wd
    if case["bits"] == 32:
        m, v = state["m"], state["v"]
    else:
        m, v = from_8_bits(state["m"], state["m_scale"]), from_8_bits(state["r"], state["r_scale"]).square()
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g * g * (1 - BETA2)
    root = v.sqrt()
    new = new - m / (root / math.sqrt(1 - BETA2 ** t) + ADAM_EPS) * (lr / (1 - BETA1 ** t))
    p.detach().copy_(new)
    if case["bits"] == 32:
        return {**got, "m": state["m"].copy_(m), "v": state["v"].copy_(v)}
    u, w = random_16(state, t, p.numel())
    for key, code in zip(("m", "m_scale", "r", "r_scale"), to_8_bits(m, u, False) + to_8_bits(root, w, True)):
        got[key] = state[key].copy_(code)
    return got


def normalised(x, weight, bias):
    mean = x.mean((0, 2, 3))
    var = (x - mean[:, None, None]).square().mean((0, 2, 3))
    y = (x - mean[:, None, None]) / (var + NORM_EPS).sqrt()[:, None, None] * weight[:, None, None] + bias[:, None, None]
    return y, mean, var


def plain_norm(state):
    x, c = state["x"], state["case"]["c"]
    y, mean, var = normalised(x.float(), state["weight"], state["bias"])
    if state["case"]["op"] == "norm_gate":
        inner = torch.relu(y.mean((2, 3)) @ state["fc1_weight"].t() + state["fc1_bias"])
        e = inner @ state["fc2_weight"].t() + state["fc2_bias"]
        gate = 1 / (1 + torch.exp(-e[:, :c]))
        y = y * gate[:, :, None, None] + e[:, c:, None, None] + state["residual"].float()
    out = torch.relu(y).to(x.dtype)
    grads = torch.autograd.grad(out, state["leaves"], state["grad"])
    count = x.numel() // c
    state["running_mean"].copy_(state["running_mean"] * (1 - MOMENTUM) + mean.detach() * MOMENTUM)
    state["running_var"].copy_(state["running_var"] * (1 - MOMENTUM) + var.detach() * (count / (count - 1) * MOMENTUM))
    return {"out": out, "grads": grads, "running_mean": state["running_mean"], "running_var": state["running_var"]}


def cross_entropy(logits, targets, mask):
    z = logits.float()
    if mask is not None:
        z = torch.where(mask, z, torch.zeros_like(z))
    top = (z if mask is None else torch.where(mask, z, torch.full_like(z, -math.inf))).detach().amax(1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    weight = torch.exp(z - top)
    if mask is not None:
        weight = torch.where(mask, weight, torch.zeros_like(weight))
        targets = torch.where(mask, targets, torch.zeros_like(targets))
    total = weight.sum(1, keepdim=True)
    log_p = z - top - torch.log(torch.where(total > 0, total, torch.ones_like(total)))
    return -(targets * log_p).sum() / z.shape[0]


def plain_loss(state):
    policy = cross_entropy(state["policy"], state["targets"], state["mask"])
    outcome = cross_entropy(state["wl"], state["outcome"], None)
    loss = policy + outcome
    return {"losses": (loss, policy, outcome), "grads": torch.autograd.grad(loss, (state["policy"], state["wl"]))}


# -------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"adam": exact_adam, "loss": exact_loss}.get(case["op"], exact_norm)(state)


def exact_adam(state):
    """One step by the formulas; a code by the distance to its neighbours rather than by exponents and floors."""
    case, t, lr, wd = state["case"], state["t"] + 1, state["lr"], state["wd"]
    p, g = state["p"].double(), state["g"].double()
    got = {}
    if case["clip"]:
        got["norm"] = torch.linalg.vector_norm(g)
        g = g * min(1.0, case["clip"] / (float(got["norm"]) + 1e-6))
    if not case["decoupled"]:
        g = g + wd * p
    if case["bits"] == 32:
        m, v = state["m"].double(), state["v"].double()
    else:
        m = state["m"].double() * state["m_scale"].double().repeat_interleave(PAD)
        v = (state["r"].double() * state["r_scale"].double().repeat_interleave(PAD)) ** 2
    m = torch.lerp(g, m, BETA1)
    v = torch.lerp(g ** 2, v, BETA2)
    step = (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)) ** 0.5 + ADAM_EPS)
    got["p"] = p - lr * step - (lr * wd * p if case["decoupled"] else 0)
    if case["bits"] == 32:
        return {**got, "m": m, "v": v}
    codes = torch.arange(127, device=DEVICE, dtype=torch.uint8).view(torch.float8_e4m3fn).double()     # 0 to 448
    mixed = torch.arange(p.numel(), device=DEVICE) + state["seed"] * 0x9E3779B9 + t * 0x85EBCA6B
    for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B), (16, 1)):
        mixed = mixed & MASK32
        mixed = (mixed ^ (mixed >> shift)) * factor
    for key, x, chance in (("m", m, mixed & 0xFFFF), ("r", v.sqrt(), (mixed >> 16) & 0xFFFF)):
        block = x.reshape(-1, PAD)
        top = block.abs().amax(1)
        scale = 2.0 ** torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** -108))).clamp(min=-108)
        y = (block / scale[:, None]).reshape(-1)
        low = torch.searchsorted(codes, y.abs(), right=True) - 1
        high = (low + 1).clamp(max=126)
        gap = torch.where(high > low, codes[high] - codes[low], torch.ones_like(y))
        up = (y.abs() - codes[low]) / gap + chance / 65536 >= 1
        if key == "r":
            up = up | ((low == 0) & (y != 0))
        got[key] = (torch.where(up, codes[high], codes[low]) * torch.sign(y)).float().to(torch.float8_e4m3fn)
        got[key + "_scale"] = scale
    return got


def exact_norm(state):
    """Forward, then the gradients written out by hand."""
    case, c = state["case"], state["case"]["c"]
    x, weight, g = state["x"].double(), state["weight"].double(), state["grad"].double()
    count = x.numel() // c

    def per_channel(v):
        return v.reshape(1, c, 1, 1)

    var, mean = torch.var_mean(x, (0, 2, 3), correction=0)
    inverse = (var + NORM_EPS).rsqrt()
    unit = (x - per_channel(mean)) * per_channel(inverse)
    y = unit * per_channel(weight) + per_channel(state["bias"].double())
    if case["op"] == "norm_gate":
        w1, w2 = state["fc1_weight"].double(), state["fc2_weight"].double()
        squeeze = y.mean((2, 3))
        inner = squeeze @ w1.T + state["fc1_bias"].double()
        e = inner.clamp(min=0) @ w2.T + state["fc2_bias"].double()
        gate = torch.sigmoid(e[:, :c])
        out = (y * gate[:, :, None, None] + e[:, c:, None, None] + state["residual"].double()).clamp(min=0)
        g = g * (out > 0)
        d_e = torch.cat(((g * y).sum((2, 3)) * gate * (1 - gate), g.sum((2, 3))), 1)
        d_inner = (d_e @ w2) * (inner > 0)
        d_y = g * gate[:, :, None, None] + (d_inner @ w1)[:, :, None, None] / (case["h"] * case["w"])
        more = [g, d_inner.T @ squeeze, d_inner.sum(0), d_e.T @ inner.clamp(min=0), d_e.sum(0)]
    else:
        out = y.clamp(min=0)
        d_y, more = g * (out > 0), []
    d_bias, d_weight = d_y.sum((0, 2, 3)), (d_y * unit).sum((0, 2, 3))
    d_x = per_channel(weight * inverse) * (d_y - per_channel(d_bias) / count - unit * per_channel(d_weight) / count)
    return {"out": out, "grads": [d_x, d_weight, d_bias] + more,
            "running_mean": state["running_mean"].double() * (1 - MOMENTUM) + mean * MOMENTUM,
            "running_var": state["running_var"].double() * (1 - MOMENTUM) + var * count / (count - 1) * MOMENTUM}


def exact_loss(state):
    n = state["case"]["n"]
    losses, grads = [], []
    for logits, targets, mask in ((state["policy"], state["targets"], state["mask"]), (state["wl"], state["outcome"], None)):
        kept = torch.ones_like(logits, dtype=torch.bool) if mask is None else mask
        z = logits.double().masked_fill(~kept, -math.inf)
        t = targets.double().masked_fill(~kept, 0.0)
        log_p = torch.nan_to_num(z - torch.logsumexp(z, 1, keepdim=True), nan=0.0, neginf=0.0)
        losses.append(-(t * log_p).sum() / n)
        grads.append((log_p.exp() * t.sum(1, keepdim=True) - t).masked_fill(~kept, 0.0) / n)
    return {"losses": (losses[0] + losses[1], losses[0], losses[1]), "grads": grads}
