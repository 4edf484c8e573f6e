"""GPU: the fused norms and the policy/value loss (alphazero_amd.ops) against plain float64 statements of their
formulas, written with gradients by hand.

Tolerances are bounds, not measurements.  Beside every reference value its magnitude is computed: the same formula with
every term's absolute value.  A sum of k float32 terms is off by at most k half-steps (2^-24) of the sum of their
magnitudes, so a result whose longest chain of additions has length k is within about k * 2^-24 * magnitude of the exact
one, plus one rounding to the output's type (eps / 2 of its value).  k below counts the chains: the places of a board,
the boards, the channels and hidden units of the gate's products, and 64 for the rest."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-5


def close(got, want, magnitude, k):
    """|got - want| <= k 2^-24 magnitude + the rounding to got's type."""
    got = got.detach()
    assert got.shape == want.shape and bool(torch.isfinite(got).all())
    info = torch.finfo(got.dtype)
    # below the type's normal range a step no longer shrinks with the value
    bound = k * 2.0 ** -24 * magnitude + info.eps / 2 * want.abs() * (1 + 1e-6) + info.smallest_normal * info.eps
    worst = float(((got.double() - want).abs() / bound).max())
    assert worst <= 1.0, f"{worst:.3g} times the bound"


def norm_reference(t, training, board=None):
    """Forward and gradients in float64, each with its magnitude: {name: (value, magnitude)}."""
    x, weight, bias, g = (t[k].double() for k in ("x", "weight", "bias", "grad"))
    n, c, h, w = x.shape
    hw, m = h * w, n * h * w
    ch = lambda v: v.view(1, c, 1, 1)                                     # noqa: E731
    bc = lambda v: v[:, :, None, None]                                    # noqa: E731
    if training:
        mean = x.mean((0, 2, 3))
        var = (x - ch(mean)).square().mean((0, 2, 3))
    else:
        mean, var = t["running_mean"].double(), t["running_var"].double()
    inv = 1 / (var + EPS).sqrt()
    xc = x - ch(mean)
    # the mean is a sum of the row's differences to one of its values: its magnitude is theirs
    spread = x.amax((0, 2, 3)) - x.amin((0, 2, 3)) if training else torch.zeros_like(mean)
    size = x.abs() + ch(mean.abs() + spread)
    a = weight * inv
    y, y_mag = xc * ch(a) + ch(bias), size * ch(a.abs()) + ch(bias.abs())
    ref = {}
    if "residual" in t:
        w1, b1, w2, b2 = (t[k].double() for k in ("fc1_weight", "fc1_bias", "fc2_weight", "fc2_bias"))
        q, q_mag = y.mean((2, 3)), y_mag.mean((2, 3))
        hid, hid_mag = q @ w1.t() + b1, q_mag @ w1.abs().t() + b1.abs()
        on = hid.clamp(min=0)
        e, e_mag = on @ w2.t() + b2, hid_mag @ w2.abs().t() + b2.abs()
        gate = torch.sigmoid(e[:, :c])
        pre = y * bc(gate) + bc(e[:, c:]) + t["residual"].double()
        pre_mag = y_mag * bc(1 + e_mag[:, :c]) + bc(e_mag[:, c:]) + t["residual"].double().abs()
    else:
        pre, pre_mag, hid = y, y_mag, None
    ref["out"] = (pre.clamp(min=0), pre_mag)
    if training:
        ref["running_mean"] = (0.9 * t["running_mean"].double() + 0.1 * mean, t["running_mean"].double().abs() + mean.abs() + spread)
        ref["running_var"] = (0.9 * t["running_var"].double() + 0.1 * var * m / (m - 1), t["running_var"].double() + var)
    g, g_abs = g * (pre > 0), g.abs()
    if hid is not None:
        s_gy, s_gy_mag, s_g, s_g_mag = (g * y).sum((2, 3)), (g_abs * y_mag).sum((2, 3)), g.sum((2, 3)), g_abs.sum((2, 3))
        slope = gate * (1 - gate)
        de = torch.cat((s_gy * slope, s_g), 1)
        de_mag = torch.cat((s_gy_mag * slope * (1 + e_mag[:, :c]), s_g_mag), 1)
        dhid, dhid_mag = de @ w2 * (hid > 0), de_mag @ w2.abs()
        dq, dq_mag = dhid @ w1, dhid_mag @ w1.abs()
        dy, dy_mag = g * bc(gate) + bc(dq) / hw, g_abs * bc(gate * (1 + e_mag[:, :c])) + bc(dq_mag) / hw
        ref |= {"residual": (g, torch.zeros_like(g)), "fc1_weight": (dhid.t() @ q, dhid_mag.t() @ q_mag), "fc1_bias": (dhid.sum(0), dhid_mag.sum(0)),
                "fc2_weight": (de.t() @ on, de_mag.t() @ hid_mag), "fc2_bias": (de.sum(0), de_mag.sum(0))}
    else:
        dy, dy_mag = g, g_abs
    db, db_mag = dy.sum((0, 2, 3)), dy_mag.sum((0, 2, 3))
    dw, dw_mag = (dy * xc).sum((0, 2, 3)) * inv, (dy_mag * size).sum((0, 2, 3)) * inv
    ref["weight"], ref["bias"] = (dw, dw_mag), (db, db_mag)
    dx, dx_mag = ch(a) * dy, ch(a.abs()) * dy_mag
    if training:
        dx = dx - ch(a) * (ch(db) / m + xc * ch(inv * dw) / m)
        dx_mag = dx_mag + ch(a.abs()) * (ch(db_mag) / m + size * ch(inv * dw_mag) / m)
    ref["x"] = (dx, dx_mag)
    return ref, pre, hid


def norm_inputs(n, c, h, w, hidden, dtype, layout=torch.contiguous_format, seed=0, training=True):
    g = torch.Generator("cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(s, device="cuda", generator=g)           # noqa: E731
    t = {"x": (rn(n, c, h, w) * (0.5 + rn(1, c, 1, 1).abs()) + rn(1, c, 1, 1)).to(dtype).contiguous(memory_format=layout),
         "weight": 1 + 0.2 * rn(c), "bias": 0.2 * rn(c), "running_mean": 0.1 * rn(c), "running_var": 0.5 + rn(c).abs()}
    if hidden:
        t |= {"residual": rn(n, c, h, w).clamp(min=0).to(dtype).contiguous(memory_format=layout), "fc1_weight": rn(hidden, c) * c ** -0.5,
              "fc1_bias": rn(hidden) * 0.3, "fc2_weight": rn(2 * c, hidden) * hidden ** -0.5, "fc2_bias": rn(2 * c) * 0.3}
    t["grad"] = (rn(n, c, h, w) * 0.01).to(dtype)
    # Where a ReLU's argument lies within rounding of zero either slope is right: no gradient arrives there.
    _, pre, hid = norm_reference(t, training)
    keep = pre.abs() > 1e-3
    if hid is not None:
        keep &= (hid.abs() > 1e-4).all(1)[:, None, None, None]
    t["grad"] = (t["grad"] * keep).contiguous(memory_format=layout)
    return t


def run_norm(t, training=True, num_batches=None):
    from alphazero_amd import ops
    names = ["x", "weight", "bias"] + (["residual", "fc1_weight", "fc1_bias", "fc2_weight", "fc2_bias"] if "residual" in t else [])
    leaf = {k: t[k].detach().requires_grad_(True) for k in names}
    stats = t["running_mean"].clone(), t["running_var"].clone()
    if "residual" in t:
        out = ops.norm_gate_residual(leaf["x"], leaf["residual"], leaf["weight"], leaf["bias"], *stats, leaf["fc1_weight"], leaf["fc1_bias"],
                                     leaf["fc2_weight"], leaf["fc2_bias"], num_batches, training=training)
    else:
        out = ops.norm_act(leaf["x"], leaf["weight"], leaf["bias"], *stats, num_batches, training=training)
    got = dict(zip(names, torch.autograd.grad(out, [leaf[k] for k in names], t["grad"])))
    got["out"] = out.detach()
    got["running_mean"], got["running_var"] = stats
    return got


def check_norm(t, training=True):
    got = run_norm(t, training)
    ref, _, _ = norm_reference(t, training)
    n, c, h, w = t["x"].shape
    k = 64 + h * w + c + n + (t["fc1_weight"].shape[0] if "residual" in t else 0)
    for name, (want, magnitude) in ref.items():
        assert got[name].dtype == t[name].dtype if name in t else got[name].dtype == t["x"].dtype
        try:
            close(got[name], want, magnitude, k)
        except AssertionError as e:
            raise AssertionError(f"{name}: {e}") from None
    if not training:
        assert torch.equal(got["running_mean"], t["running_mean"]) and torch.equal(got["running_var"], t["running_var"])
    return got


SIZES = [(2, 1, 1, 1, 0), (1, 5, 1, 2, 0), (3, 7, 3, 3, 0), (2, 4, 8, 8, 1), (33, 32, 8, 8, 4), (5, 40, 9, 9, 5), (1, 64, 8, 8, 8), (7, 130, 1, 1, 16),
         (130, 24, 5, 7, 24), (4, 260, 8, 8, 32), (2, 3, 19, 19, 3), (300, 17, 4, 4, 2), (3, 128, 13, 13, 16), (6, 1024, 2, 3, 70)]


@pytest.mark.parametrize("n, c, h, w, hidden", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", [torch.contiguous_format, torch.channels_last], ids=["nchw", "nhwc"])
def test_norms_against_float64(n, c, h, w, hidden, dtype, layout):
    if dtype != torch.float32 and n * h * w < 9:
        pytest.skip("a variance of two 16-bit values is compared in float32")
    for gated in ([False, True] if hidden else [False]):
        check_norm(norm_inputs(n, c, h, w, hidden if gated else 0, dtype, layout, seed=n + c))


@pytest.mark.parametrize("hidden", [0, 8])
@pytest.mark.parametrize("n", [1, 37])
@pytest.mark.parametrize("layout", [torch.contiguous_format, torch.channels_last], ids=["nchw", "nhwc"])
def test_norms_with_running_statistics(hidden, n, layout):
    for hw in ((1, 1), (8, 8)):
        t = norm_inputs(n, 24, *hw, hidden, torch.float32, layout, seed=3, training=False)
        check_norm(t, training=False)


@pytest.mark.parametrize("hidden", [0, 16])
def test_norms_at_the_default_batch_equal_the_torch_modules(hidden):
    """1024 boards of 128 channels against the model's own modules in float32 (they are the definition): the distance
    is that of two float32 evaluations, 1e-5 of the largest value."""
    from alphazero_amd.model import SEBlock
    t = norm_inputs(1024, 128, 8, 8, hidden, torch.float32)
    got = run_norm(t)
    bn = torch.nn.BatchNorm2d(128).cuda()
    bn.load_state_dict({"weight": t["weight"], "bias": t["bias"], "running_mean": t["running_mean"].clone(),
                        "running_var": t["running_var"].clone(), "num_batches_tracked": torch.zeros((), dtype=torch.int64)})
    x = t["x"].clone().requires_grad_(True)
    if hidden:
        se = SEBlock(128, 8).cuda()
        se.load_state_dict({k.replace("_", "."): t[k] for k in ("fc1_weight", "fc1_bias", "fc2_weight", "fc2_bias")})
        want = torch.relu(se(bn(x)) + t["residual"])
    else:
        want = torch.relu(bn(x))
    want.backward(t["grad"])
    pairs = [(got["out"], want), (got["x"], x.grad), (got["weight"], bn.weight.grad), (got["bias"], bn.bias.grad),
             (got["running_mean"], bn.running_mean), (got["running_var"], bn.running_var)]
    if hidden:
        pairs += [(got["fc1_weight"], se.fc1.weight.grad), (got["fc2_weight"], se.fc2.weight.grad), (got["fc2_bias"], se.fc2.bias.grad)]
    for a, b in pairs:
        assert float((a - b.detach()).abs().max()) <= 1e-5 * float(b.detach().abs().max())


def test_norm_gradient_against_differences():
    """The kernels' gradients along random directions of x, residual and every parameter against central differences of the
    float64 forward pass.  Across a ReLU's border a difference is no derivative: the step is halved until neither a hidden
    unit nor an output that receives gradient changes sides.  Allowed: the chain's half-steps on every gradient's
    magnitude, as above, and step^2 (2^-36) times a third derivative of the derivative's own size for the difference."""
    t = norm_inputs(6, 16, 8, 8, 4, torch.float32, seed=9)
    names = ["x", "residual", "weight", "bias", "fc1_weight", "fc1_bias", "fc2_weight", "fc2_bias"]
    got, (ref, _, _) = run_norm(t), norm_reference(t, True)
    k = 64 + 64 + 16 + 6 + 4
    gen = torch.Generator("cuda").manual_seed(21)

    def at(name, value):
        r, pre, hid = norm_reference({**t, name: value}, True)
        return float((r["out"][0] * t["grad"].double()).sum()), (pre > 0) | (t["grad"] == 0), hid > 0
    for name in names:
        d = torch.randn(t[name].shape, device="cuda", generator=gen, dtype=torch.float64)
        for step in (2.0 ** -j for j in range(18, 26)):
            up, down = at(name, t[name].double() + step * d), at(name, t[name].double() - step * d)
            if torch.equal(up[1], down[1]) and torch.equal(up[2], down[2]):
                break
        else:
            raise AssertionError("a border too near")
        diff = (up[0] - down[0]) / (2 * step)
        along = got[name].double() * d
        allowed = k * 2.0 ** -24 * float((ref[name][1] * d.abs()).sum()) + 1e-6 * float(along.norm())
        assert abs(diff - float(along.sum())) <= allowed, (name, step, diff, float(along.sum()), allowed)


@pytest.mark.parametrize("layout", [torch.contiguous_format, torch.channels_last], ids=["nchw", "nhwc"])
def test_norms_take_any_strides_and_offsets(layout):
    """Slices, permutations, unaligned storage, a gradient in the other layout or expanded: the same numbers."""
    t = norm_inputs(5, 12, 7, 6, 3, torch.bfloat16, layout, seed=2)
    want = run_norm(t)

    def unaligned(v):
        flat = torch.empty(v.numel() + 3, dtype=v.dtype, device="cuda")
        return flat[3:].as_strided(v.size(), v.stride()).copy_(v)

    def sliced(v):
        big = torch.zeros((v.shape[0], v.shape[1], v.shape[2], 2 * v.shape[3]), dtype=v.dtype, device="cuda")
        big[..., ::2] = v
        return big[..., ::2]
    other = torch.channels_last if layout == torch.contiguous_format else torch.contiguous_format
    for change in ({k: unaligned(t[k]) for k in ("x", "residual", "grad")}, {k: sliced(t[k]) for k in ("x", "residual", "grad")},
                   {"grad": t["grad"].contiguous(memory_format=other), "residual": t["residual"].contiguous(memory_format=other)},
                   {"fc1_weight": t["fc1_weight"].t().contiguous().t(), "weight": torch.stack((t["weight"], t["bias"]), 1)[:, 0]}):
        got = run_norm({**t, **change})
        for k in want:
            bound = 0 if got["x"].stride() == want["x"].stride() else 1e-2 * float(want[k].abs().max())     # another order of sums
            assert float((got[k].float() - want[k].float()).abs().max()) <= bound, k
    one = {**t, "grad": torch.ones((), dtype=torch.bfloat16, device="cuda").expand(t["x"].shape)}
    full = {**t, "grad": torch.ones_like(t["x"])}
    a, b = run_norm(one), run_norm(full)
    assert all(torch.equal(a[k], b[k]) for k in a)


def test_norms_are_reproducible_and_leave_their_surroundings_alone():
    """Two calls give the same bits; what lies behind the last board is not touched."""
    t = norm_inputs(9, 20, 9, 9, 5, torch.float16, seed=4)
    a, b = run_norm(t), run_norm(t)
    assert all(torch.equal(a[k], b[k]) for k in a)
    before = {k: v.clone() for k, v in t.items()}
    run_norm(t)
    assert all(torch.equal(before[k], t[k]) for k in t)


def test_norm_statistics_far_from_zero():
    """Values a thousand standard deviations from zero: statistics are taken about a value of the board, so nothing
    cancels.  x is exact in float32; xc / s of size 1 is known to 2^-24 * 1000 (the rounding of x - mean's operands)."""
    t = norm_inputs(64, 8, 8, 8, 0, torch.float32, seed=5)
    t["x"] = 1000.0 + torch.randn(64, 8, 8, 8, device="cuda", generator=torch.Generator("cuda").manual_seed(6))
    got, (ref, _, _) = run_norm(t), norm_reference(t, True)
    want, _ = ref["running_var"]
    assert float((got["running_var"] - want).abs().max()) <= 64 * 2.0 ** -24 * float(want.abs().max())
    assert float((got["out"] - ref["out"][0]).abs().max()) <= 8 * 1000 * 2.0 ** -24 * float(t["weight"].abs().max()) * 2


def test_norms_pass_on_what_is_not_finite():
    """A NaN or an infinity in one channel makes that channel NaN (its statistics are), as in torch, and no other."""
    from alphazero_amd import ops
    for bad in (math.nan, math.inf):
        t = norm_inputs(4, 6, 8, 8, 0, torch.float32)
        t["x"][2, 3, 1, 1] = bad
        out = ops.norm_act(t["x"], t["weight"], t["bias"], t["running_mean"], t["running_var"])
        assert bool(torch.isnan(out[:, 3]).all()) and bool(torch.isfinite(out[:, [0, 1, 2, 4, 5]]).all())
        assert not bool(torch.isfinite(t["running_mean"][3])) and bool(torch.isnan(t["running_var"][3]))


def test_norm_counts_batches_and_moves_versions():
    from alphazero_amd import ops
    t = norm_inputs(4, 6, 8, 8, 0, torch.float32)
    count = torch.full((), 7, dtype=torch.int64, device="cuda")
    versions = [v._version for v in (t["running_mean"], t["running_var"], count)]
    ops.norm_act(t["x"], t["weight"], t["bias"], t["running_mean"], t["running_var"], count)
    assert int(count) == 8 and all(v._version > o for v, o in zip((t["running_mean"], t["running_var"], count), versions))
    ops.norm_act(t["x"], t["weight"], t["bias"], t["running_mean"], t["running_var"], count, training=False)
    assert int(count) == 8


def test_norm_refusals():
    from alphazero_amd import ops
    t = norm_inputs(4, 6, 8, 8, 2, torch.float32)
    s = t["running_mean"], t["running_var"]
    gate = [t[k] for k in ("fc1_weight", "fc1_bias", "fc2_weight", "fc2_bias")]
    w, b, x, r = t["weight"], t["bias"], t["x"], t["residual"]
    for match, call in [
            ("float32, bfloat16 or float16", lambda: ops.norm_act(x.double(), w, b, *s)),
            ("must have shape", lambda: ops.norm_act(x[0], w, b, *s)),
            ("no values", lambda: ops.norm_act(x[:0], w, b, *s)),
            ("more than one value", lambda: ops.norm_act(x[:1, :, :1, :1], w, b, *s)),
            ("weight must have shape", lambda: ops.norm_act(x, w[:5], b, *s)),
            ("bias must be float32", lambda: ops.norm_act(x, w, b.half(), *s)),
            ("bias is on cpu", lambda: ops.norm_act(x, w, b.cpu(), *s)),
            ("running_mean must be", lambda: ops.norm_act(x, w, b, s[0].double(), s[1])),
            ("running_var must be", lambda: ops.norm_act(x, w, b, s[0], torch.ones(12, device="cuda")[::2])),
            ("num_batches_tracked must be", lambda: ops.norm_act(x, w, b, *s, torch.zeros((), device="cuda"))),
            ("needs running statistics", lambda: ops.norm_act(x, w, b, None, None, training=False)),
            ("residual must be like x", lambda: ops.norm_gate_residual(x, r.half(), w, b, *s, *gate)),
            ("residual must be like x", lambda: ops.norm_gate_residual(x, r[:1], w, b, *s, *gate)),
            ("fc2_weight must have shape", lambda: ops.norm_gate_residual(x, r, w, b, *s, gate[0], gate[1], gate[2][:6], gate[3])),
            ("a gate takes up to 1024", lambda: ops.norm_gate_residual(x, r, w, b, *s, torch.zeros(1025, 6, device="cuda"), *gate[1:])),
    ]:
        with pytest.raises((ValueError, TypeError), match=match):
            call()
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(ops.norm_act(leaf, w, b, *s).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("layout", [torch.contiguous_format, torch.channels_last], ids=["nchw", "nhwc"])
def test_norms_of_more_than_2_to_the_31_values(layout):
    """Offsets past 32 bits: with running statistics every board stands for itself, so the first and the last boards of a
    tensor of 2.3e9 values have to be what they are alone, forward and backward, bit for bit."""
    from alphazero_amd import ops
    n, c, h = 4300, 1024, 23
    x = torch.empty((n, c, h, h), dtype=torch.bfloat16, device="cuda", memory_format=layout)
    gen = torch.Generator("cuda").manual_seed(3)
    ends = [slice(0, 2), slice(n - 2, n)]
    x.zero_()
    for e in ends:
        x[e] = torch.randn((2, c, h, h), device="cuda", generator=gen).to(torch.bfloat16)
    t = norm_inputs(2, c, 4, 4, 8, torch.bfloat16, training=False)
    stats, gate = (t["running_mean"], t["running_var"]), [t[k] for k in ("fc1_weight", "fc1_bias", "fc2_weight", "fc2_bias")]

    def both(v):
        leaf = v.detach().requires_grad_(True)
        out = ops.norm_gate_residual(leaf, v, t["weight"], t["bias"], *stats, *gate, training=False)
        return out.detach(), torch.autograd.grad(out, leaf, out.detach())[0]
    assert x.numel() > 2 ** 31
    whole = both(x)
    for e in ends:
        alone = both(x[e].contiguous(memory_format=layout))
        for a, b in zip(whole, alone):
            assert torch.equal(a[e], b)


def test_norm_graph_used_twice_and_shared_arguments():
    """A retained graph gives the same gradients again; one tensor as x and residual gets both gradients, one weight in two
    norms their sum."""
    from alphazero_amd import ops
    t = norm_inputs(6, 10, 8, 8, 3, torch.float32, seed=14)
    x, w = t["x"].clone().requires_grad_(True), t["weight"].clone().requires_grad_(True)
    stats = torch.zeros(10, device="cuda"), torch.ones(10, device="cuda")
    gate = [t[k] for k in ("fc1_weight", "fc1_bias", "fc2_weight", "fc2_bias")]
    out = ops.norm_gate_residual(x, x, w, t["bias"], *stats, *gate)
    first = torch.autograd.grad(out, (x, w), t["grad"], retain_graph=True)
    again = torch.autograd.grad(out, (x, w), t["grad"], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    apart = run_norm({**t, "residual": t["x"]})
    # (a border of the ReLU may lie elsewhere than in norm_inputs: both runs here have the same one)
    assert torch.equal(first[0], apart["x"] + apart["residual"]) and torch.equal(first[1], apart["weight"])
    two = ops.norm_act(ops.norm_act(x, w, t["bias"], *stats), w, t["bias"], *stats)
    y = ops.norm_act(x, w, t["bias"], *stats).detach().requires_grad_(True)
    v = w.detach().clone().requires_grad_(True)
    gy, gv = torch.autograd.grad(ops.norm_act(y, v, t["bias"], *stats), (y, v), t["grad"])
    inner, = torch.autograd.grad(ops.norm_act(x, w, t["bias"], *stats), w, gy)
    assert torch.equal(torch.autograd.grad(two, w, t["grad"])[0], inner + gv)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out = ops.norm_act(x, w, t["bias"], *stats)
        with torch.no_grad():
            w.mul_(2)
        out.backward(t["grad"])


# ------------------------------------------------------------------------------------------------ the loss
def loss_reference(policy, wl, target_pis, target_wls, mask, upstream=(1.0, 0.0, 0.0)):
    """Losses and gradients in float64, with magnitudes."""
    n = policy.shape[0]
    values, mags, grads, grad_mags = [], [], [], []
    for z, t, keep, up in ((policy, target_pis, mask, upstream[0] + upstream[1]), (wl, target_wls, None, upstream[0] + upstream[2])):
        keep = torch.ones_like(z, dtype=torch.bool) if keep is None else keep.bool()
        z, t = z.double().masked_fill(~keep, -math.inf), t.double().masked_fill(~keep, 0)
        top = z.amax(1, keepdim=True)
        top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
        e = torch.exp(z - top)
        S = e.sum(1, keepdim=True)
        log_s = torch.where(S > 0, S, torch.ones_like(S)).log()
        below = torch.where(t != 0, t * (top - z), torch.zeros_like(z))
        row = (t.sum(1, keepdim=True) * log_s).squeeze(1) + below.sum(1)
        values.append(row.sum() / n)
        mags.append((t.abs().sum(1) * (1 + log_s.squeeze(1).abs()) + below.abs().sum(1)).sum() / n)
        p = torch.where(S > 0, e / S, torch.zeros_like(e))
        far = torch.where(e > 0, (top - z).clamp(max=200), torch.zeros_like(z))            # exp(-d) in float32 is off by d half-steps
        grads.append((p * t.sum(1, keepdim=True) - t) * up / n)
        grad_mags.append((p * (1 + far) * t.abs().sum(1, keepdim=True) + t.abs()) * abs(up) / n)
    return (values[0] + values[1], values[0], values[1]), (mags[0] + mags[1], mags[0], mags[1]), grads, grad_mags


def loss_inputs(n, actions, dtype, masked, outcomes=2, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    z = torch.randn(n, actions, device="cuda", generator=g) * 3
    legal = torch.rand(n, actions, device="cuda", generator=g) < 0.3
    t = torch.rand(n, actions, device="cuda", generator=g) * legal
    if masked:
        legal[::3] = False                                             # every third row has nothing
        if n > 1:
            legal[1] = True                                            # one has everything
        junk = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).min], device="cuda")
        z = torch.where(legal, z, junk[torch.arange(n * actions, device="cuda").reshape(n, actions) % 4])
        t = torch.where(legal, t, torch.full_like(t, math.nan))        # targets under the mask are not looked at either
    else:
        t[::4] = 0                                                     # rows without any target
    wl = torch.randn(n, outcomes, device="cuda", generator=g)
    tw = torch.rand(n, outcomes, device="cuda", generator=g)
    return z.to(dtype), wl.to(dtype), t, tw / tw.sum(1, keepdim=True), legal if masked else None


@pytest.mark.parametrize("n, actions", [(1, 1), (1, 2), (3, 192), (64, 192), (5, 255), (7, 1024), (3, 1025), (65, 4001), (2, 20000), (1000, 9), (257, 363)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masked", [False, True])
def test_loss_against_float64(n, actions, dtype, masked):
    from alphazero_amd import ops
    z, wl, t, tw, mask = loss_inputs(n, actions, dtype, masked, outcomes=2 + n % 3, seed=actions)
    z.requires_grad_(True), wl.requires_grad_(True)
    losses = ops.policy_value_loss(z, wl, t, tw, mask)
    up = (0.5, 2.0, -3.0)                                              # all three are differentiable
    got = torch.autograd.grad(sum(u * v for u, v in zip(up, losses)), (z, wl))
    # an upstream that is not 1 may cost a second rounding of the gradient: one more half-step, in the magnitude's bound
    want, mags, grads, grad_mags = loss_reference(z.detach(), wl.detach(), t, tw, mask, up)
    k = 64 + -(-actions // 64) + 8
    for a, b, m in zip(losses, want, mags):
        assert a.dtype == torch.float32 and a.shape == ()
        close(a, b, m, k)
    extra = torch.finfo(dtype).eps / 2 / 2.0 ** -24 if dtype != torch.float32 else 1
    for a, b, m in zip(got, grads, grad_mags):
        assert a.dtype == dtype
        close(a, b, m, k + extra)
    if masked:
        assert bool((got[0][~mask] == 0).all())


def test_loss_of_positions_without_a_legal_move_only():
    from alphazero_amd import ops
    z = torch.full((4, 70), math.nan, device="cuda", requires_grad=True)
    wl = torch.zeros(4, 2, device="cuda", requires_grad=True)
    tw = torch.tensor([[1.0, 0.0]] * 4, device="cuda")
    loss, pi, w = ops.policy_value_loss(z, wl, torch.full((4, 70), math.nan, device="cuda"), tw, torch.zeros(4, 70, dtype=torch.bool, device="cuda"))
    loss.backward()
    assert float(pi) == 0.0 and abs(float(w) - math.log(2)) < 1e-6 and float(loss) == float(w)
    assert bool((z.grad == 0).all()) and torch.equal(wl.grad, torch.tensor([[-0.125, 0.125]] * 4, device="cuda"))


def test_loss_at_the_ends_of_the_range():
    """Illegal moves held at minus infinity or at the type's lowest value, without a mask: probability zero, no NaN as
    long as their target is zero; a target on such a move is an infinite loss; a NaN logit is passed on."""
    from alphazero_amd import ops
    wl, tw = torch.zeros(1, 2, device="cuda"), torch.tensor([[0.5, 0.5]], device="cuda")
    t = torch.tensor([[0.5, 0.5, 0.0, 0.0]], device="cuda")
    for dtype in DTYPES:
        for low in (-math.inf, torch.finfo(dtype).min):
            z = torch.tensor([[1.0, 1.0, low, low]], dtype=dtype, device="cuda", requires_grad=True)
            _, pi, _ = ops.policy_value_loss(z, wl.to(dtype), t, tw)
            assert abs(float(pi) - math.log(2)) < 1e-6
            assert torch.autograd.grad(pi, z)[0].tolist() == [[0.0, 0.0, 0.0, 0.0]]
    z = torch.tensor([[1.0, -math.inf, 0.0, 0.0]], device="cuda")
    assert float(ops.policy_value_loss(z, wl, t, tw)[1]) == math.inf
    z = torch.tensor([[1.0, math.nan, 0.0, 0.0]], device="cuda")
    assert math.isnan(float(ops.policy_value_loss(z, wl, t, tw)[0]))
    for row in ([0.0, 0.0, 3e38, -3e38], [-3e38] * 4):                 # differences beyond float32
        z = torch.tensor([row], device="cuda")
        assert math.isfinite(float(ops.policy_value_loss(z, wl, torch.tensor([[0.0, 0.0, 1.0, 0.0]], device="cuda"), tw)[1]))


def test_loss_equals_the_trainers_own():
    """distributed.losses is the definition; two float32 evaluations of it."""
    from alphazero_amd import ops
    from alphazero_amd.distributed import losses
    z, wl, t, tw, _ = loss_inputs(128, 192, torch.float32, False)
    t = torch.softmax(t, 1)
    leaves = [v.clone().requires_grad_(True) for v in (z, wl)]
    want = losses(lambda _: tuple(leaves), None, t, tw)
    mine = [v.clone().requires_grad_(True) for v in (z, wl)]
    got = ops.policy_value_loss(*mine, t, tw)
    for a, b in zip(got, want):
        assert abs(float(a.detach()) - float(b.detach())) <= 1e-6 * abs(float(b.detach()))
    want[0].backward()
    got[0].backward()
    for a, b in zip(mine, leaves):
        assert float((a.grad - b.grad).abs().max()) <= 1e-6 * float(b.grad.abs().max())


def test_loss_gradient_twice_and_in_parts():
    """A retained graph gives the same gradient again; gradients of the parts add up to the whole's."""
    from alphazero_amd import ops
    for dtype in DTYPES:
        z, wl, t, tw, mask = loss_inputs(33, 300, dtype, True)
        z.requires_grad_(True), wl.requires_grad_(True)
        loss, pi, w = ops.policy_value_loss(z, wl, t, tw, mask)
        a = torch.autograd.grad(loss, (z, wl), retain_graph=True)
        kept = [v.clone() for v in a]
        b = torch.autograd.grad(loss, (z, wl), retain_graph=True)
        c = torch.autograd.grad(pi, z, retain_graph=True)[0], torch.autograd.grad(w, wl, retain_graph=True)[0]
        twice = torch.autograd.grad(loss, (z, wl), torch.full_like(loss, 2.0))
        for u, v, s, x in zip(kept, b, c, twice):
            assert torch.equal(u, v) and torch.equal(u, s)
            # doubling is exact but for values below the type's normal range
            assert float((x - 2 * u).abs().max()) <= 2 * torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert all(torch.equal(u, v) for u, v in zip(a, kept))           # the first answer was not written again


def test_loss_takes_strides_and_broadcast_targets():
    from alphazero_amd import ops
    z, wl, t, tw, mask = loss_inputs(20, 77, torch.float32, True)
    want = ops.policy_value_loss(z, wl, t, tw, mask)
    big = torch.zeros(20, 154, device="cuda")
    big[:, ::2] = z
    wide = torch.zeros(77, 20, dtype=torch.uint8, device="cuda")
    wide.copy_(mask.t())
    got = ops.policy_value_loss(big[:, ::2], wl, t, tw, wide.t())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = torch.full((1, 77), 1 / 77, device="cuda")
    a = ops.policy_value_loss(z, wl, one.expand(20, 77), tw, mask)
    b = ops.policy_value_loss(z, wl, one.repeat(20, 1), tw, mask)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_loss_refusals():
    from alphazero_amd import ops
    z, wl, t, tw, _ = loss_inputs(4, 9, torch.float32, False)
    ok = torch.ones(4, 9, dtype=torch.bool, device="cuda")
    for match, args in [("must be both", (z.double(), wl.double(), t, tw)), ("must be both", (z, wl.half(), t, tw)),
                        (r"\[n, actions\]", (z[0], wl, t, tw)), (r"\[n, actions\]", (z, wl[:3], t, tw)), ("no rows", (z[:0], wl[:0], t[:0], tw[:0])),
                        ("target_pis must be float32", (z, wl, t.double(), tw)), ("target_pis must have", (z, wl, t[:, :8], tw)),
                        ("target_wls must have", (z, wl, t, tw[:, :1])), ("not require", (z, wl, t.clone().requires_grad_(True), tw)),
                        ("mask must be", (z, wl, t, tw, ok.float())), ("mask must be", (z, wl, t, tw, ok[:, :8])),
                        ("all tensors must be on", (z, wl, t.cpu(), tw)), ("up to 4096", (z, torch.zeros(4, 4097, device="cuda"), t, torch.zeros(4, 4097, device="cuda")))]:
        with pytest.raises((ValueError, TypeError), match=match):
            ops.policy_value_loss(*args)


def test_operators_on_a_side_stream_and_in_a_graph():
    """The calls run on the current stream, and replays of a captured forward and backward follow their inputs; every
    replay is compared with the eager call, with eager work and synchronisation between them."""
    from alphazero_amd import ops
    t = norm_inputs(16, 12, 8, 8, 3, torch.bfloat16, seed=1)
    z, wl, tp, tw, mask = loss_inputs(16, 192, torch.float32, True)
    names = ["x", "residual", "weight", "bias", "fc1_weight", "fc1_bias", "fc2_weight", "fc2_bias"]
    leaves = [t[k].clone().requires_grad_(True) for k in names] + [z.clone().requires_grad_(True), wl.clone().requires_grad_(True)]
    stats = torch.zeros(12, device="cuda"), torch.ones(12, device="cuda")

    def work():
        out = ops.norm_gate_residual(*leaves[:4], *stats, *leaves[4:8])
        loss, _, _ = ops.policy_value_loss(leaves[8], leaves[9], tp, tw, mask)
        return [out, loss] + list(torch.autograd.grad((out, loss), leaves, (t["grad"], torch.ones_like(loss)))) + [s.clone() for s in stats]

    def reset():
        stats[0].zero_()
        stats[1].fill_(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        reset()
        first = [v.detach().clone() for v in work()]
    torch.cuda.current_stream().wait_stream(side)
    reset()
    assert all(torch.equal(a, b) for a, b in zip(first, work()))
    graph = torch.cuda.CUDAGraph()
    reset()
    with torch.cuda.graph(graph):
        held = [v.detach() for v in work()]
    gen = torch.Generator("cuda").manual_seed(8)
    for _ in range(4):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(leaves[0].shape, device="cuda", generator=gen).to(torch.bfloat16))
            leaves[8].copy_(torch.where(mask, torch.randn(leaves[8].shape, device="cuda", generator=gen), leaves[8]))
        reset()
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in held]
        reset()
        assert all(torch.equal(a, b.detach()) for a, b in zip(got, work()))


def test_losses_are_tensors_of_their_own():
    """Each of the three may be changed in place (a regulariser added, a factor taken) without touching the others."""
    from alphazero_amd import ops
    z, wl, t, tw, _ = loss_inputs(7, 30, torch.float32, False)
    z.requires_grad_(True)
    want = [v.detach().clone() for v in ops.policy_value_loss(z, wl, t, tw)]
    plain, = torch.autograd.grad(ops.policy_value_loss(z, wl, t, tw)[0], z)
    loss, pi, w = ops.policy_value_loss(z, wl, t, tw)
    loss += 1.0
    loss *= 2.0
    assert torch.equal(loss.detach(), (want[0] + 1.0) * 2.0) and torch.equal(pi.detach(), want[1]) and torch.equal(w.detach(), want[2])
    assert torch.equal(torch.autograd.grad(loss, z)[0], 2 * plain)


def test_a_head_whose_loss_is_not_used_gets_no_gradient():
    from alphazero_amd import ops
    for dtype in DTYPES:
        z, wl, t, tw, _ = loss_inputs(7, 30, dtype, False)
        wl[0, 0] = math.inf
        z.requires_grad_(True), wl.requires_grad_(True)
        _, pi, _ = ops.policy_value_loss(z, wl, t, tw)
        got = torch.autograd.grad(pi, (z, wl), allow_unused=True)
        assert got[1] is None and bool(torch.isfinite(got[0]).all())
        _, _, w = ops.policy_value_loss(z, wl, t, tw)
        assert torch.autograd.grad(w, (z, wl), allow_unused=True)[0] is None


def test_capture_beside_an_eager_graph_is_refused():
    """An eager graph of the same leaves on the default stream: the forward pass says so, before a backward pass could
    accumulate on a stream that is not part of the capture.  Without it the same capture works."""
    from alphazero_amd import ops
    t = norm_inputs(4, 6, 8, 8, 2, torch.float32)
    z, wl, tp, tw, _ = loss_inputs(4, 30, torch.float32, False)
    w, z = t["weight"].clone().requires_grad_(True), z.requires_grad_(True)
    stats = torch.zeros(6, device="cuda"), torch.ones(6, device="cuda")
    calls = [lambda: ops.norm_act(t["x"], w, t["bias"], *stats), lambda: ops.policy_value_loss(z, wl, tp, tw)[0]]
    for call in calls:
        alive = call()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(ValueError, match="eager graph of the same leaf"):
            with torch.cuda.graph(graph):
                call()
        with torch.no_grad():
            call()                                   # (no graph: nothing to refuse)
        del alive
        leaf = w if call is calls[0] else z
        leaf.grad = None
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call().sum().backward()
        want, = torch.autograd.grad(call().sum(), leaf)
        for _ in range(3):
            leaf.grad.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(leaf.grad, want)


def test_operators_in_inference_mode_and_beside_each_other_in_threads():
    """No graph is kept in inference mode, the statistics move all the same; two threads on streams of their own get what one
    gets."""
    import threading
    from alphazero_amd import ops
    t = norm_inputs(9, 10, 8, 8, 4, torch.float32, seed=5)
    gate = [t[k] for k in ("fc1_weight", "fc1_bias", "fc2_weight", "fc2_bias")]
    z, wl, tp, tw, mask = loss_inputs(9, 50, torch.float32, True)

    def work():
        x, r, logits = (v.detach().clone().requires_grad_(True) for v in (t["x"], t["residual"], z))
        stats = torch.zeros(10, device="cuda"), torch.ones(10, device="cuda")
        out = ops.norm_gate_residual(x, r, t["weight"], t["bias"], *stats, *gate)
        loss = ops.policy_value_loss(logits, wl, tp, tw, mask)[0]
        return [out, loss] + list(torch.autograd.grad((out, loss), (x, r, logits), (t["grad"], torch.ones_like(loss)))) + list(stats)
    want = [v.detach() for v in work()]
    with torch.inference_mode():
        stats = torch.zeros(10, device="cuda"), torch.ones(10, device="cuda")
        out = ops.norm_gate_residual(t["x"], t["residual"], t["weight"], t["bias"], *stats, *gate)
        loss = ops.policy_value_loss(z, wl, tp, tw, mask)[0]
        assert not out.requires_grad and not loss.requires_grad
        assert all(torch.equal(a, b) for a, b in zip((out, loss, *stats), (want[0], want[1], *want[-2:])))
    torch.cuda.synchronize()
    wrong = []

    def run():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                if not all(torch.equal(a.detach(), b) for a, b in zip(work(), want)):
                    wrong.append(1)
    threads = [threading.Thread(target=run) for _ in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


@pytest.mark.parametrize("outcomes", [1, 3, 300])
def test_loss_of_other_outcome_counts_and_mask_bytes(outcomes):
    """Any number of outcomes; a byte mask counts what is not zero."""
    from alphazero_amd import ops
    z, wl, t, tw, mask = loss_inputs(21, 45, torch.float32, True, outcomes=outcomes)
    z.requires_grad_(True), wl.requires_grad_(True)
    a = ops.policy_value_loss(z, wl, t, tw, mask)
    b = ops.policy_value_loss(z, wl, t, tw, mask.to(torch.uint8) * 200)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    logp = torch.log_softmax(wl.detach().double(), 1)
    want = -(tw.double() * logp).sum(1).mean()
    # a term of the sum is t (m - z) and T log S: each a few roundings of its magnitude
    magnitude = float((tw.double().abs() * (wl.detach().double().amax(1, keepdim=True) - wl.detach().double())).sum(1).mean() + math.log(outcomes + 1))
    assert abs(float(a[2].detach()) - float(want)) <= (outcomes + 16) * 2.0 ** -24 * magnitude
    g, = torch.autograd.grad(a[2], wl)
    exact = (logp.exp() * tw.double().sum(1, keepdim=True) - tw.double()) / 21
    # exp's argument is off by its own rounding, 2^-24 |z - m|, the sum by outcomes roundings
    spread = float((wl.detach().amax(1) - wl.detach().amin(1)).max())
    assert float((g.double() - exact).abs().max()) <= (spread + outcomes + 16) * 2.0 ** -24 * 2 / 21 * max(1.0, float(tw.sum(1).max()))


@pytest.mark.parametrize("n, c, h, w", [(64, 3, 8, 8), (65, 3, 8, 8), (128, 2, 8, 8), (129, 2, 8, 8), (256, 5, 8, 8), (257, 5, 8, 8), (512, 9, 8, 8),
                                        (513, 9, 8, 8), (1024, 4, 8, 8), (1025, 4, 8, 8), (390, 17, 9, 9), (391, 17, 9, 9), (745, 2, 9, 9),
                                        (1200, 6, 2, 2), (2, 3, 120, 151), (3, 2, 40, 53), (40, 8, 30, 31), (1, 2, 181, 190), (5, 9, 1, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_plain_norms_around_what_a_workgroup_holds(n, c, h, w, dtype):
    """Channels that just fit 1024, 4096 and 8192 pieces of 16 bytes and that just do not, rows that end inside a piece, long ones."""
    t = norm_inputs(n, c, h, w, 0, dtype, seed=n + h)
    check_norm(t)
    if n % 2:
        check_norm(norm_inputs(n, c, h, w, 0, dtype, seed=n + h + 1, training=False), training=False)


@pytest.mark.parametrize("n, c, h, w, hidden", [(2, 3, 120, 151, 2), (3, 2, 40, 53, 2), (6, 4, 23, 12, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gates_over_long_rows(n, c, h, w, hidden, dtype):
    check_norm(norm_inputs(n, c, h, w, hidden, dtype, seed=n + h))
