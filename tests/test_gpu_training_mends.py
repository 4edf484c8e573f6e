"""GPU: the training operators where they were wrong once.  Tolerances as in test_gpu_training_ops: k half-steps of float32
of the magnitudes plus one rounding to the output's type."""
import ctypes as C
import math

import pytest
import torch

from test_gpu_training_ops import DTYPES, check_norm, close, loss_inputs, loss_reference, norm_inputs, norm_reference, run_norm

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ the loss
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, actions", [(64, 192), (33, 4001), (9, 9000), (4, 5)])
@pytest.mark.parametrize("up", [1 / 3, 0.7, -3.0])
def test_loss_gradients_are_rounded_once_whatever_the_upstream(dtype, n, actions, up):
    """One rounding to the logits' type, as with an upstream of 1 (whose gradient is there already)."""
    from alphazero_amd import ops
    z, wl, t, tw, mask = loss_inputs(n, actions, dtype, True, seed=actions)
    z.requires_grad_(True), wl.requires_grad_(True)
    loss = ops.policy_value_loss(z, wl, t, tw, mask)[0]
    got = torch.autograd.grad(loss, (z, wl), torch.full_like(loss, up))
    _, _, grads, mags = loss_reference(z.detach(), wl.detach(), t, tw, mask, (float(torch.tensor(up)), 0.0, 0.0))
    for a, b, m in zip(got, grads, mags):
        close(a, b, m, 64 + -(-actions // 64) + 8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, actions", [(70, 192), (10000, 600)])
def test_backward_call_made_again_without_its_forward_call(dtype, n, actions):
    """As a captured backward pass is replayed: each call gives the gradient of its own upstream, whatever the one before it
    left, and both heads for themselves."""
    from alphazero_amd import _lib
    L = _lib.lib()
    z, wl, t, tw, _ = loss_inputs(n, actions, dtype, False)
    losses, stats = torch.zeros(3, device="cuda"), torch.zeros(8 * n, device="cuda")
    dz, dwl = torch.zeros_like(z), torch.zeros_like(wl)
    ups = [torch.zeros((), device="cuda") for _ in range(3)]
    a = _lib.LossArgs(n, actions, 2, {torch.float32: 0, torch.bfloat16: 1}[dtype], z.data_ptr(), wl.data_ptr(), t.data_ptr(), tw.data_ptr(), None,
                      losses.data_ptr(), stats.data_ptr(), *(u.data_ptr() for u in ups), dz.data_ptr(), dwl.data_ptr())
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert L.az_policy_value_loss_ready(C.byref(a)) == 1
    for forward in range(2):
        _lib.check(L.az_policy_value_loss_forward(C.byref(a), stream))
        for up in ((1.0, 0.0, 0.0), (3.0, 0.0, 0.0), (3.0, 0.0, 0.0), (1.0, 0.0, 0.0), (0.0, 0.5, 1.0), (0.0, 1.0, 0.25), (1.0, 0.0, 0.0)):
            for u, v in zip(ups, up):
                u.fill_(v)
            a.grads_ready = 1
            _lib.check(L.az_policy_value_loss_backward(C.byref(a), stream))
            got = dz.clone(), dwl.clone()
            fresh = torch.zeros_like(z), torch.zeros_like(wl)
            a.grads_ready, a.dpolicy, a.dwl = 0, fresh[0].data_ptr(), fresh[1].data_ptr()
            _lib.check(L.az_policy_value_loss_backward(C.byref(a), stream))
            a.dpolicy, a.dwl = dz.data_ptr(), dwl.data_ptr()
            assert torch.equal(got[0], fresh[0]) and torch.equal(got[1], fresh[1]), (forward, up)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("actions", [3, 192, 1500, 9000])
@pytest.mark.parametrize("masked", [False, True])
def test_loss_rows_of_minus_infinity_without_targets(dtype, actions, masked):
    """A row whose kept logits are all minus infinity and whose targets are zero adds nothing, and its gradient is zero: a row
    without a legal move whose program marks them so.  The other rows are as if it were a row without targets."""
    from alphazero_amd import ops
    z, wl, t, tw, mask = loss_inputs(9, actions, dtype, masked, seed=actions)
    for row in (4, 7):
        t[row] = 0
        z[row] = torch.where(mask[row], torch.full_like(z[row], -math.inf), z[row]) if masked else -math.inf
    wl[5], tw[5] = -math.inf, 0
    z.requires_grad_(True), wl.requires_grad_(True)
    for up in (1.0, 0.5):
        losses = ops.policy_value_loss(z, wl, t, tw, mask)
        got = torch.autograd.grad(losses[0], (z, wl), torch.full_like(losses[0], up))
        want, mags, grads, grad_mags = loss_reference(z.detach(), wl.detach(), t, tw, mask, (up, 0.0, 0.0))
        for a, b, m in zip(losses, want, mags):
            close(a, b, m, 72 + -(-actions // 64))
        for a, b, m in zip(got, grads, grad_mags):
            close(a, torch.nan_to_num(b, nan=0.0), torch.nan_to_num(m, nan=0.0), 72 + -(-actions // 64))
        assert bool((got[0][[4, 7]] == 0).all()) and bool((got[1][5] == 0).all())


@pytest.mark.parametrize("actions", [192, 4001, 9000])
def test_probabilities_of_far_logits(actions):
    """Logits down to 76 below the largest, without targets of their own: their gradient is exp(z - m) / S * T * (upstream / n),
    where z - m is exact (a multiple of 2^-3): 8 half-steps for the operations, and for S one for each of a thread's values (8 in
    a row of up to 512, actions / 256 in longer ones) and 8 for the sum over the threads.  An exponential that multiplies by
    1 / ln 2 and rounds is off by up to 44 of them there."""
    from alphazero_amd import ops
    z = torch.zeros(4, actions, device="cuda")
    z[:, 1:] = -(torch.arange(1, actions, device="cuda").float() / 8) % 76 - 76
    t = torch.zeros(4, actions, device="cuda")
    t[:, 0] = 1
    z.requires_grad_(True)
    wl = torch.zeros(4, 2, device="cuda")
    for up in (1.0, 0.25):
        loss = ops.policy_value_loss(z, wl, t, torch.full((4, 2), 0.5, device="cuda"))[0]
        got, = torch.autograd.grad(loss, z, torch.full_like(loss, up))
        # (on the host: the GPU's own float64 softmax of rows over 1024 is off by 60 of these steps)
        want = torch.softmax(z.detach().cpu().double(), 1)[:, 1:].cuda() / 4 * up
        assert float(((got[:, 1:].double() - want).abs() / want).max()) <= (24 + actions // 256) * 2.0 ** -24


# ----------------------------------------------------------------------------------------------- the norms
LAYOUTS = pytest.mark.parametrize("layout", [torch.contiguous_format, torch.channels_last], ids=["nchw", "nhwc"])
# one for each way that a row is read: a channel in a workgroup's registers, whole and moved pieces, rounds, less than a piece
ROWS = [(6, 5, 8, 8), (2100, 3, 8, 8), (1200, 7, 9, 9), (3, 3, 120, 151), (1200, 6, 1, 3), (60, 24, 19, 19)]


@pytest.mark.parametrize("n, c, h, w", ROWS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@LAYOUTS
def test_norms_pass_the_gradient_where_the_output_is_nan(n, c, h, w, dtype, layout):
    """As torch's ReLU does.  What makes the output NaN without being in a sum is the residual, or a plain norm's bias: every
    gradient is the one of an output that is far above zero there, bit for bit."""
    for hidden in (0, 3):
        t = norm_inputs(n, c, h, w, hidden, dtype, layout, seed=n)
        runs = []
        if hidden:
            t["grad"] = t["grad"].clone(memory_format=torch.preserve_format)
            t["grad"][:, 1, 0] = 0.01
        for value in (math.nan, 1e4):
            u = dict(t)
            if hidden:
                u["residual"] = t["residual"].clone(memory_format=torch.preserve_format)
                u["residual"][:, 1, 0] = value
            else:
                u["bias"] = t["bias"].clone()
                u["bias"][1] = value
            runs.append(run_norm(u))
        assert bool(torch.isnan(runs[0]["out"][:, 1, 0]).all())
        for name in set(runs[0]) - {"out"}:
            assert torch.equal(runs[0][name], runs[1][name]), (hidden, name)
        assert not hidden or torch.equal(runs[0]["residual"][:, 1, 0], t["grad"][:, 1, 0])


@pytest.mark.parametrize("n, c, h, w", ROWS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@LAYOUTS
def test_norms_with_running_statistics_and_an_infinite_value(n, c, h, w, dtype, layout):
    """Every value stands for itself there: a gradient of x is weight / s times the one that arrives, infinite or NaN x or not, bit
    for bit that of a large one, and so are all gradients of the other channels."""
    t = norm_inputs(n, c, h, w, 0, dtype, layout, seed=n + 1, training=False)
    t["weight"] = t["weight"].abs() + 0.1
    t["grad"] = t["grad"].clone(memory_format=torch.preserve_format)
    t["grad"][:, 1, 0] = 0.01
    runs = []
    for value in (1e4, math.inf, math.nan):
        x = t["x"].clone(memory_format=torch.preserve_format)
        x[:, 1, 0] = value
        runs.append(run_norm({**t, "x": x}, training=False))
    others = [i for i in range(c) if i != 1]
    for got in runs[1:]:
        assert not bool(torch.isfinite(got["out"][:, 1, 0]).any())
        assert torch.equal(got["x"], runs[0]["x"]) and torch.equal(got["bias"], runs[0]["bias"])
        assert torch.equal(got["weight"][others], runs[0]["weight"][others]) and not bool(torch.isfinite(got["weight"][1]))


@pytest.mark.parametrize("n, c, h, w", [(33, 12, 19, 19), (3, 9, 64, 64), (2, 3, 256, 256), (300, 5, 1, 3), (9, 300, 7, 9), (2100, 3, 8, 8), (20, 6, 8, 8)])
@pytest.mark.parametrize("off", [100.0, 1000.0])
@LAYOUTS
def test_norm_statistics_beside_an_outlier_at_the_first_place(n, c, h, w, off, layout):
    """Each board's first place lies far from the rest.  Centred sums add squares only, so the variance is off by one half-step
    for each value that a thread adds (a quarter of the places at most) and 64 for the joins: not by the squares of the distances
    to that place, which are hw times as large together."""
    for hidden in (0, 2):
        t = norm_inputs(n, c, h, w, hidden, torch.float32, layout, seed=n)
        t["x"][:, :, 0, 0] += off
        # (gradients are compared where the ReLU's border is not near, as in norm_inputs)
        _, pre, hid = norm_reference(t, True)
        t["grad"] = (t["grad"] * (pre.abs() > 1e-3 * off)).contiguous(memory_format=layout)
        if hidden:
            t["grad"] = (t["grad"] * (hid.abs() > 1e-3).all(1)[:, None, None, None]).contiguous(memory_format=layout)
        got = check_norm(t)
        ref, _, _ = norm_reference(t, True)
        want = ref["running_var"][0]
        assert float(((got["running_var"] - want).abs() / want).max()) <= (64 + h * w // 4) * 2.0 ** -24, hidden


@pytest.mark.parametrize("n, c, h, w", ROWS + [(33, 40, 64, 64)])
@LAYOUTS
def test_norms_far_from_zero(n, c, h, w, layout):
    """Values 900 standard deviations from zero.  The mean is held in float32, off by half a step, 2^-15; that times weight / s is
    what the output may be off by, beside 8 half-steps of what is added up: x - mean is exact.  Behind it stand the means of the
    n boards, in float32 too: one that is a value of the board plus a small rest is off by up to half a step more, all of them
    the same way at worst; one that is a sum of 64 to 361 values over 900 by some 1.6 half-steps (one standard deviation: the
    last additions 1, 1/2, 1/4.. of a half-step's square, and the division), so that n >= 60 of them have a mean within
    5 * 1.6 / sqrt(n) half-steps, at most 1.  A gate hears of the board's means, which are sums of hw values: 12 steps of 900 each, through the
    absolute values of its weights."""
    for hidden in (0, 3):
        t = norm_inputs(n, c, h, w, hidden, torch.float32, layout, seed=n)
        t["x"] = (900.0 + torch.randn(n, c, h, w, device="cuda", generator=torch.Generator("cuda").manual_seed(n))).contiguous(memory_format=layout)
        ref, pre, hid = norm_reference(t, True)
        keep = pre.abs() > 1e-2
        if hidden:
            keep &= (hid.abs() > 1e-2).all(1)[:, None, None, None]
        t["grad"] = (t["grad"] * keep).contiguous(memory_format=layout)
        got = check_norm(t)
        ref, pre, _ = norm_reference(t, True)
        var = ref["running_var"][0]
        assert float(((got["running_var"] - var).abs() / var).max()) <= (64 + h * w // 4) * 2.0 ** -24, hidden
        scale = (t["weight"].double() / (t["x"].double().var((0, 2, 3), correction=0) + 1e-5).sqrt()).abs()
        bound = (1 + min(1.0, 8 / math.sqrt(n))) * 2.0 ** -15 * scale[:, None, None] + 8 * 2.0 ** -24 * (5 * scale[:, None, None] + t["bias"].double().abs()[:, None, None] + pre.abs())
        if hidden:
            q = 12 * 2.0 ** -24 * 900 * scale
            inner = t["fc1_weight"].double().abs() @ q
            e = t["fc2_weight"].double().abs() @ inner
            bound = bound + ((5 * scale + t["bias"].double().abs()) * e[:c] / 4 + e[c:])[:, None, None]
        worst = float(((got["out"] - ref["out"][0]).abs() / bound).max())
        assert worst <= 1.0, (hidden, worst)


@pytest.mark.parametrize("var", [2.0 ** -132, 2.0 ** -120, 2.0 ** 126, math.inf, 0.0])
@LAYOUTS
def test_norms_of_variances_at_the_ends_of_the_range(var, layout):
    """eps = 0 is allowed.  With running statistics out = relu(weight x / sqrt(var) + bias) is 8 operations; a variance of zero
    makes x / 0, an infinite one leaves the bias.  With the batch's own, squares below 2^-126 keep 2^-149 of their size."""
    from alphazero_amd import ops
    gen = torch.Generator("cuda").manual_seed(4)
    unit = torch.randn(20, 6, 8, 8, device="cuda", generator=gen)
    w, b = torch.rand(6, device="cuda", generator=gen) + 0.5, torch.randn(6, device="cuda", generator=gen)
    size = math.sqrt(var) if 0 < var < math.inf else 1.0
    x = (unit * size).contiguous(memory_format=layout).requires_grad_(True)
    mean, held = torch.zeros(6, device="cuda"), torch.full((6,), var, device="cuda")
    out = ops.norm_act(x, w, b, mean, held, training=False, eps=0.0)
    ch = lambda v: v.double().view(1, 6, 1, 1)                            # noqa: E731
    y = x.detach().double() / math.sqrt(var) if var else x.detach().double() * math.inf
    want = torch.relu(ch(w) * y + ch(b))
    near = torch.isfinite(want)
    assert torch.equal(torch.isfinite(out), near)
    assert bool(((out - want).abs() <= 8 * 2.0 ** -24 * (ch(w) * y.abs() + ch(b).abs()))[near].all())
    if 0 < var < 1:
        out = ops.norm_act(x, w, b, None, None, training=True, eps=0.0)
        grad, = torch.autograd.grad(out, x, torch.full_like(out, 0.25))
        v, m = torch.var_mean(x.detach().double(), (0, 2, 3), correction=0)
        want = torch.relu(ch(w) * (x.detach().double() - ch(m)) / ch(v).sqrt() + ch(b))
        assert float((out - want).abs().max()) <= (64 + 64) * 2.0 ** -24 * 10 + 2.0 ** -149 / var * 5
        assert bool(torch.isfinite(grad).all())


# ------------------------------------------------------------------------------------------- the optimiser
def test_moments_of_tiny_gradients_are_those_of_elementary_operations():
    """Every operation on the moments is one of torch's, correctly rounded, down to the smallest float32: v between 1e-45 and
    1e-31 and its root, which shows in the codes that the root becomes.  8 bits with a random part of zero round down, so the
    codes of a root that is a last place too small would be others: the held roots are compared with those of the same
    operations on the host, at values whose root is a code."""
    from alphazero_amd.optim import FusedAdam
    # m = 0.1 g; one step from zero with beta2 = 0 and beta1 = 0: v = g * g, root = sqrt(g * g)
    g = torch.cat([torch.logspace(-22.4, -15, 3000, dtype=torch.float64).float(), torch.tensor([2.0 ** -k for k in range(52, 75)])]).cuda()
    p = torch.zeros_like(g).requires_grad_(True)
    p.grad = g.clone()
    opt = FusedAdam([p], lr=1.0, betas=(0.0, 0.0), eps=0.0)
    opt.step()
    v = g.cpu() * g.cpu() * torch.tensor(1.0)
    assert torch.equal(opt.state[p]["exp_avg_sq"].cpu(), v)
    # p = - m / root, the quotient by the hardware's reciprocal: two last places and the product's
    root = v.double().sqrt().float()
    live = root > 0
    want = -(g.cpu().double() / root.double())
    assert bool(((p.detach().cpu().double() - want).abs() <= 4 * 2.0 ** -24 * want.abs())[live].all())


def test_codes_of_tiny_roots():
    """In 8 bits: a root that is exactly a code stays that code whatever the random part; blocks of 2^-40 to 2^-63 times the e4m3
    values 8 to 15 and 128 to 240, whose squares are exact in float32."""
    from alphazero_amd.optim import FusedAdam, _decode
    values = torch.cat([torch.arange(8, 16), torch.arange(8, 16) * 16]).double()
    for k in range(40, 64):
        g = (values * 2.0 ** -k).float().repeat(16).cuda()
        p = torch.zeros_like(g).requires_grad_(True)
        p.grad = g.clone()
        opt = FusedAdam([p], lr=0.0, betas=(0.0, 0.0), state_bits=8)
        opt.step()
        held = opt.flat_state()
        assert torch.equal(_decode(held["exp_rms"], held["exp_rms_scale"])[:256], g), k
        assert torch.equal(_decode(held["exp_avg"], held["exp_avg_scale"])[:256], g), k


def test_update_without_eps_does_not_depend_on_the_scale():
    """m / sqrt(v) of gradients times a power of two: every operation is the same one, bit for bit, as long as v is a normal
    number, 2^-124 to 2^-4 here."""
    from alphazero_amd.optim import FusedAdam
    gen = torch.Generator("cuda").manual_seed(6)
    g = torch.randn(20000, device="cuda", generator=gen).abs().clamp(min=0.01) * 2.0 ** -54
    results = []
    for power in (0, 20, 50):
        p = torch.zeros_like(g).requires_grad_(True)
        opt = FusedAdam([p], lr=1.0, betas=(0.5, 0.25), eps=0.0)
        for factor in (1.0, -0.375, 3.0):
            p.grad = g * (factor * 2.0 ** power)
            opt.step()
        results.append(p.detach())
    assert torch.equal(results[0], results[2]) and torch.equal(results[1], results[2])


@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoint_goes_on_on_the_host(bits):
    """state_dict() into a torch.optim.Adam of parameters on the CPU, which steps, and back; without the trainer's own handling."""
    import io
    from alphazero_amd.optim import FusedAdam
    gen = torch.Generator("cuda").manual_seed(7)
    p = torch.randn(300, device="cuda", generator=gen).requires_grad_(True)
    p.grad = torch.randn(300, device="cuda", generator=gen)
    opt = FusedAdam([p], lr=1e-2, state_bits=bits)
    opt.step()
    file = io.BytesIO()
    torch.save(opt.state_dict(), file)
    file.seek(0)
    q = p.detach().cpu().requires_grad_(True)
    host = torch.optim.Adam([q], lr=1.0)
    host.load_state_dict(torch.load(file, map_location="cpu", weights_only=True))
    q.grad = p.grad.cpu()
    host.step()
    kept = {k: v.clone() for k, v in opt.state_dict()["state"][0].items()}
    opt.step()
    assert float((p.detach().cpu() - q.detach()).abs().max()) < 1e-6
    assert float(host.state[q]["step"]) == 2.0 and float(kept["step"]) == 1.0
    opt.load_state_dict(host.state_dict())
    assert float(opt.flat_state()["step"]) == 2.0 and opt.param_groups[0]["capturable"]
    graph = torch.cuda.CUDAGraph()                                      # still steps from a graph
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    torch.cuda.synchronize()
    assert float(opt.flat_state()["step"]) == 3.0


def test_updates_in_8_bits_follow_those_in_32():
    """Gradients of mean s and spread s, s over five decades in every block of 256, 1500 steps: the way that the weights have gone
    and the v that is held, beside moments in 32 bits that see the same gradients.  What the rounding does to them is known from
    the same recurrence in elementary operations: v is held 3 to 5 % high, the update is 1 % off (there a sixth of a code's step,
    12 % at most, is one standard deviation of a held value: 1 % over 3277 values is 6 of their mean)."""
    from alphazero_amd.optim import FusedAdam
    n = 256 * 64
    decade = torch.arange(n, device="cuda") % 5
    s = 10.0 ** -decade.float()
    p8, p32 = (torch.zeros(n, device="cuda", requires_grad=True) for _ in range(2))
    p8.grad, p32.grad = torch.zeros_like(p8), torch.zeros_like(p32)
    a, b = FusedAdam([p8], lr=1e-3, eps=1e-12, state_bits=8, seed=5), FusedAdam([p32], lr=1e-3, eps=1e-12)
    gen = torch.Generator("cuda").manual_seed(8)
    for _ in range(1500):
        p8.grad.copy_(s * (1 + torch.randn(n, device="cuda", generator=gen)))
        p32.grad.copy_(p8.grad)
        a.step(), b.step()
    held, v = a.state_dict()["state"][0]["exp_avg_sq"], b.state_dict()["state"][0]["exp_avg_sq"]
    for k in range(5):
        at = decade == k
        assert 1.02 <= float(held[at].mean() / v[at].mean()) <= 1.06, k
        assert 0.99 <= float(p8.detach()[at].mean() / p32.detach()[at].mean()) <= 1.03, k


@pytest.mark.parametrize("n, c, h, w, hidden", [(2, 1, 1, 1, 0), (1, 5, 1, 2, 0), (7, 130, 1, 1, 0), (7, 130, 1, 1, 16), (2, 40, 2, 2, 3), (3, 9, 1, 1, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@LAYOUTS
def test_norms_of_a_few_16_bit_values(n, c, h, w, hidden, dtype, layout):
    check_norm(norm_inputs(n, c, h, w, hidden, dtype, layout, seed=n + c))


@pytest.mark.parametrize("n, c, h, w", ROWS)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@LAYOUTS
def test_what_is_not_finite_stays_in_its_channel(n, c, h, w, bad, layout):
    """Every pass: a channel with a NaN or an infinity has NaN statistics, outputs and gradients; the others are what they are
    without it, bit for bit.  Behind a gate every board hears of it."""
    t = norm_inputs(n, c, h, w, 0, torch.float32, layout, seed=n)
    clean = run_norm(t)
    x = t["x"].clone(memory_format=torch.preserve_format)
    x[n // 2, 1, 0, w // 2] = bad
    got = run_norm({**t, "x": x})
    others = [i for i in range(c) if i != 1]
    for name in ("out", "x"):
        assert bool(torch.isnan(got[name][:, 1]).all()) and torch.equal(got[name][:, others], clean[name][:, others]), name
    for name in ("weight", "bias", "running_mean", "running_var"):
        assert torch.equal(got[name][others], clean[name][others]), name
    assert math.isnan(float(got["running_var"][1])) and not math.isfinite(float(got["running_mean"][1]))
    gated = run_norm({**norm_inputs(n, c, h, w, 2, torch.float32, layout, seed=n), "x": x})
    assert bool(torch.isnan(gated["out"]).all()) and bool(torch.isnan(gated["fc1_weight"]).all())
