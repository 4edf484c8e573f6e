"""GPU: FusedAdam against the formulas in float64 and against torch.optim.Adam / AdamW.

One step in float32 is a handful of rounded operations on each value: g' = c g + wd p, m, v, root, quotient, difference.
Each is off by a half-step (2^-24) of its result, and the chain from g to the new weight is 8 long, so the moments are
within 8 * 2^-24 of their terms' magnitudes and a weight within 2^-24 |p| + 16 * 2^-24 |update|, plus what the factor c
brings in (2^-24)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def tensors(shapes, seed=0, scale=1e-3):
    g = torch.Generator("cuda").manual_seed(seed)
    params = [(torch.randn(s, device="cuda", generator=g) * 0.05).requires_grad_(True) for s in shapes]
    for i, p in enumerate(params):
        p.grad = torch.randn(p.shape, device="cuda", generator=g) * scale * 10.0 ** -(i % 3)
    return params


SHAPES = [(3,), (1,), (256,), (255, 3), (4097,), (4096,), (64, 64, 3, 3), (2, 128), ()]


def reference_step(p, g, m, v, t, lr, wd, decoupled, c=1.0, b1=0.9, b2=0.999, eps=1e-8):
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = c * g
    if not decoupled:
        g = g + wd * p
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    update = lr / (1 - b1 ** t) * m / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps)
    return p * (1 - lr * wd if decoupled else 1) - update, m, v, update


@pytest.mark.parametrize("decoupled", [False, True])
@pytest.mark.parametrize("max_norm", [None, 1e-2, 1e3])
def test_one_step_in_32_bits(decoupled, max_norm):
    from alphazero_amd.optim import FusedAdam
    params = tensors(SHAPES)
    opt = FusedAdam(params, lr=3e-3, weight_decay=0.1, decoupled=decoupled)
    gen = torch.Generator("cuda").manual_seed(5)
    for st in opt.state.values():
        st["exp_avg"].copy_(torch.randn(st["exp_avg"].shape, device="cuda", generator=gen) * 1e-3)
        st["exp_avg_sq"].copy_(torch.rand(st["exp_avg_sq"].shape, device="cuda", generator=gen) * 1e-6)
        st["step"].fill_(9)
    before = [(p.detach().clone(), p.grad.clone(), opt.state[p]["exp_avg"].clone(), opt.state[p]["exp_avg_sq"].clone()) for p in params]
    opt.step(max_norm=max_norm)
    norm = math.sqrt(sum(float(g.double().square().sum()) for _, g, _, _ in before))
    c = min(1.0, max_norm / (norm + 1e-6)) if max_norm else 1.0
    if max_norm:
        assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
    for p, (p0, g0, m0, v0) in zip(params, before):
        want, m, v, update = reference_step(p0, g0, m0, v0, 10, 3e-3, 0.1, decoupled, c)
        st = opt.state[p]
        g_mag = c * g0.double().abs() + (0 if decoupled else 0.1 * p0.double().abs())
        assert bool(((st["exp_avg"].double() - m).abs() <= 8 * U * (m0.double().abs() + g_mag)).all())
        assert bool(((st["exp_avg_sq"].double() - v).abs() <= 8 * U * (v0.double() + g_mag ** 2)).all())
        # a quotient of moments whose terms cancel is off by their magnitudes over it
        loose = update.abs() * ((m0.double().abs() + g_mag) / m.abs().clamp(min=1e-30) + g_mag ** 2 / v)
        assert bool(((p.detach().double() - want).abs() <= 2 * U * p0.double().abs() + 16 * U * (update.abs() + loose)).all())
        assert float(st["step"]) == 10.0 and torch.equal(p.grad, g0)


@pytest.mark.parametrize("decoupled", [False, True])
def test_many_steps_beside_torch(decoupled):
    """30 steps with fresh gradients beside torch.optim.Adam / AdamW in float32, clipping included.  Both round every step by
    at most a few half-steps of the update (lr = 1e-3) and of the weight: 30 * (2^-24 * 0.3 + 32 * 2^-24 * 1e-3), times 4 for
    the moments' own drift; 1e-6 covers it, except where the terms of g' = c g + wd p cancel.  There g', and with it m and
    sqrt(v), is known to d = 8 * 2^-24 * M only, M the largest |c g| + wd |p| so far, and the update lr m / (sqrt(v) + eps)
    (v without its bias) moves by up to lr (d + |m| / sqrt(v) d) / (sqrt(v) + eps), where |m| / sqrt(v) is at most
    (1 - b1) / sqrt(1 - b2) / sqrt(1 - b1^2 / b2) < 8: each step allows lr * 9 d / (sqrt(v) + eps) for that.  (With weight
    decay in the gradient one weight of the 40,000 starts at |g'| = 2e-8, of the size of eps, and is off by 3e-6.)"""
    from alphazero_amd.optim import FusedAdam
    ours, theirs = tensors(SHAPES, 3), tensors(SHAPES, 3)
    kind = torch.optim.AdamW if decoupled else torch.optim.Adam
    a, b = FusedAdam(ours, lr=1e-3, weight_decay=1e-2, decoupled=decoupled), kind(theirs, lr=1e-3, weight_decay=1e-2)
    sched = [torch.optim.lr_scheduler.CosineAnnealingLR(o, T_max=40, eta_min=1e-5) for o in (a, b)]
    gen = torch.Generator("cuda").manual_seed(1)
    allowed, largest = [torch.full_like(p, 1e-6) for p in ours], [torch.zeros_like(p) for p in ours]
    for t in range(1, 31):
        for p, q in zip(ours, theirs):
            q.grad.copy_(torch.randn(q.shape, device="cuda", generator=gen) * 1e-3)
            p.grad.copy_(q.grad)
        torch.nn.utils.clip_grad_norm_(theirs, 0.1)
        for p, q, most in zip(ours, theirs, largest):
            most.copy_(torch.maximum(most, q.grad.abs() + (0 if decoupled else 1e-2) * q.detach().abs()))
        lr = b.param_groups[0]["lr"]
        a.step(max_norm=0.1)
        b.step()
        for q, bound, most in zip(theirs, allowed, largest):
            bound += lr * 9 * 8 * U * most / ((b.state[q]["exp_avg_sq"] / (1 - 0.999 ** t)).sqrt() + 1e-8)
        for s in sched:
            s.step()
    for p, q, bound in zip(ours, theirs, allowed):
        assert bool(((p.detach() - q.detach()).abs() <= bound).all())


def codes_reference(x, chance, positive):
    """e4m3 code values and powers of two by distances to the neighbouring codes, in float64."""
    codes = torch.arange(127, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    block = x.double().reshape(-1, 256)
    top = block.abs().amax(1)
    # (2.0 ** k and ldexp as float64 operations are off by a last place on the GPU: the bits are put together instead)
    scale = ((torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** -108))).long() + 1023) << 52).view(torch.float64)
    y = (block / scale[:, None]).reshape(-1)
    low = torch.searchsorted(codes, y.abs(), right=True) - 1
    high = (low + 1).clamp(max=126)
    part = torch.where(high > low, (y.abs() - codes[low]) / (codes[high] - codes[low]).clamp(min=1e-9), torch.zeros_like(y))
    up = part + chance >= 1
    if positive:
        up |= (low == 0) & (y != 0)
    return torch.where(up, codes[high], codes[low]) * torch.sign(y), scale, (part + chance - 1).abs()


def chances(opt, t):
    z = torch.arange(opt.flat_state()["exp_avg"].numel(), device="cuda") + opt.seed * 0x9E3779B9 + t * 0x85EBCA6B
    for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B), (16, 1)):
        z = z & 0xFFFFFFFF
        z = (z ^ (z >> shift)) * factor
    return (z & 0xFFFF).double() / 65536, (z >> 16 & 0xFFFF).double() / 65536


def test_steps_in_8_bits():
    """Five steps: each from the moments that the codes stand for.  The new moments are known to a few half-steps of float32,
    so a code has to be the reference's unless the way between its neighbours lies within that of the border (2^-24 times
    16 steps a binade times the 8 roundings: 1e-5)."""
    from alphazero_amd.optim import FusedAdam, _decode
    params = tensors(SHAPES)
    opt = FusedAdam(params, lr=1e-3, weight_decay=1e-2, decoupled=True, state_bits=8, seed=77)
    held = opt.flat_state()
    assert held["exp_avg"].dtype == torch.float8_e4m3fn and held["exp_avg"].numel() % 256 == 0
    gen = torch.Generator("cuda").manual_seed(2)
    for t in range(1, 6):
        for p in params:
            p.grad.copy_(torch.randn(p.shape, device="cuda", generator=gen) * 1e-3)
        flat_p, flat_g = torch.zeros(held["exp_avg"].numel(), device="cuda"), torch.zeros(held["exp_avg"].numel(), device="cuda")
        for i, p in enumerate(params):
            opt._view(flat_p, i).copy_(p.detach())
            opt._view(flat_g, i).copy_(p.grad)
        m0, r0 = _decode(held["exp_avg"], held["exp_avg_scale"]), _decode(held["exp_rms"], held["exp_rms_scale"])
        want, m, v, update = reference_step(flat_p, flat_g, m0, r0.double() ** 2, t, 1e-3, 1e-2, True)
        opt.step()
        for i, p in enumerate(params):
            d = (p.detach().double() - opt._view(want, i)).abs()
            assert bool((d <= 2 * U * 0.5 + 64 * U * (1e-3 + opt._view(update, i).abs())).all())
        for name, x, chance in zip(("exp_avg", "exp_rms"), (m, v.sqrt()), chances(opt, t)):
            code, scale, border = codes_reference(x, chance, name == "exp_rms")
            assert torch.equal(held[name + "_scale"].double(), scale)
            sure = border > 1e-5
            assert float(sure.double().mean()) > 0.99
            assert torch.equal(held[name].double()[sure], code[sure])
        assert float(held["step"].min()) == t


def test_rounding_in_8_bits_is_right_on_average():
    """A constant gradient: m tends to g and sqrt(v) to |g|.  Rounded to nearest both would stop at a code; rounded at random,
    the mean over 65536 values follows.  A code's step is at most 1/8 of the value; the averages of k independent
    values with spread s are off by s / sqrt(k): s <= 1/4, 5 sigma = 5e-3."""
    from alphazero_amd.optim import FusedAdam, _decode
    p = torch.zeros(65536, device="cuda", requires_grad=True)
    p.grad = torch.full_like(p, 0.013)
    p.grad[::256] = 0.02                                   # so that 0.013 lies inside its block's codes
    opt = FusedAdam([p], lr=0.0, betas=(0.9, 0.99), state_bits=8)
    held = opt.flat_state()
    for t in range(1, 301):
        opt.step()
    m, r = _decode(held["exp_avg"], held["exp_avg_scale"]), _decode(held["exp_rms"], held["exp_rms_scale"])
    rest = torch.ones(65536, dtype=torch.bool, device="cuda")
    rest[::256] = False
    assert abs(float(m[rest].mean()) / 0.013 - 1) < 5e-3
    # v's mean is known to 0.99^300 = 5 % below its limit; the root's rounding adds its variance to v (under 4 %)
    assert abs(float(r[rest].square().mean()) / 0.013 ** 2 - (1 - 0.99 ** 300)) < 0.04
    assert torch.equal(p.detach(), torch.zeros_like(p))


def test_what_is_not_finite_in_8_bits():
    """An infinite or NaN gradient spoils its own element and no other of its block."""
    from alphazero_amd.optim import FusedAdam, _decode
    p = torch.ones(512, device="cuda", requires_grad=True)
    p.grad = torch.full_like(p, 1e-3)
    p.grad[5], p.grad[300] = math.inf, math.nan
    opt = FusedAdam([p], state_bits=8)
    for _ in range(2):
        opt.step()
    held = opt.flat_state()
    bad = ~torch.isfinite(p.detach())
    assert bad.nonzero().flatten().tolist() == [5, 300]
    m = _decode(held["exp_avg"], held["exp_avg_scale"])
    assert (~torch.isfinite(m)).nonzero().flatten().tolist() == [5, 300]


def test_norm_that_is_not_finite():
    """torch's clipping: an infinite norm scales by zero (inf * 0 is NaN for the infinite ones), a NaN norm spoils all."""
    from alphazero_amd.optim import FusedAdam
    p = torch.ones(300, device="cuda", requires_grad=True)
    p.grad = torch.full_like(p, 1e-3)
    p.grad[7] = math.inf
    opt = FusedAdam([p])
    opt.step(max_norm=1.0)
    assert float(opt.grad_norm) == math.inf and (~torch.isfinite(p.detach())).nonzero().flatten().tolist() == [7]
    assert bool((p.detach()[:7] == 1).all())
    p.grad[7] = math.nan
    opt.step(max_norm=1.0)
    assert math.isnan(float(opt.grad_norm)) and not bool(torch.isfinite(p.detach()).any())


def test_norm_of_gradients_decades_apart():
    """Sums of squares from 1e-30 to 1e8 and many small ones beside a large one: exact to the float32 it is returned in."""
    from alphazero_amd.optim import FusedAdam
    params = [torch.zeros(k, device="cuda", requires_grad=True) for k in (1, 70000, 5000)]
    params[0].grad = torch.full((1,), 1e4, device="cuda")
    params[1].grad = torch.full((70000,), 1e-1, device="cuda")
    params[2].grad = torch.full((5000,), 1e-15, device="cuda")
    opt = FusedAdam(params, lr=0.0)
    opt.step(max_norm=1.0)
    want = math.sqrt(sum(float(p.grad.double().square().sum()) for p in params))
    assert abs(float(opt.grad_norm) - want) <= U * want


def test_parameters_without_gradient_groups_and_empty_ones():
    from alphazero_amd.optim import FusedAdam
    params = tensors([(10,), (300,), (0,), (7, 7)])
    params[1].grad = None
    params[2].grad = torch.zeros(0, device="cuda")
    opt = FusedAdam([{"params": params[:2], "lr": 1e-2}, {"params": params[2:], "lr": 1e-3, "weight_decay": 0.5, "decoupled_weight_decay": True}])
    kept = params[1].detach().clone()
    start = [p.detach().clone() for p in params]
    opt.step(max_norm=1.0)
    assert torch.equal(params[1].detach(), kept) and opt.flat_state()["step"].tolist() == [1.0, 0.0, 0.0, 1.0]
    # first step: m / (1 - b1) = g, sqrt(v / (1 - b2)) = |g|: the update is lr sign(g)
    assert float((params[0].detach() - start[0] + 1e-2 * params[0].grad.sign()).abs().max()) < 1e-4
    assert float((params[3].detach() - start[3] * (1 - 5e-4) + 1e-3 * params[3].grad.sign()).abs().max()) < 1e-5
    params[1].grad = torch.ones_like(params[1])
    opt.step()
    assert opt.flat_state()["step"].tolist() == [2.0, 1.0, 0.0, 2.0]
    opt.zero_grad()
    opt.step(max_norm=1.0)                                           # nothing to do
    assert opt.flat_state()["step"].tolist() == [2.0, 1.0, 0.0, 2.0]


def test_more_tensors_than_a_table_holds():
    """300 tensors of odd sizes and two large ones: several launches, every tensor as if it were alone."""
    from alphazero_amd.optim import FusedAdam
    shapes = [(1 + 37 * i % 500,) for i in range(300)] + [(9001,), (123, 77)]
    many, single = tensors(shapes, 4), tensors(shapes, 4)
    a = FusedAdam(many)
    others = [FusedAdam([p]) for p in single]
    for _ in range(2):
        a.step()
        for o in others:
            o.step()
    assert all(torch.equal(p.detach(), q.detach()) for p, q in zip(many, single))


def test_strides_and_unaligned_tensors():
    """Channels-last weights with gradients in either order, tensors that start in the middle of a buffer."""
    from alphazero_amd.optim import FusedAdam
    base = tensors([(16, 12, 3, 3), (1000,)], 6)
    want = [p.detach().clone().requires_grad_(True) for p in base]
    for w, p in zip(want, base):
        w.grad = p.grad.clone()
    FusedAdam(want).step(max_norm=0.01)
    for order in (torch.contiguous_format, torch.channels_last):
        p = base[0].detach().clone().to(memory_format=torch.channels_last).requires_grad_(True)
        p.grad = base[0].grad.clone().contiguous(memory_format=order)
        flat = torch.zeros(2010, device="cuda")
        q = flat[3:1003].copy_(base[1].detach()).requires_grad_(True)
        gq = torch.zeros(1005, device="cuda")
        q.grad = gq[1:1001].copy_(base[1].grad)
        opt = FusedAdam([p, q])
        opt.step(max_norm=0.01)
        assert torch.equal(p.detach(), want[0].detach()) and torch.equal(q.detach(), want[1].detach())
        assert float(flat[:3].abs().max()) == 0 and float(flat[1003:].abs().max()) == 0     # neighbours untouched
        assert opt.state[p]["exp_avg"].stride() == p.stride()


@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoints_go_both_ways(bits):
    """state_dict -> torch.optim.Adam -> state_dict -> FusedAdam: the same next step (8 bits: the same codes' values)."""
    import copy
    from alphazero_amd.optim import FusedAdam
    params = tensors(SHAPES, 8)
    opt = FusedAdam(params, lr=2e-3, weight_decay=1e-2, state_bits=bits)
    for _ in range(3):
        opt.step()
    sd = copy.deepcopy(opt.state_dict())
    for st in sd["state"].values():
        assert set(st) == {"step", "exp_avg", "exp_avg_sq"} and st["exp_avg"].dtype == torch.float32
    twins = [p.detach().clone().requires_grad_(True) for p in params]
    torch_opt = torch.optim.Adam(twins, lr=1.0)
    torch_opt.load_state_dict(sd)
    assert torch_opt.param_groups[0]["lr"] == 2e-3
    again = [p.detach().clone().requires_grad_(True) for p in params]
    back = FusedAdam(again, state_bits=bits)
    back.load_state_dict(copy.deepcopy(torch_opt.state_dict()))
    for name, a in opt.flat_state().items():
        b = back.flat_state()[name]
        if "scale" not in name and a.dtype == torch.float32:
            assert torch.equal(a, b), name
    sd2 = back.state_dict()
    for i, st in sd["state"].items():
        assert all(torch.equal(st[k], sd2["state"][i][k]) for k in st)
    for p, q, r in zip(params, again, twins):
        q.grad, r.grad = p.grad.clone(), p.grad.clone()
    opt.step()
    back.step()
    torch_opt.step()
    for p, q, r in zip(params, again, twins):
        assert torch.equal(p.detach(), q.detach())
        assert float((p.detach() - r.detach()).abs().max()) < 1e-6
    fresh = FusedAdam(again)
    fresh.load_state_dict(torch.optim.Adam(twins).state_dict())       # torch's has no state before its first step
    assert float(fresh.flat_state()["step"].max()) == 0


def test_step_moves_version_counters_and_follows_moved_tensors():
    from alphazero_amd.optim import FusedAdam
    params = tensors([(50,), (60,)])
    opt = FusedAdam(params)
    versions = [p._version for p in params]
    opt.step()
    assert all(p._version > v for p, v in zip(params, versions))
    params[0].data = params[0].data.clone()                           # another place, the same strides
    params[0].grad = params[0].grad.clone()
    old = params[0].detach().clone()
    opt.step()
    assert not torch.equal(params[0].detach(), old)


def test_optimiser_refusals():
    import copy
    from alphazero_amd.optim import FusedAdam
    params = tensors([(8, 4, 3, 3)])
    with pytest.raises(TypeError, match="float32 parameters"):
        FusedAdam([torch.zeros(3, dtype=torch.bfloat16, device="cuda", requires_grad=True)])
    with pytest.raises(ValueError, match="fill its memory"):
        FusedAdam([torch.zeros(4, 6, device="cuda")[:, :3].requires_grad_(True)])
    opt = FusedAdam(params)
    with pytest.raises(RuntimeError, match="at construction"):
        opt.add_param_group({"params": [torch.zeros(3, device="cuda", requires_grad=True)]})
    with pytest.raises(ValueError, match="max_norm"):
        opt.step(max_norm=0.0)
    with pytest.raises(TypeError, match="state_dict"):
        copy.deepcopy(opt)
    sd = opt.state_dict()
    sd["param_groups"][0]["amsgrad"] = True
    with pytest.raises(ValueError, match="amsgrad"):
        opt.load_state_dict(sd)
    kept = params[0].grad
    params[0].grad = torch.sparse_coo_tensor(torch.zeros(4, 1, dtype=torch.int64), torch.ones(1), (8, 4, 3, 3), device="cuda")
    with pytest.raises(ValueError, match="dense gradients"):
        opt.step()
    params[0].grad = kept
    params[0].data = params[0].data.contiguous(memory_format=torch.channels_last)
    with pytest.raises(ValueError, match="strides changed"):
        opt.step()


def test_captured_steps_equal_eager_ones():
    """Replays advance the step counters and follow the gradients; eager work and synchronisation between them."""
    from alphazero_amd.optim import FusedAdam
    for bits in (32, 8):
        a, b = tensors(SHAPES, 11), tensors(SHAPES, 11)
        eager, graphed = FusedAdam(a, state_bits=bits, seed=3), FusedAdam(b, state_bits=bits, seed=3)
        gen = torch.Generator("cuda").manual_seed(4)

        def new_grads():
            for p, q in zip(a, b):
                p.grad.copy_(torch.randn(p.shape, device="cuda", generator=gen) * 1e-2)
                q.grad.copy_(p.grad)
        graph = torch.cuda.CUDAGraph()
        new_grads()
        with torch.cuda.graph(graph):
            graphed.step(max_norm=0.5)
        for _ in range(4):
            new_grads()
            eager.step(max_norm=0.5)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p.detach(), q.detach()) for p, q in zip(a, b))
            assert torch.equal(eager.grad_norm, graphed.grad_norm)
            for name, x in eager.flat_state().items():
                assert torch.equal(x.view(torch.uint8), graphed.flat_state()[name].view(torch.uint8)), name


def test_a_parameter_that_changed_its_shape_in_place_is_refused():
    """The same address with fewer elements or another order: the moments no longer fit, and nothing is read or written."""
    from alphazero_amd.optim import FusedAdam
    for change in (lambda t: t[:5], lambda t: t.t()):
        p = torch.ones(8, 8, device="cuda", requires_grad=True)
        p.grad = torch.ones(8, 8, device="cuda")
        opt = FusedAdam([p])
        opt.step()
        p.grad = None
        p.data = change(p.data)
        p.grad = torch.ones_like(p)
        held = p.detach().clone()
        with pytest.raises(ValueError, match="after FusedAdam was built"):
            opt.step()
        assert torch.equal(p.detach(), held)


def test_a_checkpoint_of_another_shape_is_refused_whole():
    from alphazero_amd.optim import FusedAdam
    a, b = tensors([(4, 6), (5,)]), tensors([(4, 6), (7,)])
    one, two = FusedAdam(a), FusedAdam(b)
    one.step(), two.step()
    kept = {k: v.clone() for k, v in one.flat_state().items()}
    with pytest.raises(ValueError, match="has shape"):
        one.load_state_dict(two.state_dict())
    with pytest.raises(ValueError):
        one.load_state_dict(FusedAdam(tensors([(4, 6)])).state_dict())
    one.step()
    assert all(float(v.min()) == 2.0 for k, v in one.flat_state().items() if k == "step") and kept["step"].tolist() == [1.0, 1.0]


def test_groups_with_rates_of_their_own_are_one_call():
    """Three groups with other betas, decay and rates, clipped by one norm: each as an optimiser of its own that is given the
    clipped gradients."""
    from alphazero_amd.optim import FusedAdam
    shapes = [(300,), (40, 7), (9000,), (3,)]
    params, alone = tensors(shapes, 12), tensors(shapes, 12)
    opts = [dict(lr=1e-2, betas=(0.8, 0.9)), dict(lr=1e-3, weight_decay=0.1), dict(lr=3e-4, weight_decay=0.2, decoupled=True, eps=1e-4)]
    split = [params[:1], params[1:3], params[3:]]
    together = FusedAdam([{"params": p, **{"decoupled_weight_decay" if k == "decoupled" else k: v for k, v in o.items()}} for p, o in zip(split, opts)])
    together.step(max_norm=1e-2)
    norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in alone))
    assert abs(float(together.grad_norm) - norm) <= 2 * U * norm
    c = torch.tensor(1e-2 / (norm + 1e-6), dtype=torch.float32, device="cuda")
    for p in alone:
        p.grad *= c
    for p, o in zip([alone[:1], alone[1:3], alone[3:]], opts):
        FusedAdam(p, **o).step()
    assert all(torch.equal(p.detach(), q.detach()) for p, q in zip(params, alone))


def test_two_optimisers_and_gradients_that_are_shared():
    """One gradient tensor for two parameters, and two optimisers whose steps follow one another on two streams."""
    from alphazero_amd.optim import FusedAdam
    p, q = tensors([(500,), (500,)], 13)
    q.grad = p.grad
    want = [t.detach().clone().requires_grad_(True) for t in (p, q)]
    for t in want:
        t.grad = p.grad.clone()
    a, b = FusedAdam([p], seed=1), FusedAdam([q], seed=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a.step(max_norm=1.0)
    with torch.cuda.stream(side):
        b.step(max_norm=1.0)
    torch.cuda.current_stream().wait_stream(side)
    for t, o in zip(want, (FusedAdam(want[:1]), FusedAdam(want[1:]))):
        o.step(max_norm=1.0)
    assert torch.equal(p.detach(), want[0].detach()) and torch.equal(q.detach(), want[1].detach())


def test_closure_scheduler_and_scaler():
    from alphazero_amd.optim import FusedAdam
    p = torch.ones(100, device="cuda", requires_grad=True)
    opt = FusedAdam([p], lr=0.1)

    def closure():
        opt.zero_grad()
        loss = (p * p).sum()
        loss.backward()
        return loss
    assert float(opt.step(closure)) == 100.0 and abs(float(p.detach()[0]) - 0.9) < 1e-6
    scaler = torch.amp.GradScaler("cuda", init_scale=1024.0)
    opt.zero_grad()
    scaler.scale((p * p).sum()).backward()
    scaler.step(opt)
    scaler.update()
    before = p.detach().clone()
    opt.zero_grad()
    scaler.scale((p * p).sum() * math.inf).backward()
    scaler.step(opt)                                                   # infinite gradients: the step is left out
    assert torch.equal(p.detach(), before) and float(opt.flat_state()["step"]) == 2.0


def test_parameters_that_share_memory_are_refused():
    from alphazero_amd.optim import FusedAdam
    flat = torch.zeros(100, device="cuda")
    apart = [flat[:50].requires_grad_(True), flat[50:].requires_grad_(True)]
    FusedAdam(apart)
    with pytest.raises(ValueError, match="share memory"):
        FusedAdam([flat[40:60].detach().requires_grad_(True)] + apart)
