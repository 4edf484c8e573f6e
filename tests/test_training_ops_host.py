"""CPU: what the training operators refuse before anything reaches a GPU - the Python entry points' checks of
types, shapes and devices, and the C entries' checks of their arguments."""
import ctypes as C

import pytest
import torch

from alphazero_amd import _lib, ops
from alphazero_amd.optim import FusedAdam, _decode, _dense, _encode


def test_structures_match_the_header(tmp_path):
    """The ctypes mirrors have the C structures' sizes (compiled from include/azamd.h)."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "azamd.h"\nint main(void) { printf("%zu %zu %zu %zu %d %d %d", sizeof(az_norm_args), '
                   'sizeof(az_loss_args), sizeof(az_adam_config), sizeof(az_adam_group), AZ_OPTIM_CHUNK, AZ_OPTIM_PAD, AZ_OPTIM_GROUPS); return 0; }\n')
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "sizes")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "sizes")]).split()]
    assert got == [C.sizeof(_lib.NormArgs), C.sizeof(_lib.LossArgs), C.sizeof(_lib.AdamConfig), C.sizeof(_lib.AdamGroup), _lib.OPTIM_CHUNK, _lib.OPTIM_PAD,
                   _lib.OPTIM_GROUPS]


def test_host_tensors_are_refused():
    x, v = torch.zeros(2, 4, 3, 3), torch.zeros(4)
    with pytest.raises(ValueError, match="need a GPU tensor"):
        ops.norm_act(x, v, v, v, v)
    with pytest.raises(ValueError, match="need a GPU tensor"):
        ops.norm_gate_residual(x, x, v, v, v, v, torch.zeros(2, 4), torch.zeros(2), torch.zeros(8, 2), torch.zeros(8))
    with pytest.raises(ValueError, match="needs GPU tensors"):
        ops.policy_value_loss(torch.zeros(2, 5), torch.zeros(2, 2), torch.zeros(2, 5), torch.zeros(2, 2))
    with pytest.raises(ValueError, match="parameters on a GPU"):
        FusedAdam([torch.zeros(3, requires_grad=True)])


@pytest.mark.parametrize("kwargs, match", [({"state_bits": 16}, "state_bits"), ({"betas": (1.0, 0.9)}, "betas"),
                                           ({"lr": -1.0}, "negative"), ({"eps": -1.0}, "negative"), ({"weight_decay": -1.0}, "negative")])
def test_optimiser_refuses_hyper_parameters(kwargs, match):
    with pytest.raises(ValueError, match=match):
        FusedAdam([torch.zeros(3, requires_grad=True)], **kwargs)


def _norm_args(**kw):
    a = _lib.NormArgs(4, 8, 9, 0, 0, 0, 1, 1e-5, 0.1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw, match", [
    ({"n": 0}, "out of range"), ({"c": 0}, "out of range"), ({"hw": 0}, "out of range"), ({"n": 1 << 28, "c": 64}, "out of range"),
    ({"dtype": 3}, "unknown type"), ({"n": 1, "hw": 1}, "two values"), ({"hidden": -1}, "a gate takes"), ({"hidden": 1025}, "a gate takes"),
    ({"hidden": 2, "c": 1025}, "a gate takes"), ({}, "null argument"),
])
def test_c_entries_of_the_norms_check_their_arguments(kw, match):
    L = _lib.lib()
    for entry in (L.az_norm_forward, L.az_norm_backward):
        assert entry(C.byref(_norm_args(**kw)), None) == -1
        assert match.encode() in L.az_last_error()
    assert L.az_norm_forward(None, None) == -1 and L.az_norm_sizes(C.byref(_norm_args()), None) == -1


def test_c_entries_of_the_norms_check_alignment():
    L = _lib.lib()
    full = dict(x=64, weight=64, bias=64, saved=64, workspace=72, out=64)      # addresses are only looked at
    assert L.az_norm_forward(C.byref(_norm_args(**full)), None) == -1 and b"aligned" in L.az_last_error()
    full["workspace"] = 64
    assert L.az_norm_forward(C.byref(_norm_args(training=0, **full)), None) == -1 and b"running" in L.az_last_error()


@pytest.mark.parametrize("kw, match", [
    ({"n": 0}, "rows"), ({"actions": 0}, "actions"), ({"outcomes": 0}, "outcomes"), ({"outcomes": 4097}, "outcomes"),
    ({"policy": None}, "null input"), ({"stats": 68}, "aligned"), ({"losses": None}, "null output"), ({"dtype": 7}, "unknown type"),
])
def test_c_entry_of_the_loss_checks_its_arguments(kw, match):
    L = _lib.lib()
    a = _lib.LossArgs(4, 5, 2, 0, 64, 64, 64, 64, None, 64, 64)
    for k, v in kw.items():
        setattr(a, k, v)
    assert L.az_policy_value_loss_forward(C.byref(a), None) == -1
    assert match.encode() in L.az_last_error()
    a = _lib.LossArgs(4, 5, 2, 0, 64, 64, 64, 64, None, 64, 64)
    assert L.az_policy_value_loss_backward(C.byref(a), None) == -1 and b"null gradient" in L.az_last_error()


def _adam(**kw):
    a = _lib.AdamConfig(0.0, 0, 32, 64, 64, 64, None, None, 64, None, 64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _groups(*ends):
    return (_lib.AdamGroup * len(ends))(*(_lib.AdamGroup(1e-3, 0.9, 0.999, 1e-8, 0.0, 0, e) for e in ends))


@pytest.mark.parametrize("kw, size, ends, match", [
    ({"state_bits": 16}, 10, [1], "moments in 16 bits"), ({"m": None}, 10, [1], "null state"), ({"pieces": None}, 10, [1], "null state"),
    ({"scratch": None}, 10, [1], "null state"), ({"state_bits": 8}, 10, [1], "scales"), ({"m": 68}, 10, [1], "aligned"),
    ({"scratch": 72}, 10, [1], "aligned"), ({}, -1, [1], "-1 elements"), ({}, 1 << 39, [1], "elements"), ({}, 10, [2], "group 0 ends at 2 of 1"),
    ({}, 10, [0], "group 0 ends at 0 of 1"), ({}, 10, [1, 0], "group 1 ends at 0"), ({}, 10, [-1, 1], "group 0 ends at -1"),
])
def test_c_entry_of_the_step_checks_its_arguments(kw, size, ends, match):
    L = _lib.lib()
    p, s = (C.c_uint64 * 1)(64), (C.c_int64 * 1)(size)
    assert L.az_adam_step(C.byref(_adam(**kw)), len(ends), _groups(*ends), 1, p, p, s, None) == -1
    assert match.encode() in L.az_last_error()


def test_c_entry_of_the_step_refuses_misaligned_tensors_and_too_many_groups():
    L = _lib.lib()
    good, odd, s = (C.c_uint64 * 1)(64), (C.c_uint64 * 1)(66), (C.c_int64 * 1)(5000)
    for p, g in ((odd, good), (good, odd)):
        assert L.az_adam_step(C.byref(_adam()), 1, _groups(1), 1, p, g, s, None) == -1 and b"aligned to 4" in L.az_last_error()
    many = _groups(*([0] * _lib.OPTIM_GROUPS + [1]))
    assert L.az_adam_step(C.byref(_adam()), len(many), many, 1, good, good, s, None) == -1 and b"49 groups" in L.az_last_error()
    assert L.az_adam_step(C.byref(_adam()), 0, _groups(1), 1, good, good, s, None) == -1
    assert L.az_adam_step(C.byref(_adam()), 1, _groups(0), 0, None, None, None, None) == 0          # nothing to do is fine
    assert L.az_adam_scratch(0) == 0 and L.az_adam_scratch(241) == 2 * 8192 + 241 * 12 and L.az_adam_scratch(-1) == -1


def test_plan_of_the_moments():
    """Every tensor starts at a multiple of the pad, its pieces follow one another, the last one is what is left."""
    sizes = [1, 0, 256, 4096, 4097, 10000]
    n, offsets = len(sizes), (C.c_int64 * 7)()
    L = _lib.lib()
    count = L.az_adam_plan(n, (C.c_int64 * n)(*sizes), offsets, None)
    assert count == 1 + 0 + 1 + 1 + 2 + 3
    assert list(offsets) == [0, 256, 256, 512, 4608, 4608 + 4352, 4608 + 4352 + 10240]
    pieces = (C.c_uint32 * (4 * count))()
    assert L.az_adam_plan(n, (C.c_int64 * n)(*sizes), None, pieces) == count
    got = [tuple(pieces[4 * i:4 * i + 4]) for i in range(count)]
    assert got == [(0, 0, 0, 1), (2, 0, 1, 256), (3, 0, 2, 4096), (4, 0, 18, 4096), (4, 1, 34, 1), (5, 0, 35, 4096), (5, 1, 51, 4096), (5, 2, 67, 1808)]
    assert L.az_adam_plan(1, (C.c_int64 * 1)(-5), None, None) == -1 and L.az_adam_plan(-1, None, None, None) == -1


def test_eight_bit_moments_survive_a_checkpoint():
    """_encode returns exactly what _decode gave: every code of a block whatever its power of two, and a block whose
    largest value is small among its codes."""
    codes = torch.arange(256, dtype=torch.uint8)
    codes[0x7F] = codes[0xFF] = 0                                    # NaN
    for exponent in (-108, -20, 0, 40):
        x = _decode(codes.view(torch.float8_e4m3fn), torch.tensor([2.0 ** exponent]))
        back = _decode(*_encode(x, False))
        assert torch.equal(back, x)
        small = x * (x.abs() <= 3 * 2.0 ** (exponent - 9))
        assert torch.equal(_decode(*_encode(small, False)), small)
    root = torch.full((256,), 1e-12)
    root[0] = 1.0
    held = _decode(*_encode(root, True))
    assert held[0] == 1.0 and bool((held[1:] > 0).all())            # a root never becomes zero
    assert bool((_decode(*_encode(torch.zeros(512), True)) == 0).all())


def test_dense_layouts_are_told_apart():
    t = torch.zeros(4, 6, 3, 3)
    assert _dense(t) and _dense(t.to(memory_format=torch.channels_last)) and _dense(t.permute(3, 1, 0, 2)) and _dense(t[:, :, :0])
    assert not _dense(t[:, :3]) and not _dense(t[..., ::2]) and not _dense(torch.zeros(1, 4).expand(3, 4))
    assert _dense(torch.zeros(())) and _dense(torch.zeros(1)[:, None].expand(1, 1))


@pytest.mark.parametrize("given", [(1, 0, 0, 0, 0), (0, 1, 1, 1, 1), (1, 1, 0, 1, 1), (1, 1, 1, 1, 0)])
def test_a_gate_in_parts_is_refused(given):
    x = torch.zeros(2, 4, 3, 3)
    residual, *gate = [t if on else None for on, t in zip(given, (x, torch.zeros(2, 4), torch.zeros(2), torch.zeros(8, 2), torch.zeros(8)))]
    with pytest.raises(ValueError, match="a gate needs"):
        ops.norm_gate_residual(x, residual, torch.ones(4), torch.zeros(4), None, None, *gate)


@pytest.mark.parametrize("kw", [{"n": 1 << 24, "channels_last": 1}, {"n": 1 << 26, "c": 2}, {"n": 1 << 22, "c": 100, "hw": 4096},
                                {"n": 1, "c": 1 << 26}, {"n": 2, "c": (1 << 23) + 1, "channels_last": 1}])
def test_norms_of_more_workgroups_than_a_launch_takes_are_refused(kw):
    L = _lib.lib()
    sizes = (C.c_int64 * 3)()
    assert L.az_norm_sizes(C.byref(_norm_args(**kw)), sizes) == -1 and b"more than a launch takes" in L.az_last_error()
    fits = {"n": (1 << 24) - (1 << 15), "channels_last": 1}, {"n": 1 << 22, "c": 100}
    assert all(L.az_norm_sizes(C.byref(_norm_args(**k)), sizes) == 0 for k in fits)


@pytest.mark.parametrize("n, actions", [(1 << 24, 513), (1 << 26, 5)])
def test_losses_of_more_workgroups_than_a_launch_takes_are_refused(n, actions):
    L = _lib.lib()
    a = _lib.LossArgs(n, actions, 2, 0, 64, 64, 64, 64, None, 64, 64)
    assert L.az_policy_value_loss_forward(C.byref(a), None) == -1 and b"more than a launch takes" in L.az_last_error()
