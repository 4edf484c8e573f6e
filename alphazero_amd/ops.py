"""Differentiable operators of the training step on the gfx950 kernels (az_norm_*, az_policy_value_loss_*
in include/azamd.h): what the reference writes as chains of torch modules (BatchNorm + ReLU and the end of a
squeeze-excitation block, src/model.py:40-92; the two cross-entropies, src/parallel_trainer.py:251-260), in a
few launches each.  They need a GPU tensor; there is no CPU fallback.

Activations and logits: float32, bfloat16 or float16, contiguous or channels-last (other strides are copied).
Parameters and statistics: float32.  All arithmetic and all sums are float32 or wider, outputs are rounded once.
The calls run on the current stream of the tensors' device, allocate only through torch and can be captured into
a HIP graph.  First derivatives only.
"""
import ctypes as C
import functools

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}     # AZ_F32, AZ_BF16, AZ_F16


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(entry, args, device):
    """One library call on the device's current stream."""
    stream = torch.cuda.current_stream(device).cuda_stream
    if torch.cuda.current_device() == device.index:
        _lib.check(entry(args, stream))
    else:
        with torch.cuda.device(device):
            _lib.check(entry(args, stream))


def _check_parameter(name, t, shape, device):
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the activations on {device}")
    return t if t.is_contiguous() else t.contiguous()


def _check_statistic(name, t, shape, dtype, device):
    if t.dtype != dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {device}")


@functools.lru_cache(maxsize=256)
def _norm_sizes(n, c, hw, hidden, dtype, channels_last, training):
    sizes = (C.c_int64 * 3)()
    _lib.check(_lib.lib().az_norm_sizes(_lib.NormArgs(n, c, hw, hidden, dtype, channels_last, training), sizes))
    return tuple(sizes)


def _layout(x):
    """(is channels-last, memory format).  A tensor that is both counts as contiguous."""
    if not x.is_contiguous() and x.is_contiguous(memory_format=torch.channels_last):
        return 1, torch.channels_last
    return 0, torch.contiguous_format


class _Norm(Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, fc1_weight, fc1_bias, fc2_weight, fc2_bias, running_mean, running_var,
                num_batches, training, momentum, eps):
        n, c, h, w = x.shape
        last, fmt = _layout(x)
        x = x.contiguous(memory_format=fmt)
        if residual is not None:
            residual = residual.contiguous(memory_format=fmt)
        head = (n, c, h * w, 0 if residual is None else fc1_weight.shape[0], _DTYPES[x.dtype], last, int(training))
        saved_bytes, forward_bytes, ctx.backward_bytes = _norm_sizes(*head)
        saved = torch.empty(saved_bytes, dtype=torch.uint8, device=x.device)
        workspace = torch.empty(forward_bytes, dtype=torch.uint8, device=x.device)
        out = torch.empty_like(x)
        args = _lib.NormArgs(*head, eps, momentum, x.data_ptr(), _ptr(residual), weight.data_ptr(), bias.data_ptr(),
                             _ptr(running_mean), _ptr(running_var), _ptr(num_batches), _ptr(fc1_weight), _ptr(fc1_bias),
                             _ptr(fc2_weight), _ptr(fc2_bias), saved.data_ptr(), workspace.data_ptr(), out.data_ptr())
        _call(_lib.lib().az_norm_forward, args, x.device)
        ctx.head = head + (eps, momentum)
        ctx.format = fmt
        if training:
            # written behind torch's back: whoever watches the buffers' version counters has to see it
            torch.autograd.graph.increment_version([t for t in (running_mean, running_var, num_batches) if t is not None])
        ctx.save_for_backward(x, weight, bias, fc1_weight, fc1_bias, fc2_weight, fc2_bias, saved)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, bias, fc1_weight, fc1_bias, fc2_weight, fc2_bias, saved = ctx.saved_tensors
        gated = fc1_weight is not None
        grad = grad.contiguous(memory_format=ctx.format)
        workspace = torch.empty(ctx.backward_bytes, dtype=torch.uint8, device=x.device)
        dx = torch.empty_like(x)
        dresidual = torch.empty_like(x) if gated else None
        small = [torch.empty_like(t) if t is not None else None for t in (weight, bias, fc1_weight, fc1_bias, fc2_weight, fc2_bias)]
        args = _lib.NormArgs(*ctx.head, x.data_ptr(), None, weight.data_ptr(), bias.data_ptr(), None, None, None,
                             _ptr(fc1_weight), _ptr(fc1_bias), _ptr(fc2_weight), _ptr(fc2_bias), saved.data_ptr(),
                             workspace.data_ptr(), None, grad.data_ptr(), dx.data_ptr(), _ptr(dresidual), *map(_ptr, small))
        _call(_lib.lib().az_norm_backward, args, x.device)
        return (dx, dresidual, *small, None, None, None, None, None, None)


def _check_norm(x, weight, bias, running_mean, running_var, num_batches, training):
    if not x.is_cuda:
        raise ValueError(f"the fused norms need a GPU tensor, got one on {x.device}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"activations must be float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() != 4:
        raise ValueError(f"activations must have shape [boards, channels, height, width], got {tuple(x.shape)}")
    n, c, h, w = x.shape
    if x.numel() == 0:
        raise ValueError(f"no values to normalise in shape {tuple(x.shape)}")
    if training and n * h * w < 2:
        raise ValueError(f"the batch's statistics need more than one value per channel, got shape {tuple(x.shape)}")
    if not training and (running_mean is None or running_var is None):
        raise ValueError("evaluation needs running statistics")
    shape = weight.shape if weight.dim() == 1 and weight.shape[0] == c else torch.Size((c,))
    for name, t in (("running_mean", running_mean), ("running_var", running_var)):
        if t is not None:
            _check_statistic(name, t, shape, torch.float32, x.device)
    if num_batches is not None:
        _check_statistic("num_batches_tracked", num_batches, torch.Size(()), torch.int64, x.device)
    return (_check_parameter("weight", weight, shape, x.device), _check_parameter("bias", bias, shape, x.device))


def norm_act(x, weight, bias, running_mean, running_var, num_batches_tracked=None, training=True, momentum=0.1, eps=1e-5):
    """relu(batch_norm(x)) of x[boards, channels, height, width] (src/model.py:82-84).  training=True normalises
    with the batch's statistics and moves running_mean, running_var (float32 [channels], may be None) and
    num_batches_tracked (int64, may be None) in place; training=False normalises with the running ones."""
    weight, bias = _check_norm(x, weight, bias, running_mean, running_var, num_batches_tracked, training)
    return _Norm.apply(x, None, weight, bias, None, None, None, None, running_mean, running_var, num_batches_tracked,
                       bool(training), float(momentum), float(eps))


def norm_gate_residual(x, residual, weight, bias, running_mean, running_var, fc1_weight, fc1_bias, fc2_weight, fc2_bias,
                       num_batches_tracked=None, training=True, momentum=0.1, eps=1e-5):
    """The end of a squeeze-excitation residual block (src/model.py:40-53, 85-92):
        y = batch_norm(x);  w, b = fc2(relu(fc1(mean of y over the board)));  relu(y * sigmoid(w) + b + residual)
    with fc1_weight [hidden, channels] and fc2_weight [2 channels, hidden], up to 1024 channels and hidden units.
    residual has x's shape and type; the rest is as in norm_act."""
    weight, bias = _check_norm(x, weight, bias, running_mean, running_var, num_batches_tracked, training)
    if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
        raise ValueError(f"residual must be like x ({tuple(x.shape)}, {x.dtype}, {x.device}), got {tuple(residual.shape)}, "
                         f"{residual.dtype}, {residual.device}")
    if fc1_weight.dim() != 2:
        raise ValueError(f"fc1_weight must have shape (hidden, channels), got {tuple(fc1_weight.shape)}")
    hidden, c = fc1_weight.shape[0], x.shape[1]
    if not 1 <= hidden <= 1024 or c > 1024:
        raise ValueError(f"a gate takes up to 1024 channels and 1 to 1024 hidden units, got {c} and {hidden}")
    fc1_weight = _check_parameter("fc1_weight", fc1_weight, torch.Size((hidden, c)), x.device)
    fc1_bias = _check_parameter("fc1_bias", fc1_bias, torch.Size((hidden,)), x.device)
    fc2_weight = _check_parameter("fc2_weight", fc2_weight, torch.Size((2 * c, hidden)), x.device)
    fc2_bias = _check_parameter("fc2_bias", fc2_bias, torch.Size((2 * c,)), x.device)
    return _Norm.apply(x, residual, weight, bias, fc1_weight, fc1_bias, fc2_weight, fc2_bias, running_mean, running_var,
                       num_batches_tracked, bool(training), float(momentum), float(eps))


class _Loss(Function):
    @staticmethod
    def forward(ctx, policy, wl, target_pis, target_wls, mask):
        n, actions = policy.shape
        ctx.head = (n, actions, wl.shape[1], _DTYPES[policy.dtype])
        losses = torch.empty(3, dtype=torch.float32, device=policy.device)
        stats = torch.empty(8 * n, dtype=torch.float32, device=policy.device)
        args = _lib.LossArgs(*ctx.head, policy.data_ptr(), wl.data_ptr(), target_pis.data_ptr(), target_wls.data_ptr(), _ptr(mask),
                             losses.data_ptr(), stats.data_ptr())
        _call(_lib.lib().az_policy_value_loss_forward, args, policy.device)
        ctx.save_for_backward(policy, wl, target_pis, target_wls, mask, stats)
        ctx.set_materialize_grads(False)
        return losses[0], losses[1], losses[2]

    @staticmethod
    @once_differentiable
    def backward(ctx, g_loss, g_pi, g_wl):
        policy, wl, target_pis, target_wls, mask, stats = ctx.saved_tensors
        dpolicy, dwl = torch.empty_like(policy), torch.empty_like(wl)
        args = _lib.LossArgs(*ctx.head, policy.data_ptr(), wl.data_ptr(), target_pis.data_ptr(), target_wls.data_ptr(), _ptr(mask),
                             None, stats.data_ptr(), _ptr(g_loss), _ptr(g_pi), _ptr(g_wl), dpolicy.data_ptr(), dwl.data_ptr())
        _call(_lib.lib().az_policy_value_loss_backward, args, policy.device)
        return dpolicy, dwl, None, None, None


def policy_value_loss(policy_logits, wl_logits, target_pis, target_wls, mask=None):
    """(loss, loss_pi, loss_wl): the means over the rows of the soft-target cross-entropies of policy_logits[n, actions]
    and wl_logits[n, outcomes], and their sum (src/parallel_trainer.py:251-260), as float32 scalars.  Gradients go to
    the logits.  Targets are float32 of the logits' shapes; a target of zero adds nothing whatever its logit.
    mask[n, actions] (bool or uint8): places that are false take no part, whatever logits and targets hold there; a row
    without any has loss and gradient zero."""
    if not policy_logits.is_cuda:
        raise ValueError(f"policy_value_loss needs GPU tensors, got one on {policy_logits.device}")
    if policy_logits.dtype not in _DTYPES or wl_logits.dtype != policy_logits.dtype:
        raise TypeError("logits must be both float32, both bfloat16 or both float16, got "
                        f"{policy_logits.dtype} and {wl_logits.dtype}")
    if policy_logits.dim() != 2 or wl_logits.dim() != 2 or policy_logits.shape[0] != wl_logits.shape[0]:
        raise ValueError(f"logits must be [n, actions] and [n, outcomes], got {tuple(policy_logits.shape)} and {tuple(wl_logits.shape)}")
    if policy_logits.numel() == 0 or wl_logits.numel() == 0:
        raise ValueError("policy_value_loss of no rows or no classes")
    if wl_logits.shape[1] > 4096:
        raise ValueError(f"up to 4096 outcomes, got {wl_logits.shape[1]}")
    device = policy_logits.device
    for name, t, like in (("target_pis", target_pis, policy_logits), ("target_wls", target_wls, wl_logits)):
        if t.dtype != torch.float32:
            raise TypeError(f"{name} must be float32, got {t.dtype}")
        if t.shape != like.shape:
            raise ValueError(f"{name} must have the logits' shape {tuple(like.shape)}, got {tuple(t.shape)}")
        if t.requires_grad:
            raise ValueError(f"{name} must not require a gradient")
    if mask is not None and (mask.dtype not in (torch.bool, torch.uint8) or mask.shape != policy_logits.shape):
        raise ValueError(f"mask must be bool or uint8 of shape {tuple(policy_logits.shape)}, got {mask.dtype} {tuple(mask.shape)}")
    if any(t is not None and t.device != device for t in (wl_logits, target_pis, target_wls, mask)):
        raise ValueError(f"all tensors must be on {device}")
    return _Loss.apply(policy_logits.contiguous(), wl_logits.contiguous(), target_pis.contiguous(), target_wls.contiguous(),
                       None if mask is None else mask.contiguous())
