"""Differentiable operators of the training step on the gfx950 kernels (az_norm_*, az_policy_value_loss_*
in include/azamd.h): what the reference writes as chains of torch modules (BatchNorm + ReLU and the end of a
squeeze-excitation block, src/model.py:40-92; the two cross-entropies, src/parallel_trainer.py:251-260), in a
few launches each.  They need a GPU tensor; there is no CPU fallback.

Activations and logits: float32, bfloat16 or float16, contiguous or channels-last (other strides are copied).
Parameters and statistics: float32.  All arithmetic and all sums are float32 or wider, outputs are rounded once.
The calls run on the current stream of the tensors' device, allocate only through torch and can be captured into
a HIP graph (a forward pass is refused there while an eager graph of the same leaf parameters lives on the default
stream: torch would accumulate the gradients on that stream).  First derivatives only.
Arguments are checked, and the autograd nodes written, in csrc/torch_ops.cpp.
"""
from . import _lib


def norm_act(x, weight, bias, running_mean, running_var, num_batches_tracked=None, training=True, momentum=0.1, eps=1e-5):
    """relu(batch_norm(x)) of x[boards, channels, height, width] (src/model.py:82-84).  training=True normalises
    with the batch's statistics and moves running_mean, running_var (float32 [channels], may be None) and
    num_batches_tracked (int64, may be None) in place; training=False normalises with the running ones."""
    return _lib.torch_ops().norm(x, None, weight, bias, running_mean, running_var, None, None, None, None, num_batches_tracked,
                                 training, momentum, eps)


def norm_gate_residual(x, residual, weight, bias, running_mean, running_var, fc1_weight, fc1_bias, fc2_weight, fc2_bias,
                       num_batches_tracked=None, training=True, momentum=0.1, eps=1e-5):
    """The end of a squeeze-excitation residual block (src/model.py:40-53, 85-92):
        y = batch_norm(x);  w, b = fc2(relu(fc1(mean of y over the board)));  relu(y * sigmoid(w) + b + residual)
    with fc1_weight [hidden, channels] and fc2_weight [2 channels, hidden], up to 1024 channels and hidden units.
    residual has x's shape and type; the rest is as in norm_act."""
    return _lib.torch_ops().norm(x, residual, weight, bias, running_mean, running_var, fc1_weight, fc1_bias, fc2_weight, fc2_bias,
                                 num_batches_tracked, training, momentum, eps)


def policy_value_loss(policy_logits, wl_logits, target_pis, target_wls, mask=None):
    """(loss, loss_pi, loss_wl): the means over the rows of the soft-target cross-entropies of policy_logits[n, actions]
    and wl_logits[n, outcomes], and their sum (src/parallel_trainer.py:251-260), as float32 scalars.  Gradients go to
    the logits.  Targets are float32 of the logits' shapes; a target of zero adds nothing whatever its logit.
    mask[n, actions] (bool or uint8): places that are false take no part, whatever logits and targets hold there; a row
    without any has loss and gradient zero."""
    return _lib.torch_ops().policy_value_loss(policy_logits, wl_logits, target_pis, target_wls, mask)
