"""Adam and AdamW over all tensors of a model in a few launches (az_adam_plan, az_adam_step in include/azamd.h),
with gradient clipping by the global norm and moments in 32 bits or in 8.  It needs parameters on a GPU; there is
no CPU fallback."""
import torch

from . import _lib

_PAD = _lib.OPTIM_PAD


def _dense(t):
    """Whether t's elements fill one stretch of memory, in whatever order of dimensions."""
    if t.numel() == 0:
        return True
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _encode(x, positive):
    """Float32 values -> (e4m3 codes, a power of two per 256), to nearest: exact for values that came out of _decode.
    positive: what is not zero does not become zero."""
    x = x.reshape(-1, _PAD)
    magnitude = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    mantissa, exponent = torch.frexp(magnitude.amax(1))
    exponent = torch.where(mantissa > 0, exponent - 9 + (mantissa > 0.875), torch.full_like(exponent, -108)).clamp(min=-108)
    scale = ((exponent + 127) << 23).view(torch.float32)          # 2 ** exponent, exactly
    y = x / scale[:, None]
    if positive:
        y = torch.where((y > 0) & (y < 2.0 ** -9), torch.full_like(y, 2.0 ** -9), y)
    return y.to(torch.float8_e4m3fn).reshape(-1), scale


def _decode(codes, scale):
    return (codes.float().reshape(-1, _PAD) * scale[:, None]).reshape(-1)


class FusedAdam(torch.optim.Optimizer):
    """torch.optim.Adam(params, lr, betas, eps, weight_decay), or AdamW with decoupled=True, for float32 parameters on
    one GPU, as two launches for all of them (per 240 tensors and parameter group; up to 48 groups).

    step(max_norm=x) also clips by the norm over the gradients of all parameters: they are scaled by
    min(1, x / (norm + 1e-6)) on the way into the update (the .grad tensors keep their values; torch's
    clip_grad_norm_ would overwrite them).  `grad_norm` is the norm of the last such step, a float32 scalar on the GPU.

    state_bits=32 keeps the moments in float32.  state_bits=8 keeps m and sqrt(v) as e4m3 codes with one power of two
    per 256, rounded at random (reproducibly: by `seed`, the step and the place): 2 bytes per weight instead of 8.
    Replicas of a model have to be given one seed (alphazero_amd.distributed.train_step checks that).
    Weights whose gradients stay within four decades of the largest of their 256 get the updates of 32 bits to about 1 %
    on average; further below v is held too large (no smaller than (4e-6)^2 of the block's largest) and the update is smaller.

    state_dict() is torch.optim.Adam's: per parameter step, exp_avg, exp_avg_sq (float32, also with 8-bit moments, which
    a load restores exactly: exp_avg all of it, sqrt(v) from 2^-63 on, where its square is a normal float32), so checkpoints go both ways.  Step counters live on the GPU; a step can be captured into
    a HIP graph (learning rate and the other hyper-parameters are constants of the capture).  amsgrad, maximize,
    sparse gradients and parameter groups added after construction are refused."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, decoupled=False, state_bits=32, seed=0):
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        if not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0:
            raise ValueError(f"betas must lie in [0, 1), got {betas}")
        if not lr >= 0.0 or not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError(f"lr, eps and weight_decay must not be negative, got {lr}, {eps}, {weight_decay}")
        self.state_bits, self.seed = state_bits, int(seed)
        self._built = False
        # capturable: what torch.optim.Adam calls an optimiser whose step counters are on the GPU
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      decoupled_weight_decay=bool(decoupled), capturable=True))
        self._build()

    # ------------------------------------------------------------------ layout
    def add_param_group(self, param_group):
        if self._built:
            raise RuntimeError("FusedAdam takes all its parameter groups at construction")
        super().add_param_group(param_group)

    def _build(self):
        params = [p for g in self.param_groups for p in g["params"]]
        device = params[0].device
        if len(self.param_groups) > _lib.OPTIM_GROUPS:
            raise ValueError(f"FusedAdam takes up to {_lib.OPTIM_GROUPS} parameter groups, got {len(self.param_groups)}")
        if device.type != "cuda":
            raise ValueError(f"FusedAdam needs parameters on a GPU, got one on {device}")
        for p in params:
            if p.dtype != torch.float32:
                raise TypeError(f"FusedAdam takes float32 parameters, got {p.dtype}")
            if p.device != device:
                raise ValueError(f"all parameters must be on one GPU, got {device} and {p.device}")
            if not _dense(p):
                raise ValueError(f"a parameter of shape {tuple(p.shape)} and strides {p.stride()} does not fill its memory")
        spans = sorted((p.data_ptr(), p.data_ptr() + 4 * p.numel()) for p in params if p.numel())
        if any(end > start for (_, end), (start, _) in zip(spans, spans[1:])):
            raise ValueError("two parameters share memory: each weight takes one update")
        self._params, self._device = params, device
        self._plan = _lib.torch_ops().AdamPlan(params)
        *self._offsets, total = self._plan.offsets()
        self._capacity = total
        shape = dict(device=device)
        self._step = torch.zeros(len(params), dtype=torch.float32, **shape)
        if self.state_bits == 32:
            self._flat = {"exp_avg": torch.zeros(total, **shape), "exp_avg_sq": torch.zeros(total, **shape)}
        else:
            self._flat = {}
            for name in ("exp_avg", "exp_rms"):
                self._flat[name] = torch.zeros(total, dtype=torch.uint8, **shape).view(torch.float8_e4m3fn)
                self._flat[name + "_scale"] = torch.full((total // _PAD,), 2.0 ** -108, **shape)
        self.grad_norm = torch.zeros((), **shape)
        self._ends, end = [], 0
        for g in self.param_groups:
            end += len(g["params"])
            self._ends.append(end)
        m, v = ("exp_avg", "exp_avg_sq") if self.state_bits == 32 else ("exp_avg", "exp_rms")
        self._plan.attach(self.state_bits, self.seed & 0xFFFFFFFF, self._step, self._flat[m], self._flat[v],
                          self._flat.get(m + "_scale"), self._flat.get(v + "_scale"), self.grad_norm)
        self._built = True
        self._attach()

    def _view(self, flat, i):
        p = self._params[i]
        return flat.as_strided(p.size(), p.stride(), self._offsets[i])

    def _attach(self):
        """self.state as torch.optim.Adam has it: views of the flat buffers."""
        self.state.clear()
        for i, (p, step) in enumerate(zip(self._params, self._step.unbind())):
            self.state[p] = {"step": step}
            if self.state_bits == 32:
                self.state[p].update((k, self._view(v, i)) for k, v in self._flat.items())

    def flat_state(self):
        """The live buffers: `step` (float32, one per parameter) and the moments, parameter after parameter in the order of
        the groups, each in the parameter's memory order and padded with zeros to a multiple of 256 elements.
        32 bits: exp_avg, exp_avg_sq.  8 bits: exp_avg and exp_rms (the root of exp_avg_sq) as float8_e4m3fn, and
        exp_avg_scale, exp_rms_scale, the power of two that each 256 of them are multiplied with."""
        return {"step": self._step, **self._flat}

    # ------------------------------------------------------------------ checkpoints
    def __getstate__(self):
        raise TypeError("FusedAdam is not copied or pickled as a whole: use state_dict()")

    def state_dict(self):
        """As torch.optim.Adam writes it by default, wherever it is read: the step counters on the host, and no group that says
        they are on the GPU (an Adam of parameters elsewhere would not step)."""
        sd = super().state_dict()
        sd["param_groups"] = [dict(g, capturable=False) for g in sd["param_groups"]]
        steps = self._step.cpu().unbind()
        if self.state_bits == 8:
            m = _decode(self._flat["exp_avg"], self._flat["exp_avg_scale"])
            v = _decode(self._flat["exp_rms"], self._flat["exp_rms_scale"]).square()
            sd["state"] = {i: {"exp_avg": self._view(m, i), "exp_avg_sq": self._view(v, i)} for i in range(len(self._params))}
        sd["state"] = {i: {**st, "step": steps[i]} for i, st in sd["state"].items()}
        return sd

    def load_state_dict(self, state_dict):
        for g in state_dict["param_groups"]:
            if g.get("amsgrad") or g.get("maximize"):
                raise ValueError("FusedAdam has no amsgrad and no maximize")
        before = self.param_groups
        if [len(g["params"]) for g in state_dict["param_groups"]] == [len(g["params"]) for g in before]:       # else torch refuses it
            keys = [k for g in state_dict["param_groups"] for k in g["params"]]
            for key, p in zip(keys, self._params):
                for name, v in state_dict["state"].get(key, {}).items():
                    if name in ("exp_avg", "exp_avg_sq") and v.shape != p.shape:
                        raise ValueError(f"{name} of a parameter of shape {tuple(p.shape)} has shape {tuple(v.shape)}")
        super().load_state_dict(state_dict)
        for g, old in zip(self.param_groups, before):
            g.setdefault("decoupled_weight_decay", old["decoupled_weight_decay"])
            g["capturable"] = True
        moments = {k: torch.zeros(self._capacity, device=self._device) for k in ("exp_avg", "exp_avg_sq")}
        with torch.no_grad():
            for i, p in enumerate(self._params):
                st = self.state.get(p, {})
                self._step[i] = float(st["step"]) if "step" in st else 0.0
                for k, flat in moments.items():
                    if k in st:
                        self._view(flat, i).copy_(st[k])
            if self.state_bits == 32:
                for k, flat in moments.items():
                    self._flat[k].copy_(flat)
            else:
                for name, x in (("exp_avg", moments["exp_avg"]), ("exp_rms", moments["exp_avg_sq"].sqrt())):
                    codes, scale = _encode(x, name == "exp_rms")
                    self._flat[name].copy_(codes)
                    self._flat[name + "_scale"].copy_(scale)
        self._attach()

    # ------------------------------------------------------------------ the step
    def step(self, closure=None, max_norm=None):
        """One update.  max_norm (> 0): clip by the global norm first."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if max_norm is not None and not max_norm > 0:
            raise ValueError(f"max_norm must be positive, got {max_norm}")
        self._plan.step([(g["lr"], *g["betas"], g["eps"], g["weight_decay"], g["decoupled_weight_decay"], end)
                         for end, g in zip(self._ends, self.param_groups)], max_norm or 0.0)
        return loss
