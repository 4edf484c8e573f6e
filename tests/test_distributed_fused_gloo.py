"""World-size-2 gloo tests (CPU) of data-parallel training with FusedAdam's 8-bit moments: ranks whose moments are rounded
differently part after one step.  The optimiser's kernels need a GPU, so its step is stated here in elementary operations
(the same key of seed, step and place); everything around it is the package's own."""
import os

import numpy as np
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from alphazero_amd.optim import FusedAdam
from test_distributed_gloo import _free_port

PAD = 256


def _rounded(x, chance, positive):
    """x as e4m3 codes times a power of two per 256, rounded up where the way to the next code and `chance` make 1."""
    block = x.reshape(-1, PAD)
    top = block.abs().amax(1)
    mantissa, exponent = torch.frexp(top)
    scale = torch.ldexp(torch.ones_like(top), (exponent - 9 + (mantissa > 0.875)).clamp(min=-108))
    scale = torch.where(top > 0, scale, torch.full_like(scale, 2.0 ** -108))[:, None]
    y = block.abs() / scale
    place = (torch.frexp(y)[1] - 1).clamp(min=-6) - 3
    q = torch.floor(torch.ldexp(y, -place) + chance.reshape(-1, PAD))
    if positive:
        q = torch.where(y > 0, q.clamp(min=1), q)
    return (torch.copysign(torch.ldexp(q, place), block) * scale).reshape(-1)


class HostAdam(FusedAdam):
    """FusedAdam with its step on the host: Adam with clipping and the moments rounded to 8 bits at random."""

    def __init__(self, params, lr=1e-3, weight_decay=0.0, state_bits=32, seed=0):
        self.state_bits, self.seed, self._built = state_bits, int(seed), False
        torch.optim.Optimizer.__init__(self, params, dict(lr=lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=weight_decay))
        self.params, self.t = list(self.param_groups[0]["params"]), 0
        n = sum(p.numel() for p in self.params)
        self.m, self.r = torch.zeros(-(-n // PAD) * PAD), torch.zeros(-(-n // PAD) * PAD)

    def step(self, closure=None, max_norm=None):
        self.t += 1
        group = self.param_groups[0]
        p, g = (torch.cat([t.reshape(-1) for t in ts]).float() for ts in ([q.detach() for q in self.params], [q.grad for q in self.params]))
        n = p.numel()
        if max_norm:
            g = g * min(1.0, max_norm / (float(g.norm()) + 1e-6))
        g = torch.nn.functional.pad(g + group["weight_decay"] * p, (0, self.m.numel() - n))
        m = 0.9 * self.m + 0.1 * g
        r = (0.999 * self.r ** 2 + 0.001 * g ** 2).sqrt()
        step = group["lr"] / (1 - 0.9 ** self.t) * m / (r / (1 - 0.999 ** self.t) ** 0.5 + 1e-8)
        p = p - step[:n]
        for q, part in zip(self.params, p.split([q.numel() for q in self.params])):
            q.detach().copy_(part.view_as(q))
        z = torch.arange(self.m.numel()) + self.seed * 0x9E3779B9 + self.t * 0x85EBCA6B
        for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B), (16, 1)):
            z = z & 0xFFFFFFFF
            z = (z ^ (z >> shift)) * factor
        self.m, self.r = (m, r) if self.state_bits == 32 else (
            _rounded(m, (z & 0xFFFF).float() / 65536, False), _rounded(r, (z >> 16 & 0xFFFF).float() / 65536, True))


def _start(rank, world, port):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.set_num_threads(1)
    from alphazero_amd import parallel_trainer
    from alphazero_amd.model import AlphaZeroNet
    parallel_trainer.FusedAdam = HostAdam
    AlphaZeroNet.use_fused_ops = lambda self, on=True: self              # (the fused norms need a GPU too)
    torch.manual_seed(0)
    return AlphaZeroNet(num_blocks=1, num_filters=8)


def _data():
    rs = np.random.RandomState(1)
    pol = rs.rand(8, 192).astype(np.float32)
    return ((rs.rand(8, 3, 8, 8) > 0.5).astype(np.float32), pol / pol.sum(1, keepdims=True),
            np.tile(np.array([[1.0, 0.0], [0.0, 1.0]], np.float32), (4, 1)))


def _everywhere(flat, world=2):
    both = [torch.empty_like(flat) for _ in range(world)]
    dist.all_gather(both, flat)
    return torch.equal(both[0], both[1])


def _learn(rank, world, port, ret, tmp):
    model = _start(rank, world, port)
    try:
        from alphazero_amd.parallel_trainer import ParallelTrainer
        # self-play's seed differs from rank to rank, as several ranks need it
        tr = ParallelTrainer(model, device="cpu", checkpoint_dir=os.path.join(tmp, f"r{rank}"), verbose=False, seed=17 + rank,
                             fused_ops=True, optimizer_bits=8)
        tr.add_examples(list(zip(*_data())))
        torch.manual_seed(11)
        for _ in range(2):
            assert np.isfinite(tr.learn(epochs=1, batch_size=5)["loss"])   # 5, 5, 5, 1: in the last one rank 1's slice is empty
        assert tr.optimizer.t == 8 and tr.optimizer.same_rounding
        assert _everywhere(torch.cat([p.detach().reshape(-1) for p in model.parameters()]))
        assert _everywhere(tr.optimizer.m) and _everywhere(tr.optimizer.r)
        ret[rank] = 1
    finally:
        dist.destroy_process_group()


def _refused(rank, world, port, ret, tmp):
    model = _start(rank, world, port)
    try:
        from alphazero_amd.distributed import train_step
        s, p, w = (torch.from_numpy(a[4 * rank:4 * rank + 4]) for a in _data())
        for bits, seed in ((8, 3 + rank), (32 if rank else 8, 0)):
            opt = HostAdam(model.parameters(), state_bits=bits, seed=seed)
            try:
                train_step(model, opt, s, p, w, global_batch=8)
            except ValueError as e:
                assert "same state_bits and seed" in str(e)
            else:
                raise AssertionError("not refused")
            assert opt.t == 0
        train_step(model, HostAdam(model.parameters(), state_bits=32, seed=rank), s, p, w, global_batch=8)    # 32 bits: nothing is rounded at random
        assert _everywhere(torch.cat([q.detach().reshape(-1) for q in model.parameters()]))
        ret[rank] = 1
    finally:
        dist.destroy_process_group()


def _two_ranks(work, tmp_path):
    ctx = mp.get_context("spawn")
    ret, port = ctx.Manager().dict(), _free_port()
    procs = [ctx.Process(target=work, args=(r, 2, port, ret, str(tmp_path))) for r in range(2)]
    for p in procs:
        p.start()
    for p in procs:
        p.join(180)
    assert all(p.exitcode == 0 for p in procs), [p.exitcode for p in procs]
    assert dict(ret) == {0: 1, 1: 1}


def test_two_ranks_with_8_bit_moments_stay_identical(tmp_path):
    _two_ranks(_learn, tmp_path)


def test_ranks_that_round_differently_are_refused(tmp_path):
    _two_ranks(_refused, tmp_path)
