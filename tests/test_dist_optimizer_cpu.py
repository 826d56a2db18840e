"""CPU, world_size 2 over gloo: fit_mbgd with an optimizer hands every rank's optimizer the gradient summed over the
ranks, so that the replicas stay identical and equal to one process stepping on the whole batch."""
import os
import sys

import numpy as np
import torch
import torch.multiprocessing as mp

from test_dist_cpu import HERE, OracleStepper, _free_port, _problem


class HostAdamW:
    """The optimizer's interface on CPU tensors, stepping in fp64."""

    def __init__(self, params, lr):
        import wide_ref as ref
        self.params, self.lr, self.ref = params, lr, ref.AdamW(params, lr)

    def step(self, grads, lr=None, clip=None):
        assert clip is None
        self.ref.step(grads, lr=lr)
        for p, w in zip(self.params, self.ref.p):
            p.copy_(w)


def _views(p, z):
    import gcn_amd.lib as L
    d = L.dims(z)
    ends = [d.off_w0, d.off_b0, d.off_w1, d.off_b1, d.off_w2, d.off_b2, d.nparams]
    return [p[a:b] for a, b in zip(ends, ends[1:])]


def _worker(rank, world, port, z, T, B, epochs, out):
    sys.path.insert(0, HERE)
    sys.path.insert(0, os.path.dirname(HERE))
    import torch.distributed as dist
    from gcn_amd import train
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world)
    params, cubes, onehot = _problem(z, T, 5)
    sl = T // world
    lc, lo = np.ascontiguousarray(cubes[rank * sl:(rank + 1) * sl]), np.ascontiguousarray(onehot[rank * sl:(rank + 1) * sl])
    p = torch.from_numpy(params.copy())
    train.fit_mbgd(p, None, torch.from_numpy(lo), z, batch=B, min_err=0.0, max_iter=epochs, distributed=True, train_size=T,
                   stepper=OracleStepper(p, lc, lo, z), optimizer=HostAdamW(_views(p, z), 1e-3))
    out[rank] = p.numpy().copy()
    dist.destroy_process_group()


def test_two_ranks_step_alike():
    import oracle as orc
    z, T, B, epochs, world = 30, 24, 6, 2, 2
    out = mp.Manager().dict()
    mp.spawn(_worker, args=(world, _free_port(), z, T, B, epochs, out), nprocs=world, join=True)
    assert np.array_equal(out[0], out[1])
    params, cubes, onehot = _problem(z, T, 5)
    p = torch.from_numpy(params.copy())
    opt = HostAdamW(_views(p, z), 1e-3)
    sl, sub = T // world, B // world
    for _ in range(epochs):
        for i0 in range(T // B):
            total = 0
            for r in range(world):
                lo = r * sl
                _, _, g = orc.mbgd_step(p.numpy().copy(), cubes[lo:lo + sl], onehot[lo:lo + sl], i0 * sub, sub, z, 0.0)
                total = total + torch.from_numpy(g)
            opt.step(_views(total, z))
    # the same sums in another order: fp64 rounding, through at most 40 lr a step
    assert np.abs(out[0] - p.numpy()).max() <= 1e-10 * 40 * 1e-3 * epochs * (T // B)
