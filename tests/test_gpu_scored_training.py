"""GPU: the scoring, loss and optimiser operators together, as a training step and an evaluation use them: on a linear
classifier over a large vocabulary, and in the framework's own trainers."""
import numpy as np
import pytest
import torch

import oracle as orc
import synth
import wide_ref as ref
from gcn_amd import lib as L
from gcn_amd import ops, train

pytestmark = pytest.mark.gpu


def network(dtype, z=40, classes=13, n=200, seed=3):
    rng = np.random.default_rng(seed)
    geom = L.geometry(z, classes)
    d = L.dims(geom)
    cubes = torch.from_numpy(rng.random((n, 9 * z)).astype(dtype)).cuda()
    onehot = np.zeros((n, classes), dtype=np.int32)
    onehot[np.arange(n), rng.integers(0, classes, n)] = 1
    params = torch.from_numpy((rng.random(d.nparams) * 0.2 - 0.1).astype(dtype)).cuda()
    return params, cubes, torch.from_numpy(onehot).cuda(), geom


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("classes,n", [(13, 200), (9, 33), (16, 1), (13, 1700)])
def test_logits_are_what_the_probabilities_come_from(dtype, classes, n, monkeypatch):
    if n == 1700:
        monkeypatch.setenv("CCNN_FWD_CHUNK", "512")
    params, cubes, _, geom = network(dtype, classes=classes, n=n)
    logits = ops.forward_logits(params, cubes, geom)
    probs, am = ops.forward(params, cubes, geom)
    x = logits.cpu().double()
    want = torch.softmax(x, 1)
    u = ref.half_step(logits.dtype)
    # exp, sum of `classes` terms and quotient; exp's argument is exact here, its error 2 half steps and |x| of them
    bound = (classes + 8 + 2 * float(x.abs().max())) * u
    assert ((probs.cpu().double() - want).abs() <= bound * want).all()
    clear = torch.topk(want, 2, 1).values
    clear = (clear[:, 0] - clear[:, 1]) > 4 * bound
    assert torch.equal(am.cpu()[clear].long(), x.argmax(1)[clear]) and (n == 1 or clear.float().mean() > 0.9)
    assert ops.forward_logits(params, cubes[:0], geom).shape == (0, classes)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_pixels_scored_against_their_labels(dtype):
    params, cubes, onehot, geom = network(dtype, n=300)
    labels = onehot.argmax(1).int() + 1
    labels[7] = 0                                        # unlabelled
    r = train.score(params, cubes, labels, geom, top=3)
    logits = ops.forward_logits(params, cubes, geom)
    want = ref.log_probs(logits, labels - 1, 3)
    bound = ref.score_bound(logits, want, logits.dtype) + 8 * ref.half_step(logits.dtype) * want["logp"].abs()
    assert ((r.logp.cpu().double() - want["logp"]).abs() <= bound).all() and r.logp[7] == 0
    assert torch.equal(r.top_index.cpu(), want["top_index"])
    hits = (r.top_index[:, 0] + 1 == labels).sum().item()
    assert hits / 300 == pytest.approx(train.evaluate(params, cubes, labels, geom))
    with pytest.raises(ValueError):
        train.score(params, cubes, labels[:5], geom)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16], ids=str)
def test_steps_of_a_linear_classifier(kind, bits):
    """logits = x W + b -> log probabilities and entropy -> gradients -> norm, clip -> AdamW; every step's operators
    against 64 bits on the values that the step itself saw, so that nothing piles up."""
    rows, width, classes, lr = 96, 64, 5003, 1e-2
    g = torch.Generator().manual_seed(11)
    x = torch.randn(rows, width, generator=g).cuda()
    y = torch.randint(0, classes, (rows,), generator=g, dtype=torch.int32).cuda()
    y[::10] = -1
    weight, bias = (0.1 * torch.randn(width, classes, generator=g)).to(kind).cuda(), torch.zeros(classes, dtype=kind, device="cuda")
    opt = ops.AdamW([weight, bias], lr=lr, weight_decay=[0.01, 0.0], state_bits=bits)
    want = ref.AdamW([weight, bias], lr, decays=[0.01, 0.0], bits=bits)
    d_logp, d_entropy = torch.full((rows,), -1.0 / rows, device="cuda"), torch.full((rows,), -0.01 / rows, device="cuda")
    losses = []
    for step in range(4):
        logits = (x @ weight.float() + bias.float()).to(kind)
        r = ops.log_probs(logits, y, top=5)
        full = ref.log_probs(logits, y, 5)
        assert torch.equal(r.top_index.cpu(), full["top_index"])
        losses.append(float((r.logp * d_logp).sum()))
        bound = ref.score_bound(logits, full, torch.float32)
        assert ((r.logp.cpu().double() - full["logp"]).abs() <= bound + 1e-6 * full["logp"].abs()).all()
        d = ops.log_probs_grad(logits, y, r, d_logp, d_entropy)
        exact = ref.log_probs_grad(full, y, d_logp, d_entropy)
        assert (d.cpu().double() - exact).norm() <= (4 * ref.half_step(kind) + 1e-5) * exact.norm()
        grads = [(x.t() @ d.float()).contiguous(), d.float().sum(0)]
        clip = ops.grad_norm(grads, 0.05)
        norm = float(torch.cat([t.reshape(-1) for t in grads]).cpu().double().norm())
        assert clip.tolist() == pytest.approx([norm, min(1.0, 0.05 / norm)], rel=1e-12)
        grads = [t if kind == torch.float32 or i == 0 else t.to(kind) for i, t in enumerate(grads)]      # both types of gradient
        opt.step(grads, clip=clip)
        want.step(grads, scale=clip[1].item())
        if bits == 8:
            assert torch.equal(opt.m_scale.cpu(), want.codes[2]) and torch.equal(opt.v.cpu(), want.codes[1])
        held = opt.master if opt.master is not None else torch.cat([weight.reshape(-1), bias])
        u = ref.half_step(torch.float32)
        size = 40 * lr
        off = (held.cpu().double() - torch.cat(want.p)).abs()
        assert (off <= (step + 1) * u * (4 * torch.cat(want.p).abs() + 40 * size)).all()
    assert opt.step_count == 4 and all(np.isfinite(losses))


@pytest.mark.parametrize("dtype,bits", [(np.float32, 32), (np.float32, 8), (np.float64, 32)])
@pytest.mark.parametrize("max_norm", [None, 1e-3])
def test_the_trainer_steps_with_adamw(dtype, bits, max_norm):
    """fit_mbgd(optimizer=...) against the same loop written out: the framework's gradient of each batch, the norm of
    the batch mean, the 64-bit step."""
    params, cubes, onehot, geom = network(dtype, n=100)
    start = params.clone()
    d, B, lr, epochs = L.dims(geom), 25, 1e-3, 2
    opt = train.adamw(params, geom, lr=lr, weight_decay=0.1, state_bits=bits)
    hist = train.fit_mbgd(params, cubes, onehot, geom, batch=B, min_err=0.0, max_iter=epochs, optimizer=opt, max_norm=max_norm)
    assert hist.lr == [lr] * epochs and opt.step_count == epochs * 4
    p, keep = start.clone(), [0, 2, 3, 4, 5] if dtype == np.float32 else list(range(6))
    views = [ops.param_views(p, geom)[i] for i in keep]
    want = ref.AdamW(views, lr, decays=[[0.1, 0.0] * 3][0] if len(keep) == 6 else [0.1, 0.1, 0.0, 0.1, 0.0], bits=bits)
    for _ in range(epochs):
        for first in range(0, 100, B):
            g, _ = ops.mbgd_grad(p, cubes, onehot, first, B, geom)
            grads = [ops.param_views(g, geom)[i] for i in keep]
            scale = 1.0
            if max_norm is not None:
                norm = float(torch.cat([t.cpu().double() for t in grads]).norm())
                scale = min(1.0, max_norm * B / norm)
            want.step(grads, scale=scale)
            for v, w in zip(views, want.p):
                v.copy_(w.to(p.dtype))
            want.p = [v.cpu().double() for v in views]          # the next gradient is of the rounded parameters
    # a step moves a parameter by at most 40 lr; gradients of parameters apart by the steps' rounding differ by as
    # much again, relative to their size, and eight steps of it stay far below 1e-3 of a move in fp32, 1e-10 in fp64.
    # With 8 bits a code may fall on the other side of a border then: one code is an eighth of its moment.
    move = 40 * lr
    tol = move * ({32: 1e-3, 8: 0.02}[bits] if dtype == np.float32 else 1e-10)
    assert (params - p).abs().max().item() <= tol
    if dtype == np.float32:
        assert torch.equal(params[d.off_b0:d.off_w1], start[d.off_b0:d.off_w1])        # that trainer's frozen bias


def test_the_trainer_refuses_what_it_cannot_step():
    params, cubes, onehot, geom = network(np.float32, n=50)
    other = train.adamw(params.clone(), geom)
    with pytest.raises(ValueError):
        train.fit_mbgd(params, cubes, onehot, geom, batch=25, optimizer=other)
    with pytest.raises(ValueError):
        train.fit_mbgd(params, cubes, onehot, geom, batch=25, max_norm=1.0)
    rate = torch.ones(1, dtype=torch.float64, device="cuda")
    with pytest.raises(ValueError):
        train.fit_mbgd(params, cubes, onehot, geom, batch=25, optimizer=train.adamw(params, geom, lr=rate))


def test_training_with_adamw_runs_end_to_end():
    x, y, z = 24, 20, 60
    scene, labels = synth.small_scene(x, y, z, 3)
    got = train.prepare(scene, labels, x, y, z, torch.float32, 77)
    opt = train.adamw(got["params"], z, lr=2e-3)
    hist = train.fit_mbgd(got["params"], got["train_cubes"], got["onehot"], z, batch=16, min_err=0.0, max_iter=3, optimizer=opt,
                          max_norm=1.0, keep_tail=True)
    assert len(hist.loss) == 3 and np.isfinite(hist.loss).all()
    r = train.score(got["params"], got["test_cubes"], got["test_labels"], z)
    assert torch.isfinite(r.logp).all() and torch.isfinite(r.entropy).all()


@pytest.mark.parametrize("dtype,bits", [(np.float32, 32), (np.float32, 8), (np.float64, 32)])
@pytest.mark.parametrize("max_norm", [None, 1e-3])
def test_the_short_last_batch_weighs_as_much_as_the_others(dtype, bits, max_norm):
    """keep_tail: a batch of ten after four of 25 enters the moments as its mean does beside theirs."""
    params, cubes, onehot, geom = network(dtype, n=110)
    start = params.clone()
    d, B, lr, epochs = L.dims(geom), 25, 1e-3, 2
    opt = train.adamw(params, geom, lr=lr, weight_decay=0.1, state_bits=bits)
    train.fit_mbgd(params, cubes, onehot, geom, batch=B, min_err=0.0, max_iter=epochs, optimizer=opt, max_norm=max_norm,
                   keep_tail=True)
    assert opt.step_count == epochs * 5
    p, keep = start.clone(), [0, 2, 3, 4, 5] if dtype == np.float32 else list(range(6))
    views = [ops.param_views(p, geom)[i] for i in keep]
    want = ref.AdamW(views, lr, decays=[[0.1, 0.0] * 3][0] if len(keep) == 6 else [0.1, 0.1, 0.0, 0.1, 0.0], bits=bits)
    for _ in range(epochs):
        for first, nb in [(0, 25), (25, 25), (50, 25), (75, 25), (100, 10)]:
            g, _ = ops.mbgd_grad(p, cubes, onehot, first, nb, geom)
            grads = [ops.param_views(g, geom)[i].cpu().double() * (B / nb) for i in keep]
            scale = 1.0
            if max_norm is not None:
                scale = min(1.0, max_norm * B / float(torch.cat(grads).norm()))
            want.step(grads, scale=scale)
            for v, w in zip(views, want.p):
                v.copy_(w.to(p.dtype))
            want.p = [v.cpu().double() for v in views]
    # as for whole batches: a step moves a parameter by at most 40 lr, rounding stays far below 1e-3 of it in fp32 and
    # 1e-10 in fp64, a code on the other side of a border is an eighth of its moment
    tol = 40 * lr * ({32: 1e-3, 8: 0.02}[bits] if dtype == np.float32 else 1e-10)
    assert (params - p).abs().max().item() <= tol
