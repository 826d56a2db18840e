"""GPU: gradient norm and AdamW (moments in 32 and in 8 bits) against their 64-bit restatement."""
import math

import pytest
import torch

import wide_ref as ref
from gcn_amd import lib as L
from gcn_amd import ops

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
KINDS = [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)]
SIZES = [1, 255, 256, 257, 0, 1000, 4095, 4096, 4097, 13, 9000, 3, 20001]


def tensors(sizes, kind, seed, scale, offset=1):
    """Views of one flat buffer, the first starting `offset` elements in."""
    g = torch.Generator().manual_seed(seed)
    flat = (torch.randn(sum(sizes) + offset, generator=g, dtype=F64) * scale).to(kind).cuda()
    out, at = [], offset
    for n in sizes:
        out.append(flat[at:at + n])
        at += n
    return out


def mixed_scale_grads(sizes, kind, seed):
    """Gradients over many orders of magnitude, with zeros."""
    out = []
    for i, t in enumerate(tensors(sizes, F64, seed, 1.0)):
        g = torch.Generator().manual_seed(seed + i)
        mag = 10.0 ** (torch.rand(t.numel(), generator=g, dtype=F64) * 5 - 6)
        mag[torch.rand(t.numel(), generator=g) < 0.05] = 0.0
        out.append((t.cpu() * mag).to(kind).cuda())
    return out


def near(got, want, rel, floor, what):
    got, want = got.detach().cpu().double(), want.double()
    off = (got - want).abs()
    bound = rel * want.abs() + floor
    assert torch.isfinite(got).all() and (off <= bound).all(), (what, float((off - bound).max()))


def check(opt, want, params, steps, u, lr, prev=None):
    """After `steps` steps: with u half a step, one step rounds g * scale, m, v, the quotient and p.  m is off by at
    most 4u(|m| + |g|) a step and v by 5u(v + g^2), both weighted down by the betas after; the update lr * m / sqrt(v) is
    at most lr * C in size (C = 1 / sqrt(1 - beta2) for one step) and off by 16u of itself and u of p each step."""
    flat_p = torch.cat([p for p in want.p])
    size = 40 * lr                                   # |update| <= lr (1 / sqrt(1 - beta2) + decay |p|) < 40 lr
    got = opt.master if opt.master is not None else torch.cat([p.detach().reshape(-1) for p in params])
    near(got, flat_p, 4 * steps * u, steps * 40 * u * size, "p")
    if opt.master is not None:
        at = 0
        for p in params:
            assert torch.equal(p.detach().cpu(), opt.master[at:at + p.numel()].cpu().to(p.dtype)), "rounding of the master copy"
            at += p.numel()


@pytest.mark.parametrize("kind,grad_kind", KINDS + [(F64, F64)], ids=str)
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_steps_with_32_bit_moments(kind, grad_kind, offset):
    lr, u = 1e-2, ref.half_step(F64 if kind == F64 else F32)
    params = tensors(SIZES, kind, 1, 0.5, offset)
    decays = [0.1 * (i % 3) for i in range(len(SIZES))]
    want = ref.AdamW(params, lr, decays=decays)
    opt = ops.AdamW(params, lr=lr, weight_decay=decays)
    gmax = torch.zeros(sum(SIZES), dtype=F64)
    for k in range(5):
        grads = mixed_scale_grads(SIZES, grad_kind, 100 + k)
        opt.step(grads)
        want.step(grads)
        gmax = torch.maximum(gmax, torch.cat([g.cpu().double() for g in grads]).abs())
    assert opt.step_count == 5
    check(opt, want, params, 5, u, lr)
    m, v = opt.moments()
    tiny = torch.finfo(F64 if kind == F64 else F32).smallest_normal
    assert ((m.cpu().double() - torch.cat(want.m)).abs() <= 5 * 4 * u * gmax + tiny).all()
    assert ((v.cpu().double() - torch.cat(want.v)).abs() <= 5 * 5 * u * gmax ** 2 + tiny).all()


@pytest.mark.parametrize("kind,grad_kind", KINDS, ids=str)
def test_steps_with_8_bit_moments(kind, grad_kind):
    """The codes and scales are those of the 64-bit definition, bit for bit, step after step."""
    lr, u = 1e-2, ref.half_step(F32)
    params = tensors(SIZES, kind, 2, 0.5)
    want = ref.AdamW(params, lr, bits=8)
    opt = ops.AdamW(params, lr=lr, state_bits=8)
    for k in range(6):
        grads = mixed_scale_grads(SIZES, grad_kind, 200 + k)
        opt.step(grads)
        want.step(grads)
        mc, vc, ms, vs = want.codes
        assert torch.equal(opt.m_scale.cpu(), ms) and torch.equal(opt.v_scale.cpu(), vs), k
        assert torch.equal(opt.m.cpu() & 127, mc & 127) and torch.equal(opt.v.cpu(), vc), k
        assert torch.equal(ref.decode(opt.m.cpu().view(-1, 256), opt.m_scale.cpu()), ref.decode(mc.view(-1, 256), ms)), k
    check(opt, want, params, 6, u, lr)
    m, v = opt.moments()
    assert torch.equal(m.cpu(), torch.cat(want.m).float()) and torch.equal(v.cpu(), torch.cat(want.v).float())


@pytest.mark.parametrize("bits", [32, 8])
def test_magnitudes_at_the_edges(bits):
    """Gradients whose squares leave the range of fp32 at either end, next to ordinary ones and zeros, in one block
    and in blocks of their own."""
    n = 256 * 6 + 40
    g = torch.randn(n, generator=torch.Generator().manual_seed(3), dtype=F64)
    g[:256] *= 1e-30
    g[256:512] *= 1e-3
    g[300:310] = 1e-36
    g[512:768] = 0.0
    g[768:1024] *= 1e-42                              # subnormal
    g[1024:1280] *= 1e15
    g[1100:1200] = 1e-10
    g = g.float().cuda()
    p = torch.zeros(n, device="cuda")
    opt, want = ops.AdamW([p], lr=0.1, state_bits=bits), ref.AdamW([p], 0.1, bits=bits)
    for _ in range(3):
        opt.step([g])
        want.step([g])
        if bits == 8:
            mc, vc, ms, vs = want.codes
            assert torch.equal(opt.m_scale.cpu(), ms) and torch.equal(opt.v_scale.cpu(), vs)
            assert torch.equal(opt.m.cpu() & 127, mc & 127) and torch.equal(opt.v.cpu(), vc)
    # roots below sqrt of fp32's smallest squares vanish next to eps = 1e-8 and change p by less than 1e-10
    assert (p.cpu().double() - want.p[0]).abs().max() < 3 * 0.1 * 1e-5 + 1e-10


@pytest.mark.parametrize("n", [1000, 200001])
def test_a_square_beyond_fp32_stops_its_element(n):
    """A finite gradient whose square does not fit fp32 makes v infinite, and the element no longer moves; the others do."""
    p = torch.zeros(n, device="cuda")
    g = torch.full((n,), 0.1, device="cuda")
    g[n - 7] = 1e20
    opt = ops.AdamW([p], weight_decay=0.0)
    for _ in range(3):
        opt.step([g])
        g[n - 7] = 0.1
    assert torch.isfinite(p).all() and p[n - 7] == 0 and (p[: n - 7] < 0).all() and (p[n - 6:] < 0).all()
    assert opt.moments()[1][n - 7] == math.inf


@pytest.mark.parametrize("kind,bits", [(F32, 32), (F64, 32), (BF16, 8)], ids=str)
def test_a_loaded_optimiser_continues_bit_for_bit(kind, bits):
    params = tensors([700, 300], kind, 21, 0.5)
    opt = ops.AdamW(params, lr=1e-2, betas=(0.87, 0.983), state_bits=bits)
    for k in range(57):
        opt.step(tensors([700, 300], kind, 500 + k, 1e-2))
    other = [p.clone() for p in params]
    new = ops.AdamW(other, lr=1e-2, betas=(0.87, 0.983), state_bits=bits)
    new.load_state_dict(opt.state_dict())
    assert torch.equal(new._clock[:3], opt._clock[:3])
    g = tensors([700, 300], kind, 600, 1e-2)
    opt.step(g)
    new.step(g)
    assert all(torch.equal(a, b) for a, b in zip(params, other))
    assert all(torch.equal(a, b) for a, b in zip(opt.moments(), new.moments()))


def test_powers_of_long_runs():
    opt = ops.AdamW([torch.zeros(1, device="cuda")], betas=(0.0, 0.9))
    opt._set_step(10 ** 9)                       # 0.9^t has stopped changing long before
    assert opt._clock[0] == 10 ** 9 and opt._clock[1] == 0 and 0 <= opt._clock[2] < 1e-300


@pytest.mark.parametrize("kind,bits", [(F32, 32), (BF16, 32), (BF16, 8), (F64, 32)], ids=str)
def test_the_smallest_eps(kind, bits):
    """A parameter that never has a gradient stays where it is, down to the smallest eps that is taken."""
    smallest = 5e-324 if kind == F64 else 1e-45
    p = torch.ones(500, dtype=kind, device="cuda")
    opt = ops.AdamW([p], eps=smallest, weight_decay=0.0, state_bits=bits)
    opt.step([torch.zeros_like(p)])
    assert (p == 1).all()
    for eps in (0.0, smallest / 4, math.nan):
        with pytest.raises(ValueError):
            ops.AdamW([p], eps=eps, state_bits=bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_elements_beyond_32_bits(bits):
    """A tensor of more than 2^31 elements: the same gradient at a few places far apart and nowhere else."""
    n = (1 << 31) + 5003
    p = torch.zeros(n, dtype=BF16, device="cuda")
    g = torch.zeros(n, dtype=BF16, device="cuda")
    at = torch.tensor([0, 1 << 30, (1 << 31) - 1, 1 << 31, n - 257, n - 1], device="cuda")
    g[at] = 0.5
    norm = ops.grad_norm([g], math.inf)
    assert norm.tolist() == [pytest.approx(0.5 * math.sqrt(6), rel=1e-15), 1.0]
    opt = ops.AdamW([p], lr=0.25, weight_decay=0.0, state_bits=bits)
    opt.step([g])
    assert (p[at] == -0.25).all() and torch.count_nonzero(p) == 6
    m, v = opt.moments()
    assert (m[at] - 0.05).abs().max() < 0.05 * 2.0 ** -4 and torch.count_nonzero(m) == 6
    assert (v[at] - 0.00025).abs().max() < 0.00025 * 2.0 ** -2 and torch.count_nonzero(v) == 6


def test_a_root_above_zero_never_becomes_zero():
    g = torch.full((256,), 1e-7, device="cuda")
    g[0] = 1.0
    p = torch.zeros(256, device="cuda")
    opt = ops.AdamW([p], state_bits=8)
    opt.step([g])
    assert (opt.v.cpu()[1:] == 1).all() and opt.v.cpu()[0] == 0x7e
    g[5] = 0.0
    q = ops.AdamW([torch.zeros(256, device="cuda")], state_bits=8)
    q.step([g])
    assert q.v[5] == 0 and (q.v.cpu()[6:] == 1).all()


def test_ties_go_to_the_even_code():
    """beta1 = beta2 = 0 and a largest value of 448 * 2^k make the scale a power of two, so that values between two
    codes are exact ties."""
    between = (ref.VALUES[1:] + ref.VALUES[:-1]) / 2
    g = torch.zeros(256, dtype=F64)
    g[0] = 448.0
    g[1:127] = between
    g[128:254] = -between
    g = (g * 2.0 ** -10).float().cuda()
    opt = ops.AdamW([torch.zeros(256, device="cuda")], betas=(0.0, 0.0), state_bits=8)
    opt.step([g])
    assert opt.m_scale[0] == 2.0 ** -10
    want = torch.arange(126)
    want = want + want % 2
    assert torch.equal(opt.m.cpu()[1:127].long(), want) and torch.equal(opt.m.cpu()[128:254].long() & 127, want)
    assert torch.equal(opt.v.cpu()[1:127].long(), want.clamp(min=1))


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_one_launch_lists(bits):
    sizes = [(i * 37) % 411 for i in range(211)] + [70001]
    params, lr = tensors(sizes, F32, 5, 0.5), 1e-2
    want = ref.AdamW(params, lr, bits=bits)
    opt = ops.AdamW(params, lr=lr, state_bits=bits)
    for k in range(2):
        grads = tensors(sizes, F32, 300 + k, 1e-3)
        opt.step(grads)
        want.step(grads)
    check(opt, want, params, 2, ref.half_step(F32), lr)
    n = ops.grad_norm(grads, 1.0)
    assert n[0].item() == pytest.approx(float(torch.cat([g.cpu().double() for g in grads]).norm()), rel=1e-13)


@pytest.mark.parametrize("kind", [F32, F64, BF16], ids=str)
@pytest.mark.parametrize("sizes", [[98303], [98304], [3 << 15, 5], [50000, 47000, 1304], [1500001]])
def test_sizes_around_the_one_launch_step(kind, sizes):
    """Steps of middling sizes, whichever launch moves their clock."""
    params, lr, u = tensors(sizes, kind, 6, 0.5), 1e-2, ref.half_step(F64 if kind == F64 else F32)
    want, opt = ref.AdamW(params, lr), ops.AdamW(params, lr=lr)
    for k in range(3):
        grads = tensors(sizes, kind, 400 + k, 1e-3)
        opt.step(grads)
        want.step(grads)
        assert opt.step_count == k + 1
    check(opt, want, params, 3, u, lr)


@pytest.mark.parametrize("bits,sizes", [(32, [1]), (32, [64 * 256]), (32, [64 * 256 + 1]), (32, [33 * 256] * 16), (32, [1 << 20]),
                                        (32, [(1 << 20) - 1]), (32, [9000] * 64), (32, [9000] * 65), (32, [0, 5000, 0]),
                                        (8, [64 * 2048]), (8, [64 * 2048 + 1]), (8, [64 * 1024]), (8, [64 * 1024 + 1]), (8, [(5 << 20) - 1]), (8, [5 << 20]), (8, [777] * 64),
                                        (8, [777] * 65)], ids=str)
def test_the_clock_moves_once_a_step(bits, sizes):
    """Whatever launch moves it: alone, in groups that meet, in front of several; also where other work runs beside it."""
    params = tensors(sizes, F32, 30, 0.5)
    many = tensors([5000] * 40, F32, 31, 0.5)
    opt, other = ops.AdamW(params, state_bits=bits), ops.AdamW(many)
    grads, g2 = tensors(sizes, F32, 32, 1e-2), tensors([5000] * 40, F32, 33, 1e-2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    x1 = x2 = 1.0
    for k in range(20):
        opt.step(grads)
        with torch.cuda.stream(side):
            other.step(g2)
        x1, x2 = x1 * 0.9, x2 * 0.999
        if k % 7 == 3:
            assert opt._clock[:3].tolist() == [k + 1, x1, x2]
    torch.cuda.synchronize()
    for o in (opt, other):
        assert o._clock[:3].tolist() == [20, x1, x2] and not o._clock[7:].any()


def test_types_mixed_in_one_list():
    kinds = [F32, BF16, F16, BF16, F32, F16]
    params = [tensors([777 + i], k, i, 0.5)[0] for i, k in enumerate(kinds)]
    gk = [F32, BF16, F32, F32, F32, F16]
    want = ref.AdamW(params, 1e-2)
    opt = ops.AdamW(params, lr=1e-2)
    for s in range(3):
        grads = [tensors([777 + i], k, 50 + i + s, 1e-2)[0] for i, k in enumerate(gk)]
        clip = ops.grad_norm(grads, 0.1)
        assert clip[0].item() == pytest.approx(float(torch.cat([g.cpu().double() for g in grads]).norm()), rel=1e-13)
        opt.step(grads, clip=clip)
        want.step(grads, scale=clip[1].item())
    # fp32 parameters have their place in the master copy too, unused
    at = 0
    for p, w in zip(params, want.p):
        got = p.detach().cpu().double() if p.dtype == F32 else opt.master[at:at + p.numel()].cpu().double()
        near(got, w, 12 * ref.half_step(F32), 3 * 40 * ref.half_step(F32) * 0.4, "p")
        at += p.numel()


@pytest.mark.parametrize("kind", [F32, F64, BF16, F16], ids=str)
@pytest.mark.parametrize("sizes", [[1], [0, 5], [16384], [16385, 3, 100000], [3000001], [81920], [81921], [5121] * 16, [100] * 17])
def test_norm(kind, sizes):
    grads = tensors(sizes, kind, 9, 2.0)
    want = float(torch.cat([g.cpu().double() for g in grads]).norm())
    for limit in (want / 3, want * 3, math.inf):
        got = ops.grad_norm(grads, limit).tolist()
        # fp64 sums: n/256 additions at most in a row
        assert got[0] == pytest.approx(want, rel=2.0 ** -53 * (sum(sizes) / 256 + 40))
        assert got[1] == pytest.approx(min(1.0, limit / want), rel=1e-12)
    assert torch.equal(ops.grad_norm(grads, 1.0), ops.grad_norm(grads, 1.0))       # the same order every time


def test_norm_of_nothing_and_of_what_is_not_finite():
    z = torch.zeros(100, device="cuda")
    assert ops.grad_norm([z], 1.0).tolist() == [0.0, 1.0]
    assert ops.grad_norm([z[:0]], 1.0).tolist() == [0.0, 1.0]
    for bad in (math.inf, -math.inf, math.nan):
        g = torch.ones(5000, device="cuda")
        g[4321] = bad
        n, s = ops.grad_norm([z, g], 1.0).tolist()
        assert not math.isfinite(n) and math.isnan(s)
    big = torch.full((1000,), 3e38, device="cuda")                                     # squares beyond fp32
    assert ops.grad_norm([big], 1.0)[0].item() == pytest.approx(float(big[0]) * math.sqrt(1000), rel=1e-12)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind", [F32, BF16], ids=str)
def test_a_step_that_is_not_finite_is_left_out(kind, bits):
    params = tensors([300, 5000], kind, 4, 0.5)
    opt = ops.AdamW(params, state_bits=bits)
    opt.step(tensors([300, 5000], kind, 5, 1e-2))
    before, p0 = opt.state_dict(), [p.clone() for p in params]
    grads = tensors([300, 5000], kind, 6, 1e-2)
    grads[1][77] = math.inf
    opt.step(grads, clip=ops.grad_norm(grads, 1.0))
    after = opt.state_dict()
    assert after["step"] == 1 == before["step"]
    assert all(torch.equal(before[k], after[k]) for k in before if k != "step")
    assert all(torch.equal(a, b) for a, b in zip(p0, params))
    grads[1][77] = 0.5
    opt.step(grads, clip=ops.grad_norm(grads, 1.0))
    assert opt.step_count == 2 and not torch.equal(p0[1], params[1])


def test_without_a_norm_what_is_not_finite_stays_in_its_place():
    g = torch.full((1000,), 0.1, device="cuda")
    g[300] = math.nan
    g[600] = math.inf
    p32, p8 = torch.zeros(1000, device="cuda"), torch.zeros(1000, device="cuda")
    a, b = ops.AdamW([p32]), ops.AdamW([p8], state_bits=8)
    for _ in range(2):
        a.step([g])
        b.step([g])
    off = torch.isnan(p32)
    assert off.nonzero().flatten().tolist() == [300, 600]
    off = torch.isnan(b.moments()[0])
    assert off[256:768].all() and not off[:256].any() and not off[768:].any()


@pytest.mark.parametrize("bits", [32, 8])
def test_state_travels(bits):
    sizes = [1000, 7]
    params = tensors(sizes, BF16, 7, 0.5)
    opt = ops.AdamW(params, state_bits=bits)
    for k in range(3):
        opt.step(tensors(sizes, BF16, 70 + k, 1e-2))
    state = opt.state_dict()
    other = [torch.zeros_like(p) for p in params]
    new = ops.AdamW(other, state_bits=bits)
    new.load_state_dict(state)
    assert new.step_count == 3 and all(torch.equal(a, b) for a, b in zip(params, other))
    g = tensors(sizes, BF16, 80, 1e-2)
    opt.step(g)
    new.step(g)
    a, b = opt.state_dict(), new.state_dict()
    assert a["step"] == b["step"] and all(torch.equal(a[k], b[k]) for k in a if k != "step")
    assert all(torch.equal(x, y) for x, y in zip(params, other))
    with pytest.raises(ValueError):
        ops.AdamW(other, state_bits=40 - bits).load_state_dict(state)
    with pytest.raises(ValueError):
        ops.AdamW(other[:1], state_bits=bits).load_state_dict(state)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(bits):
    """Norm and step in a graph, replayed between eager work; the count, the rate and the gradients are read on the device."""
    sizes = [3000, 17, 256]
    params, eager = tensors(sizes, F32, 8, 0.5), tensors(sizes, F32, 8, 0.5)
    grads = tensors(sizes, F32, 9, 1e-2)
    rate = torch.tensor([1e-2], dtype=F64, device="cuda")
    opt, plain = ops.AdamW(params, lr=rate, state_bits=bits), ops.AdamW(eager, lr=rate, state_bits=bits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for o in (opt, plain):
            o.step(grads, clip=ops.grad_norm(grads, 0.3))
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step(grads, clip=ops.grad_norm(grads, 0.3))
    assert opt.step_count == 1
    for k in range(4):
        for t, new in zip(grads, tensors(sizes, F32, 10 + k, 10.0 ** -k)):
            t.copy_(new)
        rate.fill_(10.0 ** -(2 + k))
        g.replay()
        plain.step(grads, clip=ops.grad_norm(grads, 0.3))
        torch.cuda.synchronize()
        assert opt.step_count == plain.step_count == 2 + k
        assert all(torch.equal(a, b) for a, b in zip(params, eager))
        assert all(torch.equal(a, b) for a, b in zip(opt.moments(), plain.moments()))


def test_network_views_cover_the_flat_vector():
    z = L.geometry(103, 9)
    d = L.dims(z)
    flat = torch.arange(d.nparams, dtype=F32, device="cuda")
    views = ops.param_views(flat, z)
    assert [v.numel() for v in views] == [3420, 20, 100 * d.pout, 100, 900, 9]
    assert torch.equal(torch.cat(views), flat)


def test_refused():
    p, g = torch.zeros(10, device="cuda"), torch.zeros(10, device="cuda")
    opt = ops.AdamW([p])
    two = torch.zeros(4, 6, device="cuda")
    for call, err in [
        (lambda: ops.AdamW([]), ValueError),
        (lambda: ops.AdamW([p.cpu()]), TypeError),
        (lambda: ops.AdamW([p.int()]), TypeError),
        (lambda: ops.AdamW([two.t()]), ValueError),
        (lambda: ops.AdamW([p, p[5:]]), ValueError),
        (lambda: ops.AdamW([p, p.double()]), TypeError),
        (lambda: ops.AdamW([p.double()], state_bits=8), TypeError),
        (lambda: ops.AdamW([p], state_bits=16), ValueError),
        (lambda: ops.AdamW([p], betas=(0.9, 1.0)), ValueError),
        (lambda: ops.AdamW([p], eps=-1.0), ValueError),
        (lambda: ops.AdamW([p], weight_decay=[0.1, 0.1]), ValueError),
        (lambda: opt.step([]), ValueError),
        (lambda: opt.step([g[:9]]), ValueError),
        (lambda: opt.step([g.bfloat16()]), TypeError),
        (lambda: opt.step([g.cpu()]), TypeError),
        (lambda: opt.step([torch.zeros(20, device="cuda")[::2]]), ValueError),
        (lambda: opt.step([g], clip=g), TypeError),
        (lambda: opt.step([g], lr=g), TypeError),
        (lambda: opt.load_state_dict({"step": -1, "m": opt.m, "v": opt.v}), ValueError),
        (lambda: ops.grad_norm([], 1.0), ValueError),
        (lambda: ops.grad_norm([g], 0.0), ValueError),
        (lambda: ops.grad_norm([g], math.nan), ValueError),
        (lambda: ops.grad_norm([g.cpu()], 1.0), TypeError),
        (lambda: ops.grad_norm([two.t()], 1.0), ValueError),
    ]:
        with pytest.raises(err):
            call()
    assert opt.step_count == 0 and not p.any()
    moved = torch.zeros(10, device="cuda")
    other = ops.AdamW([moved])
    moved.data = torch.zeros(10, device="cuda")           # the memory the optimiser knew is gone
    with pytest.raises(ValueError):
        other.step([g])


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_are_those_that_the_optimiser_was_made_for(bits):
    """The list, the memory, the size and the type are looked at before a step; what is read out does not hang on the list."""
    p, g = torch.zeros(512, device="cuda"), torch.full((512,), 0.5, device="cuda")
    more = torch.zeros(512, device="cuda")
    opt = ops.AdamW([p], state_bits=bits)
    opt.step([g])
    m, v = opt.moments()
    for change, back in [(lambda: opt.params.append(more), lambda: opt.params.pop()),
                         (lambda: opt.params.extend([more] * 200), lambda: opt.params.__delitem__(slice(1, None))),
                         (lambda: opt.params.clear(), lambda: opt.params.append(p)),
                         (lambda: setattr(opt, "params", (p,)), lambda: setattr(opt, "params", [p]))]:
        change()
        for grads in ([g], [g] * len(opt.params), [g] * 2):
            with pytest.raises(ValueError):
                opt.step(grads)
        assert all(torch.equal(a, b) for a, b in zip(opt.moments(), (m, v)))
        back()
    whole = p.data
    for other in (whole[:500], whole.view(torch.bfloat16), whole.view(torch.bfloat16)[:512], whole.view(torch.int32)):
        p.data = other
        for grads in ([g], [g[:500]], [g.bfloat16()]):
            with pytest.raises((ValueError, TypeError)):
                opt.step(grads)
        p.data = whole
    opt.params[0] = None
    with pytest.raises(TypeError):
        opt.step([g])
    opt.params[0] = p
    assert opt.step_count == 1 and not more.any()
    opt.step([g])
    assert opt.step_count == 2


@pytest.mark.parametrize("kind,bits", [(F32, 32), (F64, 32), (BF16, 32), (F32, 8), (BF16, 8)], ids=str)
def test_state_of_another_size_or_type_is_refused(kind, bits):
    """The state is in public attributes; a step writes to no tensor that is too small for it."""
    params, grads = tensors([700, 0, 300], kind, 60, 0.5), tensors([700, 0, 300], kind, 61, 1e-2)
    opt = ops.AdamW(params, state_bits=bits)
    opt.step(grads)
    for name in ("m", "v", "m_scale", "v_scale", "master", "_clock"):
        own = getattr(opt, name)
        if own is None:
            others = [torch.zeros(4, device="cuda")]
        else:
            others = [own[:-1], own.cpu(), own.to(torch.float16), torch.cat([own, own])[::2], torch.cat([own, own]), None, 3]
        for other in others:
            setattr(opt, name, other)
            with pytest.raises((ValueError, TypeError)):
                opt.step(grads)
            if bits == 8 and name != "_clock" and own is not None:
                with pytest.raises((ValueError, TypeError)):
                    opt.moments()
        setattr(opt, name, own)
    assert opt.step_count == 1
    opt.step(grads)
    assert opt.step_count == 2


@pytest.mark.parametrize("kinds", [[F32], [F32, BF16]], ids=str)
def test_bytes_behind_a_tensor_stay_0_in_a_block_that_is_not_finite(kinds):
    """One launch (one type) and several."""
    n = 300
    params = [torch.zeros(n, dtype=k, device="cuda") for k in kinds]
    opt = ops.AdamW(params, state_bits=8)
    for value in (math.nan, 0.1, math.inf):
        grads = [torch.full((n,), 0.1, dtype=k, device="cuda") for k in kinds]
        for g in grads:
            g[290] = value
        opt.step(grads)
        for codes, scale in ((opt.m, opt.m_scale), (opt.v, opt.v_scale)):
            for i in range(len(kinds)):
                c, s = codes[i * 512:(i + 1) * 512].cpu(), scale[2 * i:2 * i + 2].cpu()
                assert torch.isfinite(s[0]) and torch.isnan(s[1])
                assert (c[256:300] == 0x7f).all() and not c[300:].any() and (c[:256] == 0x7e).all()


def scaled_norm(tensors):
    """The norm of fp64 gradients of any size: of the values over their largest, summed without rounding."""
    flat = torch.cat([t.cpu().double().reshape(-1) for t in tensors])
    high = 2.0 ** math.floor(math.log2(float(flat.abs().max())))
    return math.sqrt(math.fsum(((flat / high) ** 2).tolist())), high


@pytest.mark.parametrize("sizes", [[1], [1000], [81921, 5], [300001], [100] * 40 + [7]], ids=str)
@pytest.mark.parametrize("scale,other", [(1e200, 1.0), (1e200, 1e200), (1e-200, 0.0), (1e-200, 1e-200), (1e-310, 0.0), (1e-170, 1e-130),
                                         (3e153, 1e154), (1e300, 1e-300)])
def test_norm_of_doubles_whose_squares_leave_the_range(sizes, scale, other):
    """A finite norm is found whatever its squares do: sums of n terms of one size, and a rounding of each square."""
    grads = tensors(sizes, F64, 12, 1.0)
    for g in grads:
        g.clamp_(-4, 4)
        g.mul_(scale)
        g[1::3] = other
    norm, high = scaled_norm(grads)
    limit = 1e-3 * high
    out = ops.grad_norm(grads, limit).tolist()
    rel = 2.0 ** -53 * (sum(sizes) / 256 + 40) + 2.0 ** -1074 / (norm * high)
    assert out[0] / high == pytest.approx(norm, rel=rel)
    assert out[1] == pytest.approx(min(1.0, limit / high / norm), rel=1e-12 + rel)


@pytest.mark.parametrize("n", [1000, 300001])
def test_norm_beyond_doubles_and_a_step_just_below(n):
    g = torch.full((n,), 1.7e308, dtype=F64, device="cuda")
    norm, factor = ops.grad_norm([g], 1.0).tolist()
    assert norm == math.inf and math.isnan(factor)
    g.fill_(1e300)
    mixed = [g, torch.full((50,), 3e38, device="cuda")]
    clip = ops.grad_norm(mixed, 1.0)
    assert clip[0].item() == pytest.approx(1e300 * math.sqrt(n), rel=1e-12)
    for others in (1e300, 1.0, 1e-200, 0.0):
        g.fill_(others)
        g[5] = math.nan
        assert all(map(math.isnan, ops.grad_norm([g], 1.0).tolist()))
        g[5] = -0.0
        assert ops.grad_norm([g], 1.0)[0].item() == pytest.approx(others * math.sqrt(n - 1), rel=1e-12)
    g[5] = -math.inf
    assert math.isnan(ops.grad_norm([g], 1.0)[1].item())
    g.fill_(1e300)
    p = torch.zeros(n, dtype=F64, device="cuda")
    opt = ops.AdamW([p])
    opt.step([g], clip=ops.grad_norm([g], 1.0))
    assert opt.step_count == 1
    assert (opt.moments()[0] * (10 * math.sqrt(n)) - 1).abs().max() < 1e-12


@pytest.mark.parametrize("kind,grad_kind", [(F32, F32), (BF16, F32), (BF16, BF16), (F64, F64)], ids=str)
@pytest.mark.parametrize("n", [1000, 200001, 1500001])
@pytest.mark.parametrize("limit", [1e-3, 1e-9])
def test_a_clip_factor_below_fp32(kind, grad_kind, n, limit):
    """Gradients near the largest fp32 clipped to a small norm: the factor is no normal fp32 number, the clipped
    gradient is.  m rounds g * factor (twice, a factor of two numbers) and its own two operations: 4 half steps."""
    grads = [g.mul_(3e37) for g in tensors([n], grad_kind, 40, 1.0)]
    params = tensors([n], kind, 41, 0.5)
    opt = ops.AdamW(params)
    clip = ops.grad_norm(grads, limit)
    assert 0 < clip[1].item() < 1e-39
    opt.step(grads, clip=clip)
    want = 0.1 * (grads[0].cpu().double() * clip[1].item())
    wide = F64 if kind == F64 else F32
    off = (opt.moments()[0].cpu().double() - want).abs()
    # products that are no normal fp32 numbers are off by half their distance, m by that of its own
    assert (off <= 6 * ref.half_step(wide) * want.abs() + 3 * 2.0 ** -149).all()
    assert want.abs().max() > 1e-8 * limit


@pytest.mark.parametrize("n", [1000, 200001])
def test_a_clip_factor_above_fp32(n):
    """A factor from elsewhere that brings tiny gradients up."""
    g = torch.full((n,), 2.0 ** -140, device="cuda")
    opt = ops.AdamW([torch.zeros(n, device="cuda")])
    opt.step([g], clip=torch.tensor([1.0, 2.0 ** 140], dtype=F64, device="cuda"))
    assert (opt.moments()[0] * 10 - 1).abs().max() < 1e-6


@pytest.mark.parametrize("kind", [F32, F64, BF16], ids=str)
@pytest.mark.parametrize("n", [1000, 200001])
@pytest.mark.parametrize("beta1,lr", [(0.9, 1e-3), (0.0, 1e-3), (0.9, 100.0)])
def test_gradients_near_the_largest_number_of_both_signs(kind, n, beta1, lr):
    """Finite gradients leave m finite, and an element whose v is beyond the type where it is, also where g - m or
    lr * m is beyond it too; one that is not finite is seen."""
    big = 0.95 * torch.finfo(kind).max
    p = torch.zeros(n, dtype=kind, device="cuda")
    g = torch.full((n,), 0.1, dtype=kind, device="cuda")
    opt, m = ops.AdamW([p], lr=lr, betas=(beta1, 0.999), weight_decay=0.0), 0.0
    for k in range(40):
        g[n - 7] = big if k < 30 else -big
        opt.step([g])
        m = beta1 * m + (1 - beta1) * (g[n - 7].item() / big)
    got = opt.moments()[0][n - 7].double().item() / big
    assert abs(got - m) <= 1e-5
    assert p[n - 7] == 0 and torch.isfinite(p).all() and torch.count_nonzero(p < 0) == n - 1
    g[n - 7] = math.inf
    opt.step([g])
    assert torch.isnan(p[n - 7]) and torch.count_nonzero(torch.isfinite(p)) == n - 1


@pytest.mark.parametrize("kind", [F32, F64, BF16], ids=str)
@pytest.mark.parametrize("lr", [1.0, 3.0, 1e6, -5.0])
def test_rates_of_one_or_more(kind, lr):
    """The quotient is that of the formula, and of an element without a gradient still 0 with the smallest eps."""
    u = ref.half_step(F64 if kind == F64 else F32)
    params, grads = tensors([3000, 70], kind, 70, 0.5), tensors([3000, 70], kind, 71, 1e-2)
    opt, want = ops.AdamW(params, lr=lr, weight_decay=0.0), ref.AdamW(params, lr, decays=[0.0, 0.0])
    opt.step(grads)
    want.step(grads)
    held = opt.master if opt.master is not None else torch.cat(params)
    # the first step is of size lr; its quotient, roots and products round 16 times at most, p once
    assert ((held.cpu().double() - torch.cat(want.p)).abs() <= 16 * u * abs(lr) + u * torch.cat(want.p).abs()).all()
    p = torch.ones(500, dtype=kind, device="cuda")
    still = ops.AdamW([p], lr=lr, eps=5e-324 if kind == F64 else 1e-45, weight_decay=0.0)
    still.step([torch.zeros_like(p)])
    assert (p == 1).all()
