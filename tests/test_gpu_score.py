"""GPU: log_probs and log_probs_grad against their 64-bit restatement, at the sizes, strides, masks and
values where they can go wrong."""
import math
import sys

import pytest
import torch

import wide_ref as ref
from gcn_amd import lib as L
from gcn_amd import ops

pytestmark = pytest.mark.gpu

KINDS = [torch.float32, torch.float64, torch.bfloat16, torch.float16]
INF = math.inf


def wide(kind):
    return torch.float64 if kind == torch.float64 else torch.float32


def problem(rows, classes, kind, seed=0, pad=0, spread=3.0, ids=torch.int32):
    g = torch.Generator().manual_seed(seed * 7919 + rows * 31 + classes)
    x = torch.randn(rows, classes + pad, generator=g, dtype=torch.float64) * spread
    y = torch.randint(0, classes, (rows,), generator=g).to(ids)
    return x.to(kind).cuda()[:, :classes], y.cuda()


def close(got, want, bound, what):
    """Equal where not finite, within `bound` elsewhere."""
    got, want = got.detach().cpu().double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    fine = torch.isfinite(want)
    odd = ~fine & ~torch.isnan(want)
    assert torch.equal(got[odd], want[odd]), what
    assert torch.isfinite(got[fine]).all(), what
    off = (got - want).abs()[fine]
    limit = bound.expand_as(want)[fine] if isinstance(bound, torch.Tensor) else bound
    assert (off <= limit).all(), (what, float(off.max()), float((off / limit).max()))


def check_scores(x, y, top, got=None, want_entropy=True):
    r = got if got is not None else ops.log_probs(x, y, top=top, want_entropy=want_entropy)
    want = ref.log_probs(x, y, top)
    b = ref.score_bound(x, want, wide(x.dtype))
    assert r.logp.dtype == wide(x.dtype)
    u = ref.half_step(wide(x.dtype))
    close(r.logp, want["logp"], b + 4 * u * want["logp"].abs().nan_to_num(0, 0, 0), "logp")
    close(r.stats[2], want["m"], 0.0, "m")
    close(r.stats[3], want["l"], b, "l")
    if want_entropy:
        p, lp = want["p"], want["lp"]
        weight = torch.where(p > 0, p * (lp.abs() + 1), 0.0).sum(1)        # t carries the terms' errors times |x - m|
        close(r.entropy, want["entropy"], 2 * b * (1 + weight.nan_to_num(0)) , "entropy")
    else:
        assert r.entropy is None
    if top:
        assert torch.equal(r.top_index.cpu(), want["top_index"])
        close(r.top_logp, want["top_logp"], b[:, None] + 4 * u * want["top_logp"].abs().nan_to_num(0, 0, 0), "top_logp")
    else:
        assert r.top_logp is None and r.top_index is None
    return r, want


def check_grad(x, y, r, want, d_logp, d_entropy, out=None):
    got = ops.log_probs_grad(x, y, r, d_logp, d_entropy, out=out)
    g = ref.log_probs_grad(want, y, d_logp, d_entropy)
    b = ref.score_bound(x, want, wide(x.dtype))[:, None]
    u = ref.half_step(wide(x.dtype))
    zero = torch.zeros(x.shape[0], dtype=torch.float64)
    dl = zero if d_logp is None else d_logp.cpu().double().abs()
    dh = zero if d_entropy is None else d_entropy.cpu().double().abs()
    p, lp = want["p"].nan_to_num(0), want["lp"].nan_to_num(0, 0, 0).abs()
    h = want["entropy"].nan_to_num(0)[:, None]
    # p is off by b + 4u(|log p| + 1) of itself, log p by b, H by 2 b (1 + H); then each product and sum rounds once
    rel = 3 * b + 8 * u * (lp + 1)
    parts = dl[:, None] * (p + (g.abs() > 0)) + dh[:, None] * p * (lp + h + 1)
    tiny = torch.finfo(x.dtype).smallest_normal * ref.half_step(x.dtype) * 2
    bound = rel * parts * (1 + h) + ref.half_step(x.dtype) * 1.01 * g.abs().nan_to_num(0) + tiny
    assert got.dtype == x.dtype
    close(got, g, bound, "gradient")
    return got


def weights(rows, kind, seed=1):
    g = torch.Generator().manual_seed(seed)
    return (-torch.rand(rows, generator=g, dtype=torch.float64)).to(wide(kind)).cuda(), \
        (0.1 * torch.randn(rows, generator=g, dtype=torch.float64)).to(wide(kind)).cuda()


SHAPES = [(1, 1), (1, 2), (3, 13), (257, 13), (5, 16), (7, 17), (130, 31), (4, 64), (3, 65), (9, 255), (2, 1000), (5, 1024),
          (16385, 13), (16400, 41), (16390, 200), (20000, 5), (3, 1025), (2, 2049), (3, 4097), (1, 32003), (4, 50251), (520, 1025), (513, 1037), (600, 8190), (3, 65536), (2, 65537), (1, 128000), (2, 131073), (70, 8191), (600, 70001), (2050, 8190)]


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("rows,classes", SHAPES)
def test_scores_and_gradient(rows, classes, kind):
    if kind == torch.float64 and rows * classes > 4000000:
        rows = 1
    x, y = problem(rows, classes, kind)
    r, want = check_scores(x, y, min(classes, 20))
    dl, dh = weights(rows, kind)
    check_grad(x, y, r, want, dl, dh)


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("rows,classes", [(6, 13), (5, 777), (3, 9000)])
@pytest.mark.parametrize("top", [0, 1, 2, 13, 64])
def test_every_count_of_alternatives(rows, classes, kind, top):
    x, y = problem(rows, classes, kind, seed=2)
    check_scores(x, y, min(top, classes), want_entropy=top % 2 == 0)


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("rows,classes,pad", [(5, 13, 3), (4, 333, 1), (3, 5001, 7), (2, 40000, 13), (37, 2000, 8)])
def test_strided_rows_in_and_out(rows, classes, pad, kind):
    x, y = problem(rows, classes, kind, seed=3, pad=pad)
    r, want = check_scores(x, y, 7, want_entropy=True)
    dl, dh = weights(rows, kind)
    buf = torch.full((rows, classes + 5), 7.0, dtype=kind, device="cuda")
    check_grad(x, y, r, want, dl, dh, out=buf[:, 2:2 + classes])
    assert (buf[:, :2] == 7).all() and (buf[:, 2 + classes:] == 7).all()       # nothing beside the rows is touched
    whole = torch.empty(rows * classes + 1, dtype=kind, device="cuda")
    whole[1:].view(rows, classes).copy_(x)
    odd = whole[1:].view(rows, classes)                                          # starts one element into an allocation
    check_scores(odd, y, 7)


def odd_rows(classes, kind):
    low = torch.finfo(kind).min
    rows = 12
    x, y = problem(rows, classes, kind, seed=4)
    x = x.clone()
    x[0] = -INF                                   # nothing allowed
    x[1] = low                                    # everything at the type's lowest value
    x[2, : classes // 2] = -INF
    x[3] = -INF
    x[3, classes - 1] = 2.0                       # one class allowed
    x[4] = 0.0                                    # all equal
    x[5, classes // 2] = INF
    x[6, classes - 1] = math.nan
    x[7] = math.nan
    x[8, ::2] = low
    x[9] = -INF
    x[9, 0] = low
    x[10, :] = -0.0
    x[10, classes // 2:] = 0.0                    # zeros of both signs are equal
    y = y.clone()
    y[2] = classes - 1
    y[3] = 0
    y[11] = -100                                  # no target
    return x, y


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("classes", [1, 5, 13, 300, 9001, 70000, 200000])
def test_masked_and_odd_values(classes, kind):
    x, y = odd_rows(classes, kind)
    r, want = check_scores(x, y, min(classes, 20))
    dl, dh = weights(len(y), kind)
    check_grad(x, y, r, want, dl, dh)
    check_grad(x, y, r, want, dl, None)
    check_grad(x, y, r, want, None, dh)


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("classes,times", [(13, 1400), (50, 1400), (200, 1400), (1500, 45), (9001, 43), (4096, 90)])
def test_masked_and_odd_values_in_many_rows(classes, times, kind):
    """The row counts from which other shapes of the kernels take over."""
    x, y = odd_rows(classes, kind)
    x, y = x.repeat(times, 1), y.repeat(times)
    r, want = check_scores(x, y, min(classes, 20))
    dl, dh = weights(len(y), kind)
    check_grad(x, y, r, want, dl, dh)


@pytest.mark.parametrize("kind", KINDS, ids=str)
def test_ranges_that_do_not_fit_the_type(kind):
    top = torch.finfo(kind).max
    x = torch.tensor([[top, -top, 0.0, top, 1.0], [-top, -top, -top, 0.0, top]], dtype=kind).cuda()
    y = torch.tensor([0, 3], dtype=torch.int32).cuda()
    r = ops.log_probs(x, y, top=5)
    assert r.logp.tolist()[0] == pytest.approx(-math.log(2.0), rel=1e-6)
    assert r.entropy.tolist() == pytest.approx([math.log(2.0), 0.0], abs=1e-6)
    assert r.top_index.tolist() == [[0, 3, 4, 2, 1], [4, 3, 0, 1, 2]]
    g = ops.log_probs_grad(x, y, r, torch.ones(2, dtype=r.logp.dtype, device="cuda"))
    assert torch.isfinite(g).all()


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("offset", [1000.0, -30000.0])
def test_large_common_offset(offset, kind):
    """Only differences between logits count: the offset's own size must not reach the sums."""
    x, y = problem(6, 3001, torch.float64, seed=5)
    x = (x + offset).to(kind)
    r, want = check_scores(x, y, 11)
    dl, dh = weights(6, kind)
    check_grad(x, y, r, want, dl, dh)


def clustered_rows(classes, top):
    rows = 10
    x = torch.zeros(rows, classes, dtype=torch.float64)
    ar = torch.arange(classes, dtype=torch.float64)
    x[0] = ar / classes * 4
    x[1] = -ar / classes * 4
    x[2, : top] = 1.0
    x[3, -top:] = 1.0
    for i, step in enumerate((8, 64, 512, 2048, 4096)):
        x[4 + i, ::step] = 2.0 + torch.arange(len(x[0, ::step]), dtype=torch.float64) / 1e3
    x[9] = (torch.arange(classes) * 2654435761 % 17).double() / 16
    return x, torch.arange(rows, dtype=torch.int64)


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("classes", [16, 50, 200, 500, 4096, 20000, 128000])
def test_ties_and_clustered_alternatives(classes, kind):
    """Alternatives that sit together, far apart, all equal, or on one stride that a single lane would own."""
    top = min(64, classes)
    x, y = clustered_rows(classes, top)
    check_scores(x.to(kind).cuda(), y.cuda(), top)


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("classes,times", [(16, 1640), (50, 1640), (200, 1640), (1025, 52), (4096, 52), (16384, 52), (4096, 105)])
def test_ties_and_clustered_alternatives_in_many_rows(classes, times, kind):
    top = min(64, classes)
    x, y = clustered_rows(classes, top)
    check_scores(x.to(kind).cuda().repeat(times, 1), y.cuda().repeat(times), top)


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("rows,classes", [(3, 1025), (3, 4096), (1100, 4096), (3, 20000), (2, 128000)])
@pytest.mark.parametrize("count", [1, 40, 51, 52, 53, 60, 63, 64, 65])
def test_few_large_values_each_in_a_load_of_its_own(rows, classes, kind, count):
    """With 64 alternatives: as many groups hold large values, one each, as there are, and the rest of the row is equal."""
    if rows > 3 and kind == torch.float64:
        rows = 2100
    x = torch.zeros(rows, classes, dtype=torch.float64)
    width = 128 // torch.finfo(kind).bits
    at = torch.randperm(min(classes // width, 512), generator=torch.Generator().manual_seed(count))[:count] * width
    x[:, at] = 2.0 + torch.arange(count, dtype=torch.float64) / 64
    x[0, at] = 2.0
    check_scores(x.to(kind).cuda(), torch.zeros(rows, dtype=torch.int64, device="cuda"), 64)


SIGNALLING = {torch.float32: (torch.int32, 0x7f800001), torch.float64: (torch.int64, 0x7ff0000000000001),
              torch.bfloat16: (torch.int16, 0x7f81), torch.float16: (torch.int16, 0x7c01)}


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("rows,classes", [(3, 13), (3, 700), (3, 5000), (600, 5000), (2, 200000)])
def test_rows_of_signalling_nans(rows, classes, kind):
    """Arithmetic turns these NaNs into others, so a largest value of theirs need not be found again; the results of
    the calls before lie in the memory that is written."""
    x, y = problem(rows, classes, kind, seed=9)
    bits, code = SIGNALLING[kind]
    x = x.contiguous()
    x.view(bits)[0] = code
    x.view(bits)[1, ::3] = code
    top = min(classes, 40)
    for _ in range(3):
        torch.full((rows, top), 5, dtype=torch.int32, device="cuda")
        torch.full((rows, top), 5, dtype=wide(kind), device="cuda")
        r = ops.log_probs(x, y, top=top)
        for k in (0, 1):
            assert torch.isnan(r.logp[k]) and torch.isnan(r.entropy[k]) and torch.isnan(r.top_logp[k]).all()
            assert (r.top_index[k] == -1).all()
    x[:2] = 0.5
    check_scores(x, y, top)


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("rows,classes", [(64, 2), (40, 13), (40, 200), (40, 1000), (40, 5000), (600, 5000), (40, 100000)])
def test_no_log_probability_above_zero_and_no_entropy_below(rows, classes, kind):
    """One class with all of the weight, or nearly all of it."""
    g = torch.Generator().manual_seed(rows + classes)
    x = torch.full((rows, classes), -1e4, dtype=torch.float64)
    x[1::2] = -20.0 * torch.rand(len(x[1::2]), 1, generator=g, dtype=torch.float64)
    at = torch.randint(0, classes, (rows,), generator=g)
    x[torch.arange(rows), at] = 17.0 * torch.rand(rows, generator=g, dtype=torch.float64)
    x, y = x.to(kind).cuda(), at.int().cuda()
    r, _ = check_scores(x, y, min(classes, 5))
    assert (r.logp <= 0).all() and (r.top_logp <= 0).all() and (r.stats[3] >= 0).all() and (r.entropy >= 0).all()


def test_target_out_of_range_is_seen():
    x, _ = problem(4, 13, torch.float32)
    y = torch.tensor([12, 13, 2 ** 31 - 1, -1], dtype=torch.int32).cuda()
    r, want = check_scores(x, y, 3)
    assert torch.isnan(r.logp).tolist() == [False, True, True, False]
    dl, dh = weights(4, torch.float32)
    check_grad(x, y, r, want, dl, dh)
    y64 = torch.tensor([12, 2 ** 40, -2 ** 40, 3], dtype=torch.int64).cuda()
    r, want = check_scores(x, y64, 3)
    check_grad(x, y64, r, want, dl, dh)


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("classes", [13, 5000])
def test_gradient_in_place(classes, kind):
    x, y = problem(9, classes, kind, seed=6, pad=3)
    r, want = check_scores(x, y, 0)
    dl, dh = weights(9, kind)
    keep = x.clone()
    g = ops.log_probs_grad(keep, y, r, dl, dh)
    same = ops.log_probs_grad(x, y, r, dl, dh, out=x)
    assert same.data_ptr() == x.data_ptr() and torch.equal(same, g)


@pytest.mark.parametrize("classes", [13, 700, 6000])
def test_gradient_against_differences(classes):
    """Central differences in fp64: step h leaves h^2/6 of a third derivative (at most 1 here) and the values'
    own rounding over h."""
    x, y = problem(3, classes, torch.float64, seed=7)
    dl, dh = weights(3, torch.float64)
    r = ops.log_probs(x, y)
    g = ops.log_probs_grad(x, y, r, dl, dh)
    h = 1e-4
    for j in [0, 1, classes // 2, classes - 1] + y.tolist():
        f = []
        for s in (h, -h):
            z = x.clone()
            z[:, j] += s
            q = ops.log_probs(z, y)
            f.append(dl * q.logp + dh * q.entropy)
        numeric = (f[0] - f[1]) / (2 * h)
        assert (numeric - g[:, j]).abs().max() < h * h * (1 + dh.abs().max() * 20) + 1e-13 * 40 / h


def test_rows_and_streams_without_waiting():
    """Calls on two streams at once, results used on a third after its wait; no state is shared."""
    main = torch.cuda.current_stream()
    probs = [problem(40, 30011, torch.bfloat16, seed=s) for s in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for (x, y), st in zip(probs, streams):
        st.wait_stream(main)
        with torch.cuda.stream(st):
            got.append(ops.log_probs(x, y, top=9))
    for st in streams:
        main.wait_stream(st)
    for (x, y), r in zip(probs, got):
        check_scores(x, y, 9, got=r)


@pytest.mark.parametrize("rows,classes", [(128, 13), (2, 90000), (64, 5000)])
def test_captured_and_replayed(rows, classes):
    x, y = problem(rows, classes, torch.bfloat16, seed=8)
    dl, dh = weights(rows, torch.bfloat16)
    ops.log_probs_grad(x, y, ops.log_probs(x, y, top=4), dl, dh)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = ops.log_probs(x, y, top=4)
            d = ops.log_probs_grad(x, y, r, dl, dh)
        graphs.append((g, r, d))
    for seed in range(4):
        nx, ny = problem(rows, classes, torch.bfloat16, seed=20 + seed)
        x.copy_(nx)
        y.copy_(ny)
        for g, _, _ in graphs:
            g.replay()
        eager = ops.log_probs(x, y, top=4)
        grad = ops.log_probs_grad(x, y, eager, dl, dh)
        torch.cuda.synchronize()
        for _, r, d in graphs:
            assert all(torch.equal(a, b) for a, b in zip(r, eager)) and torch.equal(d, grad)


def test_rows_beyond_32_bits():
    """Element offsets past 2^31 (bf16, 2.2e9 logits), first and last rows looked at."""
    classes, rows = 131072, 17000
    x = torch.zeros((rows, classes), dtype=torch.bfloat16, device="cuda")
    for r in (0, 16383, 16384, rows - 1):
        x[r] = torch.randn(classes, device="cuda").to(torch.bfloat16)
    y = torch.full((rows,), 5, dtype=torch.int32, device="cuda")
    some = torch.tensor([0, 1, 16383, 16384, rows - 2, rows - 1])
    r = ops.log_probs(x, y, top=3)
    picked = ops.LogProbs(*(t[some.cuda()] for t in r[:4]), r.stats[:, some.cuda()].contiguous())
    _, want = check_scores(x[some.cuda()], y[some.cuda()], 3, got=picked)
    dl = torch.ones(rows, device="cuda")
    ops.log_probs_grad(x, y, r, dl, None, out=x)
    g = ref.log_probs_grad(want, y[some.cuda()], dl[some.cuda()], None)
    assert (x[some.cuda()].cpu().double() - g).abs().max() < 2.0 ** -8


def test_empty_and_refused():
    x, y = problem(4, 13, torch.float32)
    r = ops.log_probs(x[:0], y[:0], top=2)
    assert r.logp.shape == (0,) and r.top_index.shape == (0, 2)
    assert ops.log_probs_grad(x[:0], y[:0], r, r.logp).shape == (0, 13)
    ok = ops.log_probs(x, y)
    bare = ops.log_probs(x, y, want_entropy=False)
    for call, err in [
        (lambda: ops.log_probs(x.cpu(), y), TypeError),
        (lambda: ops.log_probs(x.int(), y), TypeError),
        (lambda: ops.log_probs(x, y.cpu()), TypeError),
        (lambda: ops.log_probs(x, y.float()), TypeError),
        (lambda: ops.log_probs(x, y[:3]), ValueError),
        (lambda: ops.log_probs(x, torch.stack([y, y], 1)[:, 0]), ValueError),
        (lambda: ops.log_probs(x[0], y), ValueError),
        (lambda: ops.log_probs(x[:, :0], y), ValueError),
        (lambda: ops.log_probs(x.t(), y), ValueError),
        (lambda: ops.log_probs(x[:1].expand(4, 13), y), ValueError),
        (lambda: ops.log_probs(x, y, top=14), ValueError),
        (lambda: ops.log_probs(x, y, top=-1), ValueError),
        (lambda: ops.log_probs_grad(x, y, ok), ValueError),
        (lambda: ops.log_probs_grad(x, y, bare, None, ok.logp), ValueError),
        (lambda: ops.log_probs_grad(x, y, ok, ok.logp.double()), TypeError),
        (lambda: ops.log_probs_grad(x, y, ok, ok.logp[:3]), ValueError),
        (lambda: ops.log_probs_grad(x, y, ok, ok.logp, out=x.double()), TypeError),
        (lambda: ops.log_probs_grad(x, y, ok, ok.logp, out=x[:3]), ValueError),
        (lambda: ops.log_probs_grad(x[:, :12], y, ops.log_probs(x[:, :12], y), ok.logp, out=x[:, 1:]), ValueError),
    ]:
        with pytest.raises(err):
            call()
    x64, _ = problem(70, 70, torch.float32)
    with pytest.raises(ValueError):
        ops.log_probs(x64, torch.zeros(70, dtype=torch.int32, device="cuda"), top=65)


def scored_into(x, y, top, fill):
    """ccnn_log_probs into results that hold `fill` before -> (logp, entropy, top_logp, top_index)."""
    rows, classes = x.shape
    stats, top_logp = (torch.full((n, rows), fill, dtype=wide(x.dtype), device="cuda") for n in (4, top))
    index = torch.full((rows, top), int(fill), dtype=torch.int32, device="cuda")
    kind = ops._TYPES[x.dtype]
    need = L.load().ccnn_log_probs_workspace_bytes(rows, classes, top, kind)
    ws = torch.full((need + 1,), 7, dtype=torch.uint8, device="cuda")
    L.check(L.load().ccnn_log_probs(x.data_ptr(), kind, rows, classes, classes, y.data_ptr(), 4, top, 1, stats.data_ptr(),
                                    top_logp.data_ptr(), index.data_ptr(), ws.data_ptr() if need else None, need,
                                    torch.cuda.current_stream().cuda_stream), "ccnn_log_probs")
    return stats[0], stats[1], top_logp.view(rows, top), index


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("rows,classes", [(6, 13), (6, 700), (6, 1025), (6, 1030), (6, 2047), (6, 4095), (6, 40001), (6, 70003), (600, 1025),
                                          (600, 4095)])
@pytest.mark.parametrize("top", [1, 2, 13])
def test_rows_of_negative_nans_have_no_alternatives(rows, classes, kind, top):
    """A NaN with its sign bit set orders below -inf, so no element may reach the bar; every place says so, whatever
    the memory held before."""
    x, y = problem(rows, classes, kind, seed=12)
    x = x.contiguous()
    bits = {2: torch.int16, 4: torch.int32, 8: torch.int64}[x.element_size()]
    part = classes % (16 // x.element_size()) or 1
    x.view(bits)[0::6] = -1
    x.view(bits)[1::6, classes - part:] = -1           # all of the last, partial load
    x.view(bits)[2::6, 1:] = -1
    x[3::6] = math.nan
    x[4::6, classes - 1] = INF
    logp, entropy, top_logp, index = scored_into(x, y, top, 5.0)
    bad = torch.arange(rows, device="cuda") % 6 != 5
    assert torch.isnan(logp[bad]).all() and torch.isnan(entropy[bad]).all()
    assert (index[bad] == -1).all() and torch.isnan(top_logp[bad]).all()
    want = ref.log_probs(x[~bad], y[~bad], top)
    assert torch.equal(index[~bad].cpu(), want["top_index"]) and torch.isfinite(logp[~bad]).all()


def test_calls_keep_no_references_to_none():
    """An absent result is one reference to None, given back with the result."""
    x, y = problem(4, 13, torch.float32)
    for top, want_entropy in [(0, False), (0, True), (2, False), (2, True)]:
        ops.log_probs(x, y, top=top, want_entropy=want_entropy)
        before = sys.getrefcount(None)
        for _ in range(1000):
            ops.log_probs(x, y, top=top, want_entropy=want_entropy)
        assert abs(sys.getrefcount(None) - before) < 100, (top, want_entropy)


def tight_bound(logits, want, dtype):
    """How far the log sum may be off where a row has 512 parts at least (64 with 512 rows or more), u half a step.

    A thread adds n / parts terms, then 6 + 8 + 6 steps join lanes, waves and slices, and the slices of a lane: n / parts
    + 64 additions, u each.  A term e^d at d from a reference carries 3u|d| + 2u; the reference is at most 4
    above or below the largest element's neighbourhood, so on average over the sum that is 3u (E|x - m| + 4) + 2u.  A thread's
    reference moves up by more than 4 at a time, at most R / 4 + 1 times over the row's range R, and each
    joining step moves a sum once: 3u of every distance, which add up to R + 4, and 3u of each of the at most
    R / 4 + 8 moves.  The logarithm and its argument: 4u of it."""
    x = logits.detach().cpu().double()
    u = ref.half_step(dtype)
    d = (x - torch.where(want["m"] == -INF, 0.0, want["m"])[:, None]).abs()
    span = torch.where(torch.isfinite(d), d, 0.0).clamp(max=120.0 if dtype == torch.float32 else 760.0).amax(1).nan_to_num(0.0)
    near = torch.where(want["p"] > 0, want["p"] * d, 0.0).sum(1).nan_to_num(0.0)
    parts = 64 if x.shape[0] >= 512 else 512
    adds = x.shape[1] / parts + 64
    return u * (adds + 3 * (near + 4) + 2 + 3 * (span + 4) + 3 * (span / 4 + 8) + 4 * want["l"].abs().nan_to_num(0.0, 0.0, 0.0)), near


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("rows,classes", [(4, 1027), (4, 4099), (513, 1037), (4, 32003), (4, 65543), (4, 70003), (3, 131077), (2, 200005)])
def test_no_element_is_lost_from_a_long_row(rows, classes, kind):
    """Sums within the bound that the real number of additions gives, at sizes that end inside a load; the last elements of
    some rows, or the only ones of all slices but one, carry the whole sum."""
    width = 128 // torch.finfo(kind).bits
    x, y = problem(rows, classes, kind, seed=13)
    x = x.contiguous()
    u = ref.half_step(wide(kind))

    def check():
        r, want = check_scores(x, y, min(classes, 3))
        b, near = tight_bound(x, want, wide(kind))
        close(r.stats[3], want["l"], b, "l")
        close(r.logp, want["logp"], b + 4 * u * want["logp"].abs().nan_to_num(0, 0, 0), "logp")
        # l is off by b; t / s, with the reference at most 4 above and 4 below where it ends, by b (near + 8), and s takes b near more
        close(r.entropy, want["entropy"], b * (9 + 2 * near) + 4 * u * want["entropy"].abs(), "entropy")

    check()
    x[:] = 1.0
    check()
    rest = classes % width or 1
    x[:] = -INF
    x[:, classes - rest:] = torch.arange(rest, dtype=torch.float64).to(kind).cuda() / 4
    y[:] = classes - 1
    check()
    x[:] = -20.0
    x[:, classes - rest:] = 5.0
    check()
    x[:, 0] = 5.0
    y[:] = 0
    check()


@pytest.mark.parametrize("rows,classes,kind", [((1 << 24) + 77, 3, torch.float32), ((1 << 22) + 67, 1025, torch.bfloat16), (70001, 1027, torch.float32),
                                               (70001, 1025, torch.float64), ((1 << 22) + 67, 1000, torch.float64)], ids=str)
def test_more_rows_than_one_launch_takes(rows, classes, kind):
    """Rows that repeat every 61 have results that do, whichever launch they are in; some against 64 bits."""
    base, by = problem(61, classes, kind, seed=14)
    at = torch.arange(rows, device="cuda") % 61
    x, y = base[at], by[at]
    r = ops.log_probs(x, y, top=2)
    picked = [0, 1, 60, 61, 65534, 65535, 65536, (1 << 22) - 1, 1 << 22, (1 << 24) - 1, 1 << 24, rows - 1]
    some = torch.tensor([i for i in picked if i < rows], device="cuda")
    part = ops.LogProbs(*(t[some] for t in r[:4]), r.stats[:, some].contiguous())
    _, want = check_scores(x[some], y[some], 2, got=part)
    for t in r[:4]:
        assert torch.equal(t, t[:61][at])
    dl, dh = (w[at] for w in weights(61, kind))
    g = ops.log_probs_grad(x, y, r, dl, dh, out=x)
    assert g.data_ptr() == x.data_ptr()
    exact = ref.log_probs_grad(want, y[some], dl[some], dh[some])
    # probabilities within the bound of the sums, the result rounded once
    off = (g[some].cpu().double() - exact).abs()
    assert (off <= 8 * ref.score_bound(base, ref.log_probs(base, by), wide(kind)).max() + ref.half_step(kind) * exact.abs()).all()
    first = g[:61].clone()
    for a in range(0, rows, 1 << 20):
        assert torch.equal(g[a:a + (1 << 20)], first[at[a:a + (1 << 20)]])


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16], ids=str)
def test_the_longest_row(kind):
    """2^30 classes: equal ones but for a few, so that the sums are known."""
    classes = 1 << 30
    x = torch.zeros((1, classes), dtype=kind, device="cuda")
    at = torch.tensor([classes - 1, 0, (1 << 29) + 5], device="cuda")
    x[0, at] = torch.tensor([12.0, 11.0, 10.0], dtype=kind, device="cuda")
    y = torch.tensor([classes - 1], device="cuda")
    r = ops.log_probs(x, y, top=5)
    total = math.fsum([classes - 3, math.exp(12), math.exp(11), math.exp(10)])
    weighed = math.fsum([12 * math.exp(12), 11 * math.exp(11), 10 * math.exp(10)])
    u = ref.half_step(torch.float32)
    # 512 slices of 512 threads: 4096 additions each and 64 to join; the terms' own errors and the log's as in score_bound
    bound = u * (4096 + 64 + 6 * 12 + 30 + 4 * math.log(total))
    assert abs(r.logp.item() - (12 - math.log(total))) <= bound
    assert abs(r.entropy.item() - (math.log(total) - weighed / total)) <= 30 * bound
    assert r.top_index.tolist() == [[classes - 1, 0, (1 << 29) + 5, 1, 2]]
    d = ops.log_probs_grad(x, y, r, torch.ones(1, device="cuda"), None, out=x)
    want = -1.0 / total
    assert abs(d[0, 7].item() / want - 1) < 0.01 and abs(d[0, classes - 2].item() / want - 1) < 0.01
    assert abs(d[0, classes - 1].item() - (1 - math.exp(12) / total)) < 2 ** -8 and abs(d[0, 0].item() / (math.exp(11) * want) - 1) < 0.01
