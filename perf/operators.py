"""Cases, plain forms and 64-bit definitions of the scoring and optimiser operators of gcn_amd.ops:

    log_probs        log probability of a given class per row, entropy, the most likely alternatives
    log_probs_grad   gradient of log probability and entropy to the logits (cases "loss": both calls)
    grad_norm        norm over many gradient tensors and the factor that clips it
    AdamW            one decoupled-decay step over many tensors, moments in 32 bits or in 8

`own` false: elementary torch operations; true: the library's kernels, called as a program calls them.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f64": torch.float64, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 256          # elements of a tensor that share one scale in 8 bits
BETAS, EPS, LR, DECAY = (0.9, 0.999), 1e-8, 1e-3, 0.01


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # every labelled-scene pixel of a 610 x 340 image scored against its 13-class label
        {"name": "score pixels", "op": "score", "rows": 207400, "classes": 13, "type": "f32", "top": 3, "pad": 0, "masked": False},
        # one new position of one request over a large vocabulary: the smallest call, latency
        {"name": "score one row", "op": "score", "rows": 1, "classes": 128000, "type": "bf16", "top": 20, "pad": 0, "masked": False},
        # a batch of requests, vocabulary of odd size out of a padded buffer, part of it masked away
        {"name": "score requests", "op": "score", "rows": 61, "classes": 50251, "type": "f16", "top": 8, "pad": 7, "masked": True},
        # the positions of prompts that are scored at once
        {"name": "score prompts", "op": "score", "rows": 2048, "classes": 128000, "type": "bf16", "top": 5, "pad": 0, "masked": False},
        # the loss of one minibatch of the pixel classifier
        {"name": "loss minibatch", "op": "loss", "rows": 128, "classes": 13, "type": "f32", "pad": 0, "entropy": True},
        # a training batch over a vocabulary of odd size, with an entropy bonus
        {"name": "loss odd", "op": "loss", "rows": 3001, "classes": 32003, "type": "f32", "pad": 1, "entropy": True},
        # a training batch over a large vocabulary
        {"name": "loss batch", "op": "loss", "rows": 4096, "classes": 128000, "type": "bf16", "pad": 0, "entropy": False},
        # the six tensors of the pixel classifier at 103 bands
        {"name": "step network", "op": "step", "net": True, "layers": 0, "width": 103, "type": "f32", "bits": 32, "clip": True},
        # a large model in bf16 with its fp32 master copy, clipped
        {"name": "step large", "op": "step", "net": False, "layers": 16, "width": 1024, "type": "bf16", "bits": 32, "clip": True},
        # tensors of odd sizes with moments in 8 bits
        {"name": "step 8 odd", "op": "step", "net": False, "layers": 3, "width": 333, "type": "f32", "bits": 8, "clip": False},
        # a large model with moments in 8 bits
        {"name": "step 8 large", "op": "step", "net": False, "layers": 8, "width": 1024, "type": "bf16", "bits": 8, "clip": False},
        # the norm of a large model's gradients by itself, as a monitor reads it
        {"name": "norm large", "op": "norm", "net": False, "layers": 16, "width": 1024, "type": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm, odd and even alike."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["score", "loss", "step", "step", "norm"])
    if op in ("score", "loss"):
        kind = rng.choice(["f32", "bf16", "f16", "bf16", "f64"])
        classes = _spread(rng, 2, 1024 if kind == "f64" else 128000)
        rows = _spread(rng, 1, min(207400, max(1, (1 << 28) // classes)))
        case = {"op": op, "rows": rows, "classes": classes, "type": kind, "pad": rng.choice([0, 0, 1, 8, 13])}
        if op == "score":
            return {**case, "top": rng.randint(0, min(classes, 32)), "masked": rng.random() < 0.3}
        return {**case, "entropy": rng.random() < 0.5}
    kind = rng.choice(["f32", "bf16", "f16"])
    net = rng.random() < 0.2
    width = rng.randint(21, 448) if net else _spread(rng, 32, 1024)
    layers = 0 if net else rng.randint(1, 8)
    case = {"op": op, "net": net, "layers": layers, "width": width, "type": "f32" if net else kind}
    return case if op == "norm" else {**case, "bits": rng.choice([8, 32]), "clip": rng.random() < 0.5}


def _sizes(case):
    """Elements of each tensor of a case's parameter list."""
    w = case["width"]
    if case["net"]:      # conv filters, FC-100, 13 classes (20 filters of 171 taps, pooled by two)
        features = 20 * (((w - 20) // 2) // 2 + 1)
        return [3420, 20, 100 * features, 100, 1300, 13]
    sizes = [1000 * w]
    for _ in range(case["layers"]):
        sizes += [w, w * w, w * w, w * w, w * w, w, 4 * w * w, 4 * w * w]
    return sizes + [w, 13 * w, 13]


# ---------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]

    def normal(*shape, kind=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=kind)

    if case["op"] in ("score", "loss"):
        rows, classes = case["rows"], case["classes"]
        whole = normal(rows, classes + case["pad"], kind=kind if kind == torch.float64 else torch.float32).mul_(2.5)
        targets = torch.randint(0, classes, (rows,), generator=g, device="cuda", dtype=torch.int32)
        if case.get("masked"):     # a third of the classes not allowed; the given class always is
            off = torch.rand(rows, classes, generator=g, device="cuda") < 0.33
            off.scatter_(1, targets.long()[:, None], False)
            whole[:, :classes].masked_fill_(off, -math.inf)
        logits = whole.to(kind)[:, :classes]
        s = {"op": case["op"], "logits": logits, "targets": targets, "top": case.get("top", 0)}
        if case["op"] == "loss":   # padding positions carry no class; weights as a mean over the rest has them
            targets[torch.rand(rows, generator=g, device="cuda") < 0.05] = -1
            wide = torch.float64 if kind == torch.float64 else torch.float32
            mean = 1 if kind == torch.float16 else rows     # half-precision gradients are scaled up
            s["d_logp"] = (-torch.rand(rows, generator=g, device="cuda") / mean).to(wide)
            s["d_entropy"] = (-0.01 * torch.rand(rows, generator=g, device="cuda") / mean).to(wide) if case["entropy"] else None
        return s

    sizes = _sizes(case)
    n, starts = sum(sizes), [sum(sizes[:i]) for i in range(len(sizes))]
    grad = normal(n).mul_(1e-3).to(kind)
    s = {"op": case["op"], "grad": grad, "grads": [grad[a:a + k] for a, k in zip(starts, sizes)], "max_norm": 1.0}
    s["max_norm"] = 0.5e-3 * math.sqrt(n)
    if case["op"] == "norm":
        return s
    param = normal(n).mul_(0.05)
    s["clip"], s["bits"], s["step"] = case["clip"], case["bits"], 100
    s["master"] = param if kind != torch.float32 else None
    s["param"] = param.to(kind)
    decays = [DECAY if k > case["width"] else 0.0 for k in sizes]
    s["decay"] = torch.repeat_interleave(torch.tensor(decays, device="cuda"), torch.tensor(sizes, device="cuda"))
    m, v = normal(n).mul_(3e-4), normal(n).mul_(1e-3).square_()
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
        moments = {"m": m, "v": v}
    else:
        blocks = [-(-k // BLOCK) for k in sizes]
        first = [sum(blocks[:i]) * BLOCK for i in range(len(sizes))]
        counts = torch.tensor(sizes, device="cuda")
        s["place"] = torch.arange(n, device="cuda") + torch.repeat_interleave(torch.tensor([a - b for a, b in zip(first, starts)], device="cuda"), counts)
        s["table"] = _e4m3()
        moments = {}
        for name, x in (("m", m), ("v", v.sqrt())):
            moments[name], moments[name + "_scale"] = _encode(_blocks(x.double(), s["place"], sum(blocks)))
        s.update(moments)
    if own:
        from gcn_amd import ops
        params = [s["param"][a:a + k] for a, k in zip(starts, sizes)]
        s["optimizer"] = ops.AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=decays, state_bits=case["bits"])
        s["optimizer"].load_state_dict({"step": s["step"], "master": s["master"], **moments})
        for name in ("m", "v", "m_scale", "v_scale", "decay", "place", "table"):
            s.pop(name, None)
    return s


# ---------------------------------------------------------------------------- one pass
def run(s):
    if s["op"] == "score":
        return _score_own(s) if own else _score(s["logits"], s["targets"], s["top"])
    if s["op"] == "loss":
        return _loss_own(s) if own else _loss(s)
    if s["op"] == "norm":
        return _norm_own(s) if own else _norm(s["grad"], s["max_norm"])
    return _step_own(s) if own else _step(s)


def _score_own(s):
    from gcn_amd import ops
    r = ops.log_probs(s["logits"], s["targets"], top=s["top"])
    return [r.logp, r.entropy, r.top_logp, r.top_index]


def _loss_own(s):
    from gcn_amd import ops
    r = ops.log_probs(s["logits"], s["targets"], want_entropy=s["d_entropy"] is not None)
    return [r.logp, r.entropy, ops.log_probs_grad(s["logits"], s["targets"], r, s["d_logp"], s["d_entropy"])]


def _norm_own(s):
    from gcn_amd import ops
    return ops.grad_norm(s["grads"], s["max_norm"])


def _step_own(s):
    from gcn_amd import ops
    clip = ops.grad_norm(s["grads"], s["max_norm"]) if s["clip"] else None
    s["optimizer"].step(s["grads"], clip=clip)
    m, v = s["optimizer"].moments()
    return [s["param"], s["optimizer"].master, m, v, clip]


# ---------------------------------------------------------------------------- plain forms
def _wide(x):
    return x if x.dtype == torch.float64 else x.float()


def _score(logits, targets, top, want_entropy=True):
    x = _wide(logits)
    high = x.amax(1, keepdim=True)
    d = x - torch.where(high == -math.inf, 0.0, high)
    e = d.exp()
    total = e.sum(1)
    log_total = total.log()
    given = targets.clamp(min=0).long()[:, None]
    logp = torch.where(targets < 0, 0.0, d.gather(1, given)[:, 0] - log_total).to(x.dtype)
    entropy = None
    if want_entropy:
        entropy = log_total - torch.where(e > 0, e * d, 0.0).sum(1) / total
    if not top:
        return [logp, entropy, None, None]
    if x.dtype == torch.float64:                 # few classes: a stable order keeps the lowest index of equals first
        value, index = torch.sort(x, dim=1, descending=True, stable=True)
        value, index = value[:, :top], index[:, :top]
    else:                                        # the value's order above the index's in one whole number
        bits = (x + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
        key = (order << 32) - torch.arange(x.shape[1], device=x.device)
        index = -torch.topk(key, top, 1).values
        index = index - ((index >> 32) << 32)
        value = x.gather(1, index)
    return [logp, entropy, d.gather(1, index) - log_total[:, None], index.int()]


def _loss(s):
    x, entropy = _wide(s["logits"]), None
    d = x - x.amax(1, keepdim=True)
    e = d.exp()
    total = e.sum(1, keepdim=True)
    p, lp = e / total, d - total.log()
    taken = s["targets"] >= 0
    given = s["targets"].clamp(min=0).long()[:, None]
    logp = torch.where(taken, lp.gather(1, given)[:, 0], 0.0)
    w = torch.where(taken, s["d_logp"], 0.0)
    grad = -w[:, None] * p
    grad.scatter_add_(1, given, w[:, None])
    if s["d_entropy"] is not None:
        entropy = -(p * lp).sum(1)
        grad = grad - s["d_entropy"][:, None] * p * (lp + entropy[:, None])
    return [logp, entropy, grad.to(s["logits"].dtype)]


def _norm(grad, max_norm):
    norm = grad.double().square().sum().sqrt()
    return torch.stack([norm, torch.clamp(max_norm / norm, max=1.0)])


def _step(s):
    clip = _norm(s["grad"], s["max_norm"]) if s["clip"] else None
    s["step"] += 1
    c1, c2 = 1 - BETAS[0] ** s["step"], 1 - BETAS[1] ** s["step"]
    wide = torch.float32 if s["bits"] == 32 else torch.float64      # borders between codes are decided in 64 bits
    g = s["grad"].to(wide)
    if clip is not None:
        g = g * clip[1].to(wide)
    if s["bits"] == 32:
        m, v = s["m"], s["v"]
        m.mul_(BETAS[0]).add_(g, alpha=1 - BETAS[0])
        v.mul_(BETAS[1]).addcmul_(g, g, value=1 - BETAS[1])
        root = v.sqrt()
    else:
        m = _decode(s["m"], s["m_scale"], s["table"])[s["place"]] * BETAS[0] + (1 - BETAS[0]) * g
        v = _decode(s["v"], s["v_scale"], s["table"])[s["place"]].square() * BETAS[1] + (1 - BETAS[1]) * g.square()
        root = v.sqrt()
        nb = s["m"].numel() // BLOCK
        s["m"], s["m_scale"] = _encode(_blocks(m, s["place"], nb))
        s["v"], s["v_scale"] = _encode(_blocks(root, s["place"], nb), floor=True)
    p = s["param"] if s["master"] is None else s["master"]
    p.copy_(p - LR * (s["decay"] * p + (m / c1) / (root / math.sqrt(c2) + EPS)))
    if s["master"] is not None:
        s["param"].copy_(p)
    if s["bits"] == 8:
        m = _decode(s["m"], s["m_scale"], s["table"])[s["place"]].float()
        v = _decode(s["v"], s["v_scale"], s["table"])[s["place"]].square().float()
    return [s["param"], s["master"], m, v, clip]


def _e4m3():
    """The value of each 8-bit code: a sign, 4 bits of exponent, 3 of fraction; the largest is 448."""
    code = torch.arange(256, device="cuda")
    power, part = (code >> 3) & 15, (code & 7).double() / 8
    size = torch.where(power == 0, part * 2.0 ** -6, (1 + part) * torch.pow(2.0, power.double() - 7))
    size[127] = size[255] = math.nan
    return torch.where(code >= 128, -size, size)


def _blocks(x, place, count):
    padded = torch.zeros(count * BLOCK, dtype=x.dtype, device=x.device)
    padded[place] = x
    return padded.view(count, BLOCK)


def _encode(x, floor=False):
    """Blocks of 64-bit values as 8-bit codes and one 32-bit scale each; `floor`: what is not zero keeps the smallest code."""
    high = x.abs().amax(1).float()
    scale = high / torch.full_like(high, 448.0)            # a division, where a plain number would be multiplied by its inverse
    y = torch.where(scale[:, None] > 0, x.abs() / scale[:, None].double(), 0.0).clamp_(max=448.0)
    power = (torch.frexp(y).exponent - 1).clamp_(min=-6)
    eighths = torch.round(torch.ldexp(y, 3 - power))       # 8..16 eighths of 2^power, fewer below 2^-6
    code = eighths.long() + ((power + 6).long() << 3)
    if floor:
        code = torch.where((x > 0) & (scale[:, None] > 0), code.clamp(min=1), code)
    return torch.where(x < 0, code + 128, code).to(torch.uint8).view(-1), scale


def _decode(code, scale, table):
    return (table[code.int()].view(-1, BLOCK) * scale[:, None].double()).view(-1)


# ---------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] in ("score", "loss"):
        n, size = case["rows"] * case["classes"], TYPES[case["type"]].itemsize
        out = 8 if size == 8 else 4
        if case["op"] == "score":
            return {"bytes": n * size + case["rows"] * (4 + 2 * out + case["top"] * (out + 4)), "flops": 6.0 * n}
        return {"bytes": 2 * n * size + case["rows"] * (4 + 3 * out), "flops": 10.0 * n}
    n, size = sum(_sizes(case)), TYPES[case["type"]].itemsize
    if case["op"] == "norm":
        return {"bytes": n * size + 16, "flops": 2.0 * n}
    params = 2 * size if size == 4 else size + 8
    moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 8     # in 8 bits also read out as values
    return {"bytes": n * (params + size + moments), "flops": 16.0 * n}


# ---------------------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "norm":
        return _exact_norm(s["grad"], s["max_norm"])
    if s["op"] == "step":
        return _exact_step(s)
    x = s["logits"].double()
    lp = x - torch.logsumexp(x, 1, keepdim=True)
    logp = lp.gather(1, s["targets"].clamp(min=0).long()[:, None])[:, 0].masked_fill(s["targets"] < 0, 0.0)
    p = lp.exp()
    if s["op"] == "score":
        entropy = -torch.special.xlogy(p, p).sum(1)
        if not s["top"]:
            return [logp, entropy, None, None]
        if x.numel() > 1 << 27:                 # a stable order of so many takes too long
            return [logp, entropy, torch.topk(lp, s["top"], 1).values, None]
        index = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :s["top"]]
        return [logp, entropy, lp.gather(1, index), index.int()]
    one = torch.zeros_like(p).scatter_(1, s["targets"].clamp(min=0).long()[:, None], 1.0)
    grad = (one - p) * torch.where(s["targets"] < 0, 0.0, s["d_logp"].double())[:, None]
    if s["d_entropy"] is None:
        return [logp, None, grad]
    entropy = -(p * lp).sum(1)
    return [logp, entropy, grad + s["d_entropy"].double()[:, None] * (-p * lp - p * entropy[:, None])]


def _exact_norm(grad, max_norm):
    norm = torch.linalg.vector_norm(grad.double())
    return torch.stack([norm, torch.minimum(max_norm / norm, torch.ones_like(norm))])


def _exact_step(s):
    clip = _exact_norm(s["grad"], s["max_norm"]) if s["clip"] else None
    g = s["grad"].double() * (1.0 if clip is None else clip[1])
    t = s["step"] + 1
    p = (s["param"] if s["master"] is None else s["master"]).double()
    if s["bits"] == 32:
        m, v = s["m"].double(), s["v"].double()
    else:
        m = (s["table"][s["m"].long()] * s["m_scale"].double().repeat_interleave(BLOCK))[s["place"]]
        v = (s["table"][s["v"].long()] * s["v_scale"].double().repeat_interleave(BLOCK))[s["place"]] ** 2
    m = torch.lerp(m, g, 1 - BETAS[0])
    v = torch.lerp(v, g * g, 1 - BETAS[1])
    p = p * (1 - LR * s["decay"].double()) - LR * (m / (1 - BETAS[0] ** t)) / (torch.sqrt(v / (1 - BETAS[1] ** t)) + EPS)
    if s["bits"] == 8:
        m, v = _nearest(m, s), _nearest(v.sqrt(), s, floor=True).square()
    return [p.to(s["param"].dtype).double() if s["master"] is not None else p, p if s["master"] is not None else None, m, v, clip]


def _nearest(x, s, floor=False):
    """Each element as the nearest value that its block's 8-bit codes have, by the borders between the codes; equally near: the even code."""
    values = s["table"][:127]
    borders = (values[1:] + values[:-1]) / 2
    padded = torch.zeros(s["m"].numel(), dtype=torch.float64, device=x.device).index_copy_(0, s["place"], x)
    high = padded.abs().view(-1, BLOCK).max(1).values.to(torch.float32)
    scale = (high / torch.full_like(high, 448.0)).double().repeat_interleave(BLOCK)
    y = (padded.abs() / scale).nan_to_num(0.0)
    low, up = torch.bucketize(y, borders), torch.bucketize(y, borders, right=True)
    code = torch.where((low != up) & (low % 2 == 1), up, low)
    if floor:
        code = code.clamp(min=1) * (y > 0)
    return (torch.sign(padded) * values[code] * scale)[s["place"]]
