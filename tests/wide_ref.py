"""64-bit restatements, on the CPU, of the scoring and optimiser operators, with the bounds their
32-bit forms are held to."""
import math

import torch

INF = math.inf


def half_step(dtype):
    """A rounding to `dtype` is off by at most this, relative to the value."""
    return torch.finfo(dtype).eps / 2


def log_probs(logits, targets, top=0):
    """dict(logp, entropy, top_logp, top_index, m, l, p, lp) of float64 / int tensors."""
    x = logits.detach().cpu().double()
    y = targets.detach().cpu().long()
    rows, classes = x.shape
    m = x.max(1).values
    bad = torch.isnan(x).any(1) | (x == INF).any(1)
    empty = (x == -INF).all(1)
    d = x - torch.where(empty, 0.0, m)[:, None]
    e = d.exp()
    s = e.sum(1)
    l = s.log()
    lp = d - l[:, None]
    p = e / s[:, None]
    lp[empty], p[empty] = -INF, 0.0
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(1)
    logp = lp.gather(1, y.clamp(0, classes - 1)[:, None])[:, 0]
    logp[y < 0] = 0.0
    logp[(y >= classes) | bad] = math.nan
    m, l = m.clone(), l.clone()
    m[bad], l[bad], entropy[bad], lp[bad], p[bad] = (math.nan,) * 5
    l[empty], entropy[empty] = -INF, 0.0
    top_index = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top].int()
    top_logp = lp.gather(1, top_index.long())
    top_index[bad] = -1
    return dict(logp=logp, entropy=entropy, top_logp=top_logp, top_index=top_index, m=m, l=l, p=p, lp=lp)


def log_probs_grad(ref, targets, d_logp, d_entropy):
    y = targets.detach().cpu().long()
    p, lp = ref["p"], ref["lp"]
    rows, classes = p.shape
    one = torch.zeros_like(p)
    ok = (y >= 0) & (y < classes)
    one[torch.arange(rows)[ok], y[ok]] = 1.0
    dl = torch.zeros(rows, dtype=torch.float64) if d_logp is None else d_logp.detach().cpu().double().clone()
    dl[y < 0] = 0.0
    dh = torch.zeros(rows, dtype=torch.float64) if d_entropy is None else d_entropy.detach().cpu().double()
    safe = torch.where(p > 0, lp + ref["entropy"][:, None], 0.0)
    g = dl[:, None] * (one - p) - dh[:, None] * p * safe
    g[(ref["m"] == -INF)] = 0.0
    g[(y >= classes) | torch.isnan(ref["l"])] = math.nan
    return g


def score_bound(logits, ref, wide):
    """How far log probabilities computed in `wide` may be off, per row.

    With u half a step: a term e^(x-m) carries the rounding of x-m and of its product with log2 e (3u|x-m|
    in the exponent at most) and 2u of the exponential; moving a sum to a larger maximum multiplies it by
    another such factor, and over all moves the distances add up to the range R of the row, their count to no
    more than the additions.  A sum of n terms in at least 16 independent parts takes n/16 + 64 additions
    at most.  So sum e^(x-m) is within (n/16 + 64)(1 + 3)u + 6 R u of itself, where R e^-R < 1 lets far terms
    weigh no more than near ones: log of it is off by that much, plus the roundings of l, x-m and
    logp themselves."""
    x = logits.detach().cpu().double()
    u = half_step(wide)
    far = torch.where(torch.isfinite(x), x, ref["m"][:, None])
    span = (ref["m"][:, None] - far).abs().amax(1).nan_to_num(0.0, 0.0, 0.0)
    span = span.clamp(max=120.0 if wide == torch.float32 else 760.0)     # terms farther down are 0 in `wide`
    n = x.shape[1]
    return u * (4 * (n / 16 + 64) + 6 * span + 4 * ref["l"].abs().nan_to_num(0.0, 0.0, 0.0))


# ------------------------------------------------------------------ AdamW
def e4m3_values():
    v = []
    for code in range(127):
        power, part = code >> 3, code & 7
        v.append(part / 8 * 2.0 ** -6 if power == 0 else (1 + part / 8) * 2.0 ** (power - 7))
    return torch.tensor(v, dtype=torch.float64)


VALUES = e4m3_values()


def encode(x, floor=False):
    """[blocks, 256] float64 -> (codes uint8, scales float32): the nearest of the block's values, ties to the even code."""
    scale = x.abs().amax(1).float() / torch.full((x.shape[0],), 448.0)
    y = torch.where(scale[:, None] > 0, x.abs() / scale[:, None].double(), 0.0).clamp(max=448.0)
    hi = torch.searchsorted(VALUES, y).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    below, above = y - VALUES[lo], VALUES[hi] - y
    code = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    if floor:
        code = torch.where((y > 0) & (code == 0), 1, code)
    return torch.where(x < 0, code + 128, code).to(torch.uint8), scale


def decode(code, scale):
    c = code.long()
    v = torch.where(c >= 128, -VALUES[(c & 127).clamp(max=126)], VALUES[(c & 127).clamp(max=126)])
    return v * scale.double()[:, None]


def to_blocks(tensors):
    """List of 1-d float64 tensors -> [blocks, 256], every tensor filled up with zeros to whole blocks."""
    out = []
    for t in tensors:
        k = -(-t.numel() // 256) * 256
        out.append(torch.cat([t.reshape(-1), torch.zeros(k - t.numel(), dtype=t.dtype)]))
    return torch.cat(out).view(-1, 256) if out else torch.zeros(0, 256, dtype=torch.float64)


def from_blocks(blocks, sizes):
    flat, out, at = blocks.reshape(-1), [], 0
    for n in sizes:
        out.append(flat[at:at + n])
        at += -(-n // 256) * 256
    return out


class AdamW:
    """One step at a time in float64 on lists of 1-d CPU tensors; bits=8 rounds the moments as the codes do."""

    def __init__(self, params, lr, betas=(0.9, 0.999), eps=1e-8, decays=None, bits=32):
        self.p = [p.detach().cpu().double().reshape(-1).clone() for p in params]
        self.m = [torch.zeros_like(p) for p in self.p]
        self.v = [torch.zeros_like(p) for p in self.p]
        self.lr, self.betas, self.eps, self.bits, self.t = lr, betas, eps, bits, 0
        self.decays = decays or [0.01] * len(self.p)
        self.codes = None

    def step(self, grads, scale=1.0, lr=None):
        self.t += 1
        lr = self.lr if lr is None else lr
        (b1, b2), t = self.betas, self.t
        root = []
        for i, g in enumerate(grads):
            g = g.detach().cpu().double().reshape(-1) * scale
            self.m[i] = b1 * self.m[i] + (1 - b1) * g
            self.v[i] = b2 * self.v[i] + (1 - b2) * (g * g)
            up = (self.m[i] / (1 - b1 ** t)) / ((self.v[i] / (1 - b2 ** t)).sqrt() + self.eps)
            self.p[i] = self.p[i] - lr * (self.decays[i] * self.p[i] + up)
        if self.bits == 8:
            sizes = [p.numel() for p in self.p]
            mc, ms = encode(to_blocks(self.m))
            vc, vs = encode(to_blocks([v.sqrt() for v in self.v]), floor=True)
            self.codes = (mc.reshape(-1), vc.reshape(-1), ms, vs)
            self.m = from_blocks(decode(mc, ms), sizes)
            self.v = [r * r for r in from_blocks(decode(vc, vs), sizes)]
